"""Cases and plain forms of the operators on a paged key/value cache held in 4 bits.

Three operators: attention that reads the cache, writing rows into the cache (and reading
them back), and the handling of its pages (reserve, fork, copy, free, compact).  `run` computes
them in elementary torch operations where `own` is false, and through larynx_b200.kv where it
is true.  Both work on the same buffers, laid out as include/larynx_kv.h says:

  pool    uint8 [layers][pages][kv heads][page / 16][block bytes]: a block is 16 tokens of a head
  block   K codes, then V codes (1024 bytes for every 64 channels), then K and V parameters
          (16 slots of bf16 (step, minimum) for every group of channels)
  table   int32 [slots][max pages], lengths int32 [slots], refs int32 [pages]

A group of 32 or 64 channels of a token is held as codes c = rint((x - m) / s) in 0..15 with
m = min(x) rounded down to bf16 and s = (max(x) - m) / 15 rounded up to bf16; it stands for c s + m.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one live stream of the audio pipeline: a single new frame against 560 cached ones; latency
        dict(name="attend 1x1 over 560, 16 heads", op="attention", n=1, q_min=1, q_max=1, len_min=560, len_max=560,
             kv_heads=16, per_kv=1, dim=64, group=64, page=16, chunk=1, left=-1, dtype="bf16"),
        # a batch of token generators at every age, seven query heads on a kv head, odd lengths
        dict(name="attend 64x1 over 41-2100, 14/2", op="attention", n=64, q_min=1, q_max=1, len_min=41, len_max=2100,
             kv_heads=2, per_kv=7, dim=64, group=32, page=32, chunk=1, left=-1, dtype="bf16"),
        # one very long sequence: the key axis has to be split over the whole GPU
        dict(name="attend 1x1 over 131071, 32/8", op="attention", n=1, q_min=1, q_max=1, len_min=131071,
             len_max=131071, kv_heads=8, per_kv=4, dim=128, group=64, page=64, chunk=1, left=-1, dtype="bf16"),
        # a full serving batch: bound by the bytes of the cache
        dict(name="attend 64x1 over 4099-8191, 32/8", op="attention", n=64, q_min=1, q_max=1, len_min=4099,
             len_max=8191, kv_heads=8, per_kv=4, dim=128, group=64, page=32, chunk=1, left=-1, dtype="fp16"),
        # streaming: 48 streams x 2 guidance rows, a 50-frame chunk and its 6-frame look-ahead after up to 500 frames
        dict(name="attend 96x56 over 56-556, chunk 50", op="attention", n=96, q_min=56, q_max=56, len_min=56,
             len_max=556, kv_heads=16, per_kv=1, dim=64, group=64, page=16, chunk=50, left=-1, dtype="bf16"),
        # prompts taken in whole behind a cached prefix, causal
        dict(name="attend 4x701-1500 over 1500-2100", op="attention", n=4, q_min=701, q_max=1500, len_min=1500,
             len_max=2100, kv_heads=4, per_kv=4, dim=64, group=64, page=64, chunk=1, left=-1, dtype="bf16"),
        # the row that each of 64 generators adds at a step; latency
        dict(name="write 64x1, 2 heads", op="write", n=64, rows_min=1, rows_max=1, start_min=40, start_max=2099,
             kv_heads=2, dim=64, group=32, page=32, dtype="bf16"),
        # the 50 frames that each stream adds at a hop
        dict(name="write 96x50, 16 heads", op="write", n=96, rows_min=50, rows_max=50, start_min=6, start_max=506,
             kv_heads=16, dim=64, group=64, page=16, dtype="bf16"),
        # long prompts, still in 32 bits
        dict(name="write 8x3001-4099, 8 heads, fp32", op="write", n=8, rows_min=3001, rows_max=4099, start_min=0,
             start_max=77, kv_heads=8, dim=128, group=64, page=64, dtype="fp32"),
        # four continuations tried from one prefix: the old ones end, new ones share and grow by a token; latency
        dict(name="pages branch 4 of 300", op="branch", n=4, len_min=297, len_max=303, grow=1, layers=22, kv_heads=16,
             dim=64, group=64, page=16),
        # streams duplicated outright (all layers), as before edits of the prefix itself
        dict(name="pages copy 12 of 1000-1500", op="copy", n=12, len_min=1000, len_max=1500, grow=0, layers=22,
             kv_heads=16, dim=64, group=64, page=64),
        # two generations of streams take turns and the pool is kept dense
        dict(name="pages turnover 2x24 of 500-556", op="turnover", n=24, len_min=500, len_max=556, grow=0, layers=22,
             kv_heads=16, dim=64, group=64, page=16),
    ]


def _between(rng, a, b):
    """A whole number of [a, b], spread over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    dim, group, page = rng.choice([64, 64, 128]), rng.choice([32, 64]), rng.choice([16, 32, 64, 128])
    kind = rng.choice(["attention"] * 5 + ["write"] * 3 + ["branch", "copy", "turnover"])
    base = dict(op=kind, dim=dim, group=group, page=page)
    if kind == "attention":
        few = rng.random() < 0.65
        q_max = rng.choice([1, 1, 1, 2, 5]) if few else _between(rng, 17, 600)
        length = _between(rng, 33, 20000 if few else 2000)
        heads, per = rng.choice([1, 2, 3, 4, 8, 16]), rng.choice([1, 1, 2, 4, 5, 7, 8])
        n = max(1, min(_between(rng, 1, 150), (1 << 28) // (length * heads * dim), (1 << 27) // (length * q_max * heads * per)))
        chunk = rng.choice([0, 1, 1, 1, 25, 50])
        return dict(base, n=n, q_min=max(1, q_max - rng.randrange(0, 1 + q_max // 2)), q_max=q_max,
                    len_min=max(1, int(length * rng.uniform(0.2, 1.0))), len_max=length, kv_heads=heads, per_kv=per,
                    chunk=chunk, left=rng.choice([-1, -1, 0, 100, 777]) if chunk else -1,
                    dtype=rng.choice(["bf16", "bf16", "fp16"]))
    if kind == "write":
        rows, heads = _between(rng, 1, 3000), rng.choice([1, 2, 3, 8, 16])
        n = max(1, min(_between(rng, 1, 200), (1 << 25) // (rows * heads * dim)))
        start = _between(rng, 1, 3000)
        return dict(base, n=n, rows_min=max(1, rows - rng.randrange(0, 1 + rows // 2)), rows_max=rows,
                    start_min=rng.randrange(0, start), start_max=start, kv_heads=heads,
                    dtype=rng.choice(["bf16", "fp16", "fp32"]))
    layers, heads = rng.choice([4, 12, 22, 24]), rng.choice([2, 8, 16])
    per_token = layers * heads * (dim + 8 * (dim // group))
    length = _between(rng, 20, 3000)
    n = max(1, min(_between(rng, 1, 200), (1 << 28) // (per_token * length)))
    return dict(base, n=n, len_min=max(1, int(length * rng.uniform(0.5, 1.0))), len_max=length,
                grow=_between(rng, 1, 60) if kind == "branch" else 0, layers=layers, kv_heads=heads)


def _spread(low, high, n):
    """n whole numbers from low to high."""
    return [low + (high - low) * i // max(1, n - 1) if n > 1 else high for i in range(n)]


def _visible(case):
    """Per entry: (rows, length, visible keys over all rows)."""
    got = []
    for rows, length in zip(_spread(case["q_min"], case["q_max"], case["n"]), _spread(case["len_min"], case["len_max"], case["n"])):
        pairs, chunk, left = 0, case["chunk"], case["left"]
        for p in range(length - rows, length):
            high = min(length, (p // chunk + 1) * chunk) if chunk else length
            low = max(0, p // chunk * chunk - left) if chunk and left >= 0 else 0
            pairs += max(0, high - low)
        got.append((rows, length, pairs))
    return got


def work(case):
    token = case["kv_heads"] * (case["dim"] + 8 * (case["dim"] // case["group"]))  # bytes of a token in the cache
    if case["op"] == "attention":
        heads, seen = case["kv_heads"] * case["per_kv"], _visible(case)
        rows, chunk, left = sum(r for r, _, _ in seen), case["chunk"], case["left"]
        keys = 0
        for r, length, _ in seen:
            first = length - r
            low = max(0, first // chunk * chunk - left) if chunk and left >= 0 else 0
            high = min(length, ((length - 1) // chunk + 1) * chunk) if chunk else length
            keys += max(0, high - low)
        return {"bytes": keys * token + rows * heads * (2 * 2 * case["dim"] + 4),
                "flops": 4.0 * case["dim"] * heads * sum(p for _, _, p in seen)}
    if case["op"] == "write":
        rows, size = sum(_spread(case["rows_min"], case["rows_max"], case["n"])), DTYPES[case["dtype"]].itemsize
        values = rows * case["kv_heads"] * case["dim"] * 2
        return {"bytes": 2 * values * size + 2 * rows * token, "flops": 6.0 * values}
    lens, page, n_pages, slots, width = _page_plan(case)
    tables = 4 * (2 * slots * width + 2 * slots + 2 * n_pages)
    whole = [-(-v // page) for v in lens]
    moved = {"branch": sum(v % page != 0 for v in lens), "copy": sum(whole), "turnover": 2 * sum(whole)}[case["op"]]
    return {"bytes": 2 * moved * page * token * case["layers"] + tables, "flops": 0.0}


# ---------------------------------------------------------------------------
# the block's bytes
# ---------------------------------------------------------------------------
def _block_bytes(dim, group):
    return dim // 64 * 1024 + 128 * (dim // group)


def _code_places(t, dim):
    """Byte offsets in a block of the K and the V codes of tokens `t` (0..15): [..., dim / 2] each.
    K's byte b holds the channels _k_channels gives; V's byte b holds channels 2 b and 2 b + 1."""
    t, b = t[..., None], torch.arange(dim // 2, device=t.device)
    k = b // 32 * 512 + (t % 8 * 4 + b % 16 // 4) * 16 + t // 8 * 8 + b % 32 // 16 * 4 + b % 4
    v = dim // 64 * 512 + b // 32 * 512 + (b % 16 // 2 * 4 + t % 8 // 2) * 16 + t // 8 * 8 + b % 32 // 16 * 4 + t % 2 * 2 + b % 2
    return k, v


def _k_channels(dim, device):
    """The channels in the low and the high half of each byte of a token's K codes: [dim / 2, 2]."""
    b = torch.arange(dim // 2, device=device)[:, None]
    p = b % 4 * 2 + torch.arange(2, device=device)  # place in the 32-bit word
    return b // 32 * 64 + b % 32 // 16 * 32 + b % 16 // 4 * 8 + p % 4 * 2 + p // 4


def _param_places(t, dim, group):
    """Byte offsets in a block of K's and V's parameters of tokens `t`: [..., groups, 4] each."""
    g = torch.arange(dim // group, device=t.device)[:, None]
    at = dim // 64 * 1024 + g * 64 + (t % 8 // 2 * 4 + t // 8 * 2 + t % 2)[..., None, None] * 4 + torch.arange(4, device=t.device)
    return at, at + 64 * (dim // group)


def _quantise(x, group):
    """[..., dim] -> codes uint8 [..., dim], step and minimum (fp32 holding bf16 values) [..., groups]; in 64 bits,
    for a code next to a border is off by a whole step."""
    x = x.unflatten(-1, (-1, group))
    low, high = x.amin(-1).float(), x.amax(-1).double()
    bits = low.view(torch.int32)
    m = (torch.where(bits < 0, bits + 0xFFFF, bits) & -65536).view(torch.float32)
    exact_step = (high - m.double()) / torch.full_like(high, 15.0)
    s = exact_step.float()
    s = torch.where(s.double() < exact_step, torch.nextafter(s, torch.full_like(s, math.inf)), s)
    s = ((s.view(torch.int32) + 0xFFFF) & -65536).view(torch.float32).clamp_min(2.0 ** -126)
    codes = torch.round((x.double() - m[..., None].double()) / s[..., None].double()).clamp(0, 15).to(torch.uint8)
    return codes.flatten(-2), s, m


def _store(pool, base, t, k, v, group):
    """Quantises rows k, v [..., heads, dim] into the flat pool: `base` [..., heads] byte offsets of their blocks, `t` [...] tokens in the block."""
    dim = k.shape[-1]
    kc, ks, km = _quantise(k, group)
    vc, vs, vm = _quantise(v, group)
    at_k, at_v = _code_places(t, dim)
    par_k, par_v = _param_places(t, dim, group)
    pair = kc[..., _k_channels(dim, k.device)]
    pool[base[..., None] + at_k[..., None, :]] = pair[..., 0] | pair[..., 1] << 4
    pool[base[..., None] + at_v[..., None, :]] = vc[..., 0::2] | vc[..., 1::2] << 4
    pool[base[..., None, None] + par_k[..., None, :, :]] = torch.stack((ks, km), -1).to(torch.bfloat16).view(torch.uint8)
    pool[base[..., None, None] + par_v[..., None, :, :]] = torch.stack((vs, vm), -1).to(torch.bfloat16).view(torch.uint8)


def _load(pool, base, t, dim, group):
    """The values of rows in the cache: fp32 k, v [..., heads, dim]."""
    at_k, at_v = _code_places(t, dim)
    par_k, par_v = _param_places(t, dim, group)
    order = torch.argsort(_k_channels(dim, pool.device).flatten())
    out = []
    for at, par, turn in ((at_k, par_k, order), (at_v, par_v, None)):
        byte = pool[base[..., None] + at[..., None, :]]
        code = torch.stack((byte & 15, byte >> 4), -1).flatten(-2)
        code = (code if turn is None else code[..., turn]).float().unflatten(-1, (-1, group))
        p = pool[base[..., None, None] + par[..., None, :, :]].view(torch.bfloat16).float()
        out.append((code * p[..., 0:1] + p[..., 1:2]).flatten(-2))
    return out


def _unpack(blocks, dim, group):
    """Whole blocks uint8 [..., heads, blocks, bytes] -> fp32 k, v [..., heads, blocks * 16, dim]."""
    halves, groups, lead = dim // 64, dim // group, blocks.shape[:-1]
    codes = blocks[..., : halves * 1024].reshape(*lead, 2, halves, 8, 4, 2, 2, 4)
    codes = torch.stack((codes & 15, codes >> 4), -1).reshape(*lead, 2, halves, 8, 4, 2, 2, 2, 4)  # K/V, half, n, j, kh, w, po, r
    par = blocks[..., halves * 1024:].reshape(*lead, 2, groups, 4, 2, 2, 4).view(torch.bfloat16).float()  # K/V, group, j, kh, par, (s, m)
    par = par.reshape(*lead, 2, groups, 4, 2, 2, 2)
    z, i = len(lead), list(range(len(lead)))
    k, v, out = codes.select(z, 0), codes.select(z, 1), []
    k = k.permute(*i, z + 3, z + 1, z, z + 4, z + 2, z + 6, z + 5)  # kh n | half w j r po
    v = v.permute(*i, z + 3, z + 2, z + 5, z, z + 4, z + 1, z + 6)  # kh j par | half w n i
    for kv, c in enumerate((k, v)):
        p = par.select(z, kv).permute(*i, z + 2, z + 1, z + 3, z, z + 4).reshape(*lead, 16, groups, 2)  # kh j par | group (s, m)
        c = c.reshape(*lead, 16, groups, group).float()
        out.append((c * p[..., 0:1] + p[..., 1:2]).reshape(*lead[:-1], lead[-1] * 16, dim))
    return out


# ---------------------------------------------------------------------------
# what a program has in hand
# ---------------------------------------------------------------------------
def _page_plan(case):
    """Lengths, page, pages of the pool, slots and table width of a case on pages."""
    lens, page = _spread(case["len_min"], case["len_max"], case["n"]), case["page"]
    whole = sum(-(-v // page) for v in lens)
    if case["op"] == "branch":
        extra = case["n"] * (-(-case["grow"] // page) + 1)
    else:
        extra = whole
    n_pages = whole + extra + 7
    return lens, page, n_pages, 2 * case["n"] + 1, -(-(max(lens) + case["grow"]) // page) + 1


def _rows(t, heads, values, dtype, seed_gen, offset):
    """Keys or values as a model makes them: keys have channels with a mean and channels that are larger."""
    x = torch.randn(t, heads, values, device="cuda", generator=seed_gen)
    if offset:
        size = torch.rand(heads, values, device="cuda", generator=seed_gen).pow(4) * 3 + 0.5
        x = x * size + torch.randn(heads, values, device="cuda", generator=seed_gen) * 0.5
    return x.to(dtype)


def prepare(case, seed):
    gen, rng = torch.Generator("cuda").manual_seed(seed), random.Random(seed)
    int32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    dim, group, page, heads = case["dim"], case["group"], case["page"], case["kv_heads"]
    s = dict(case=case, dim=dim, group=group, page=page, kv_heads=heads)
    if case["op"] in ("attention", "write"):
        n, layers = case["n"], 2
        if case["op"] == "attention":
            lens, rows = _spread(case["len_min"], case["len_max"], n), _spread(case["q_min"], case["q_max"], n)
            starts = [a - b for a, b in zip(lens, rows)]
        else:
            starts, rows = _spread(case["start_min"], case["start_max"], n), _spread(case["rows_min"], case["rows_max"], n)
            lens = [a + b for a, b in zip(starts, rows)]
        whole = [-(-v // page) for v in lens]
        n_pages, width = sum(whole) + 3, max(whole) + 1
        ids = list(range(n_pages))
        rng.shuffle(ids)
        table = [[-1] * width for _ in range(n)]
        for i, w in enumerate(whole):
            table[i][:w] = [ids.pop() for _ in range(w)]
        refs = torch.zeros(n_pages, dtype=torch.int32)
        refs[[p for t in table for p in t if p >= 0]] = 1
        s.update(layers=layers, layer=1, n=n, n_pages=n_pages, n_seq=n, width=width, table=int32(table), lengths=int32(lens),
                 refs=refs.cuda(), max_rows=max(rows), max_len=max(lens), total=sum(rows))
        s["row0"] = int32([sum(rows[:i]) for i in range(n + 1)])
        s["start"], s["counts"] = int32(starts), int32(rows)
        entry = torch.repeat_interleave(torch.arange(n), torch.tensor(rows)).cuda()
        row = torch.cat([torch.arange(r) for r in rows]).cuda()
        s["entry"], s["row"] = entry, row
        size = heads * (page // 16) * _block_bytes(dim, group)
        s["pool"] = torch.zeros(layers * n_pages * size, dtype=torch.uint8, device="cuda")
        if case["op"] == "attention":
            for i, length in enumerate(lens):  # the cache as earlier steps filled it
                pos = torch.arange(length, device="cuda")
                _store(s["pool"], _bases(s, torch.full_like(pos, i), pos), pos % 16, _rows(length, heads, dim, torch.float32, gen, True),
                       _rows(length, heads, dim, torch.float32, gen, False), group)
            dtype = DTYPES[case["dtype"]]
            s["q"] = torch.randn(s["total"], heads * case["per_kv"], dim, device="cuda", generator=gen).to(dtype)
            s["out"] = torch.empty_like(s["q"])
            s["lse"] = torch.empty(s["total"], heads * case["per_kv"], device="cuda")
        else:
            dtype = DTYPES[case["dtype"]]
            s["k"], s["v"] = (_rows(s["total"], heads, dim, dtype, gen, o) for o in (True, False))
            s["k_out"], s["v_out"] = torch.empty_like(s["k"]), torch.empty_like(s["v"])
        return s
    lens, page, n_pages, slots, width = _page_plan(case)
    n = case["n"]
    whole, ids = [-(-v // page) for v in lens], list(range(n_pages))
    if case["op"] != "turnover":
        rng.shuffle(ids)
    table, lengths = [[-1] * width for _ in range(slots)], [0] * slots
    refs = torch.zeros(n_pages, dtype=torch.int32)
    for g in range(2 if case["op"] == "turnover" else 1):
        for i in range(n):
            pages, ids = ids[: whole[i]], ids[whole[i]:]
            table[g * n + i][: whole[i]], lengths[g * n + i] = pages, lens[i]
            refs[pages] = 1
    order = list(range(n))
    rng.shuffle(order)
    size = heads * (page // 16) * _block_bytes(dim, group)
    s.update(layers=case["layers"], n=n, n_pages=n_pages, n_seq=slots, width=width, table=int32(table), lengths=int32(lengths),
             refs=refs.cuda(), used=torch.zeros(1, dtype=torch.int32, device="cuda"), size=size, most=sum(whole),
             pool=torch.randint(0, 256, (case["layers"] * n_pages * size,), dtype=torch.uint8, device="cuda", generator=gen))
    s["src"], s["dst"] = int32(order), int32([n + i for i in order])
    s["zeros"], s["grow"] = int32([0] * n), int32([max(1, case["grow"])] * n)
    s["start"], s["whole"] = int32([0] * n), int32([lens[i] for i in order])
    return s


def _bases(s, slot, pos):
    """Byte offsets in the flat pool of the blocks of position `pos` of `slot`, for every head: [..., heads]."""
    block = _block_bytes(s["dim"], s["group"])
    page = s["table"][slot, pos // s["page"]].long()
    head = torch.arange(s["kv_heads"], device=pos.device)
    at = ((s["layer"] * s["n_pages"] + page)[..., None] * s["kv_heads"] + head) * (s["page"] // 16)
    return (at + (pos % s["page"] // 16)[..., None]) * block


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _attention(s):
    case, dim, heads, page = s["case"], s["dim"], s["kv_heads"], s["page"]
    n, per, wide = s["n"], case["per_kv"], s["max_rows"]
    used = -(-s["max_len"] // page)
    pool = s["pool"].view(s["layers"], s["n_pages"], heads, page // 16, -1)[s["layer"]]
    blocks = pool[s["table"][:, :used].long().clamp_min(0)]  # [n, pages, heads, blocks, bytes]
    k, v = _unpack(blocks.transpose(1, 2).flatten(2, 3), dim, s["group"])  # [n, heads, keys, dim]
    keys = torch.arange(used * page, device="cuda")
    v = v * (keys < s["lengths"][:, None])[:, None, :, None]  # nothing behind the end counts
    q = torch.zeros(n, wide, heads * per, dim, device="cuda")
    q[s["entry"], s["row"]] = s["q"].float()
    q = q.view(n, wide, heads, per, dim).permute(0, 2, 1, 3, 4).flatten(2, 3)  # [n, heads, rows * per, dim]
    pos = s["start"][:, None] + torch.arange(wide, device="cuda")
    length = s["lengths"][:, None]
    chunk, left = case["chunk"], case["left"]
    high = torch.minimum(length, (torch.div(pos, chunk, rounding_mode="floor") + 1) * chunk) if chunk else length.expand_as(pos)
    low = (torch.div(pos, chunk, rounding_mode="floor") * chunk - left).clamp_min(0) if chunk and left >= 0 else torch.zeros_like(pos)
    seen = ((keys >= low[..., None]) & (keys < high[..., None])).repeat_interleave(per, 1)[:, None]  # [n, 1, rows * per, keys]
    score = torch.where(seen, torch.matmul(q, k.transpose(-1, -2)) * dim ** -0.5, float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isinf(top), 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    lse = top + torch.log(total)
    back = lambda x: x.unflatten(2, (wide, per)).permute(0, 2, 1, 3, 4).flatten(2, 3)[s["entry"], s["row"]]  # noqa: E731
    return back(out).to(s["q"].dtype), back(lse)[..., 0]


def _write(s):
    slot, pos = s["entry"], s["start"][s["entry"]] + s["row"]
    base = _bases(s, slot, pos)
    _store(s["pool"], base, pos % 16, s["k"], s["v"], s["group"])
    k, v = _load(s["pool"], base, pos % 16, s["dim"], s["group"])
    return k.to(s["k"].dtype), v.to(s["v"].dtype)


def _pages_of(s, length):
    return torch.div(length + s["page"] - 1, s["page"], rounding_mode="floor")


def _ranked(mask):
    """The indices where `mask` holds, in ascending order, behind them anything."""
    n = mask.numel()
    at = torch.where(mask, torch.cumsum(mask, 0) - 1, n)
    return torch.zeros(n + 1, dtype=torch.int64, device=mask.device).scatter_(0, at, torch.arange(n, device=mask.device))


def _count(s, pages, held, by):
    """refs of the pages where `held` holds, up or down."""
    s["refs"].index_add_(0, torch.where(held, pages, 0).flatten(), (held * by).to(torch.int32).flatten())


def _free(s, slots, keep):
    slots, column = slots.long(), torch.arange(s["width"], device="cuda")
    old, length = s["table"][slots], s["lengths"][slots]
    new = torch.minimum(length, keep)
    gone = (column >= _pages_of(s, new)[:, None]) & (column < _pages_of(s, length)[:, None])
    _count(s, old, gone, -1)
    s["table"][slots] = torch.where(gone, -1, old)
    s["lengths"][slots] = new


def _fork(s, src, dst):
    src, dst = src.long(), dst.long()
    rows = s["table"][src]
    _count(s, rows, rows >= 0, 1)
    s["table"][dst] = rows
    s["lengths"][dst] = s["lengths"][src]


def _move(s, src, dst):
    pool = s["pool"].view(s["layers"], s["n_pages"], s["size"])
    pool[:, dst] = pool[:, src]


def _extend(s, slots, counts):
    slots, column = slots.long(), torch.arange(s["width"], device="cuda")
    rows, length = s["table"][slots], s["lengths"][slots]
    old, new = _pages_of(s, length), _pages_of(s, length + counts)
    tail = torch.gather(rows, 1, (old - 1).clamp_min(0).long()[:, None])[:, 0].clamp_min(0).long()
    shared = (length % s["page"] != 0) & (s["refs"][tail] > 1) & (counts > 0)
    need = new - old + shared.int()
    before = torch.cumsum(need, 0) - need
    free = _ranked(s["refs"] == 0)
    at = before[:, None] + column - old[:, None] + shared[:, None]
    fresh = ((column >= old[:, None]) & (column < new[:, None])) | (shared[:, None] & (column == old[:, None] - 1))
    got = free[torch.where(fresh, at, 0).long()].int()
    copy = torch.where(shared, free[torch.where(shared, before, 0).long()], tail)
    if s["case"]["op"] == "branch":  # elsewhere no page is shared
        _move(s, tail, copy)
    _count(s, tail, shared, -1)
    _count(s, got, fresh, 1)
    s["table"][slots] = torch.where(fresh, got, rows)
    s["lengths"][slots] = length + counts
    s["start"].copy_(length)


def _copy(s, src, dst):
    src, dst, column = src.long(), dst.long(), torch.arange(s["width"], device="cuda")
    rows, length = s["table"][src], s["lengths"][src]
    need = _pages_of(s, length)
    before, held = torch.cumsum(need, 0) - need, column < need[:, None]
    at = torch.minimum(column, need[:, None] - 1)  # past the last page: the last one again
    got = _ranked(s["refs"] == 0)[(before[:, None] + at).long()]
    _move(s, torch.gather(rows, 1, at.long()).long().flatten(), got.flatten())
    _count(s, got, held, 1)
    s["table"][dst] = torch.where(held, got.int(), -1)
    s["lengths"][dst] = length


def _compact(s):
    held, page = s["refs"] > 0, torch.arange(s["n_pages"], device="cuda")
    used = held.sum()
    hole, mover = ~held & (page < used), held & (page >= used)
    moves, holes, movers = hole.sum(), _ranked(hole), _ranked(mover)
    k = torch.minimum(torch.arange(s["most"], device="cuda"), (moves - 1).clamp_min(0))  # past the last move: the last one again
    to, come = torch.where(moves > 0, holes[k], 0), torch.where(moves > 0, movers[k], 0)
    _move(s, come, to)
    place = torch.arange(s["n_pages"], device="cuda").scatter_(0, come, to)
    s["refs"].copy_(torch.where(page < used, 1, 0) * s["refs"].scatter(0, to, s["refs"][come]))
    s["table"].copy_(torch.where(s["table"] >= 0, place[s["table"].clamp_min(0).long()].int(), -1))
    s["used"].copy_(used)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _cache(s):
    """The framework's cache on the state's buffers; a program keeps it."""
    if "cache" not in s:
        from larynx_b200.kv import KVCache, scratch_ints

        s["scratch"] = torch.empty(scratch_ints(s["n_pages"], s["n_seq"], s["width"]), dtype=torch.int32, device="cuda")
        s["error"] = torch.zeros(1, dtype=torch.int32, device="cuda")
        s["cache"] = KVCache(s["layers"], s["n_pages"], s["n_seq"], s["width"], s["kv_heads"], s["dim"], s["group"], s["page"],
                             s["pool"].data_ptr(), s["table"].data_ptr(), s["lengths"].data_ptr(), s["refs"].data_ptr(),
                             s["scratch"].data_ptr(), s["error"].data_ptr(), device=s["pool"].device.index)
        if "row0" in s:
            s["rows"] = s["cache"].rows(s["n"], s["total"], s["max_rows"], row0=s["row0"].data_ptr(), start=s["start"].data_ptr())
    return s["cache"]


def run(state):
    s, case = state, state["case"]
    op = case["op"]
    if own:
        cache, stream = _cache(s), torch.cuda.current_stream().cuda_stream
        if op == "attention":
            cache.attention(s["layer"], s["rows"], s["kv_heads"] * case["per_kv"], case["dtype"], s["q"].data_ptr(), s["out"].data_ptr(),
                            lse=s["lse"].data_ptr(), scale=s["dim"] ** -0.5, chunk=case["chunk"], left=case["left"], max_len=s["max_len"],
                            stream=stream)
            return s["out"], s["lse"]
        if op == "write":
            cache.write(s["layer"], s["rows"], case["dtype"], s["k"].data_ptr(), s["v"].data_ptr(), stream=stream)
            cache.read(s["layer"], s["rows"], case["dtype"], s["k_out"].data_ptr(), s["v_out"].data_ptr(), stream=stream)
            return s["k_out"], s["v_out"]
        n, src, dst, zeros = s["n"], s["src"].data_ptr(), s["dst"].data_ptr(), s["zeros"].data_ptr()
        if op == "branch":
            cache.free(n, dst, zeros, stream=stream)
            cache.fork(n, src, dst, stream=stream)
            cache.extend(n, dst, s["grow"].data_ptr(), s["start"].data_ptr(), stream=stream)
        elif op == "copy":
            cache.free(n, dst, zeros, stream=stream)
            cache.copy(n, src, dst, stream=stream)
        else:
            for slots in (src, dst):
                cache.free(n, slots, zeros, stream=stream)
                cache.compact(s["used"].data_ptr(), stream=stream)
                cache.extend(n, slots, s["whole"].data_ptr(), s["start"].data_ptr(), stream=stream)
    elif op == "attention":
        return _attention(s)
    elif op == "write":
        return _write(s)
    elif op == "branch":
        _free(s, s["dst"], s["zeros"])
        _fork(s, s["src"], s["dst"])
        _extend(s, s["dst"], s["grow"])
    elif op == "copy":
        _free(s, s["dst"], s["zeros"])
        _copy(s, s["src"], s["dst"])
    else:
        for slots in (s["src"], s["dst"]):
            _free(s, slots, s["zeros"])
            _compact(s)
            _extend(s, slots, s["whole"])
    return {"pool": s["pool"], "table": s["table"], "lengths": s["lengths"], "refs": s["refs"], "start": s["start"], "used": s["used"]}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------
def _held(s, slot, length):
    """Keys and values of a slot in fp64 [heads, length, dim], each nibble read where the format puts it."""
    dim, group, heads, page = s["dim"], s["group"], s["kv_heads"], s["page"]
    block = dim // 64 * 1024 + 128 * (dim // group)
    pos = torch.arange(length, device="cuda")
    ids = s["table"][slot].long()[pos // page]
    head, d = torch.arange(heads, device="cuda")[:, None, None], torch.arange(dim, device="cuda")
    at = ((((s["layer"] * s["n_pages"] + ids)[None, :, None] * heads + head) * page + (pos % page)[None, :, None]) // 16) * block
    t = (pos % 16)[None, :, None]
    key, half, pair, odd = t % 8, t // 8, t % 8 // 2, t % 2
    lane_k, e = 4 * key + d % 32 // 8, d % 8
    byte_k = 512 * (d // 64) + 16 * lane_k + 8 * half + 4 * (d % 64 // 32) + 2 * (e % 2) + e // 4
    shift_k = 4 * (e // 2 % 2)
    lane_v, e = 4 * (d % 32 // 4) + pair, d % 4
    byte_v = 512 * (dim // 64) + 512 * (d // 64) + 16 * lane_v + 8 * half + 4 * (d % 64 // 32) + 2 * odd + e // 2
    shift_v = 4 * (e % 2)
    out = []
    for kv, (byte, shift) in enumerate(((byte_k, shift_k), (byte_v, shift_v))):
        code = (s["pool"][at + byte] >> shift.to(torch.uint8) & 15).double()
        where = at + 1024 * (dim // 64) + 64 * (kv * (dim // group) + d // group) + 4 * (4 * pair + 2 * half + odd)
        word = lambda o: torch.ldexp(s["pool"][where + o + 1].int() * 256 + s["pool"][where + o].int(), torch.tensor(16, device="cuda")).to(torch.int64)  # noqa: E731
        step, low = (word(o).to(torch.int32).view(torch.float32).double() for o in (0, 2))
        out.append(code * step + low)
    return out


def _bf16_toward(x, up):
    """fp64 -> the next bf16 value up or down (no overflow, no subnormals)."""
    part, power = torch.frexp(x)
    part = part * 256
    return torch.ldexp(torch.ceil(part) if up else torch.floor(part), power - 8)


def exact(case, seed):
    if case["op"] not in ("attention", "write"):
        return None
    s = prepare(case, seed)
    if case["op"] == "write":
        out = []
        for x in (s["k"], s["v"]):
            x = x.double().reshape(s["total"], s["kv_heads"], -1, s["group"])
            m = _bf16_toward(x.min(-1, keepdim=True).values, False)
            step = _bf16_toward((x.max(-1, keepdim=True).values - m) / 15, True).clamp_min(2.0 ** -126)
            out.append((torch.round((x - m) / step).clamp(0, 15) * step + m).flatten(-2))
        return tuple(out)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["lse"].shape, -math.inf, dtype=torch.float64, device="cuda")
    first = 0
    for i, (rows, length, _) in enumerate(_visible(case)):
        k, v = _held(s, i, length)
        for h in range(s["kv_heads"]):
            mine = slice(h * case["per_kv"], (h + 1) * case["per_kv"])
            pos = torch.arange(length - rows, length, device="cuda")
            score = torch.einsum("rgd,kd->rgk", s["q"][first: first + rows, mine].double(), k[h]) / math.sqrt(s["dim"])
            j, chunk = torch.arange(length, device="cuda"), case["chunk"]
            if chunk:
                own_chunk = torch.floor(pos / chunk)
                hidden = j >= ((own_chunk + 1) * chunk)[:, None]
                if case["left"] >= 0:
                    hidden |= j < (own_chunk * chunk - case["left"])[:, None]
                score = score.masked_fill(hidden[:, None, :], -math.inf)
            lse[first: first + rows, mine] = torch.logsumexp(score, -1)
            some = torch.isfinite(lse[first: first + rows, mine])[..., None]
            w = torch.where(some, torch.exp(score - lse[first: first + rows, mine][..., None]), 0.0)
            out[first: first + rows, mine] = torch.einsum("rgk,kd->rgd", w, v[h])
        first += rows
    return out, lse
