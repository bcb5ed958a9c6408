"""CPU checks of the paged 4-bit cache's boundary: the header's entry points
are exported and bound, sizes follow the documented layout, every refusal of
the arguments is made before any device work, and the oracle's quantiser is
right on its own terms."""

import ctypes
import os
import re

import numpy as np
import pytest

from oracle import kv_oracle as ko

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20  # a pointer that is never followed


def _cache(**kw):
    from larynx_b200 import kv
    a = dict(device=0, n_layers=2, n_pages=10, n_seq=3, max_pages=4, kv_heads=2, head_dim=64, group=64, page=16,
             pool=P, table=P, lengths=P, refs=P, scratch=P, error=P)
    a.update(kw)
    return kv.LxKvCache(**a)


def _rows(**kw):
    from larynx_b200 import kv
    a = dict(n=2, total=6, max_rows=3, seqs=None, row0=None, start=None)
    a.update(kw)
    return kv.LxKvRows(**a)


def _lib():
    from larynx_b200 import flow, kv
    return kv._declare(flow.load_library())


def test_header_and_binding_name_the_same_entry_points():
    from larynx_b200.kv import KV_EXPORTS
    src = open(os.path.join(REPO, "include", "larynx_kv.h")).read()
    declared = set(re.findall(r"^(?:int|size_t)\s+(lx_\w+)\s*\(", src, re.M))
    assert declared == set(KV_EXPORTS)
    lib = _lib()
    for name in declared:
        assert ctypes.cast(getattr(lib, name), ctypes.c_void_p).value


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group", [32, 64])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_sizes(dim, group, page):
    from larynx_b200 import kv
    token = dim + 8 * (dim // group)  # bytes of a token and head: 2 x 4 bits a channel, 2 x 4 bytes a group
    assert kv.pool_bytes(3, 7, 5, dim, group, page) == 3 * 7 * 5 * page * token
    assert kv.scratch_ints(7, 2, 9) > 3 * 7


@pytest.mark.parametrize("bad", [dict(head_dim=80), dict(head_dim=0), dict(group=16), dict(page=24), dict(page=0),
                                 dict(kv_heads=0), dict(n_pages=0), dict(n_layers=0), dict(n_seq=0),
                                 dict(max_pages=0), dict(max_pages=1 << 27)])
def test_geometry_refused(bad):
    lib = _lib()
    c = _cache(**bad)
    assert lib.lx_kv_pool_bytes(ctypes.byref(c)) == 0
    assert lib.lx_kv_scratch_ints(ctypes.byref(c)) == 0
    assert lib.lx_kv_reset(ctypes.byref(c), None) == 1
    from larynx_b200 import kv
    with pytest.raises(kv.KVError):
        kv.KVCache(c.n_layers, c.n_pages, c.n_seq, c.max_pages, c.kv_heads, c.head_dim, c.group, c.page, P, P, P, P, P, P)


@pytest.mark.parametrize("bad", [dict(pool=None), dict(pool=P + 8), dict(table=None), dict(lengths=None),
                                 dict(refs=None), dict(scratch=None), dict(error=None), dict(table=P + 2),
                                 dict(device=-1)])
def test_buffers_refused(bad):
    lib = _lib()
    c, r = _cache(**bad), _rows()
    ref, rows = ctypes.byref(c), ctypes.byref(r)
    bits = ctypes.c_int32()
    assert lib.lx_kv_reset(ref, None) == 1
    assert lib.lx_kv_status(ref, ctypes.byref(bits), None) == 1
    assert lib.lx_kv_extend(ref, 1, P, P, P, None) == 1
    assert lib.lx_kv_fork(ref, 1, P, P, None) == 1
    assert lib.lx_kv_copy(ref, 1, P, P, None) == 1
    assert lib.lx_kv_free(ref, 1, P, P, None) == 1
    assert lib.lx_kv_compact(ref, P, None) == 1
    assert lib.lx_kv_write(ref, 0, rows, 0, P, 128, 64, P, 128, 64, None) == 1
    assert lib.lx_kv_read(ref, 0, rows, 0, P, 128, 64, P, 128, 64, None) == 1
    assert lib.lx_kv_attention(ref, 0, rows, 2, 0, P, 128, 64, P, 128, 64, None, 0.1, 1, -1, 0, None) == 1


def test_batches_refused():
    lib, c = _lib(), _cache()
    ref = ctypes.byref(c)
    for n, a, b in ((0, P, P), (-1, P, P), (4097, P, P), (1, None, P), (1, P, None), (1, P + 1, P)):
        assert lib.lx_kv_extend(ref, n, a, b, P, None) == 1
        assert lib.lx_kv_fork(ref, n, a, b, None) == 1
        assert lib.lx_kv_copy(ref, n, a, b, None) == 1
        assert lib.lx_kv_free(ref, n, a, b, None) == 1
    assert lib.lx_kv_extend(ref, 1, P, P, None, None) == 1
    assert lib.lx_kv_compact(ref, None, None) == 1
    assert lib.lx_kv_reset(None, None) == 1


@pytest.mark.parametrize("bad", [dict(n=0), dict(n=-3), dict(total=-1), dict(max_rows=-1), dict(total=5),
                                 dict(total=1 << 30, max_rows=1 << 29)])
def test_rows_refused(bad):
    lib, c, r = _lib(), _cache(), _rows(**bad)
    ref, rows = ctypes.byref(c), ctypes.byref(r)
    assert lib.lx_kv_write(ref, 0, rows, 0, P, 128, 64, P, 128, 64, None) == 1
    assert lib.lx_kv_read(ref, 0, rows, 0, P, 128, 64, P, 128, 64, None) == 1
    assert lib.lx_kv_attention(ref, 0, rows, 2, 0, P, 128, 64, P, 128, 64, None, 0.1, 1, -1, 0, None) == 1


@pytest.mark.parametrize("bad", [dict(seqs=P + 2), dict(row0=P + 1), dict(start=P + 3)])
def test_unaligned_rows_refused(bad):
    lib, c, r = _lib(), _cache(), _rows(**bad)
    ref, rows = ctypes.byref(c), ctypes.byref(r)
    assert lib.lx_kv_write(ref, 0, rows, 0, P, 128, 64, P, 128, 64, None) == 1
    assert lib.lx_kv_read(ref, 0, rows, 0, P, 128, 64, P, 128, 64, None) == 1
    assert lib.lx_kv_attention(ref, 0, rows, 2, 0, P, 128, 64, P, 128, 64, None, 0.1, 1, -1, 0, None) == 1


def test_row_calls_refused():
    lib, c, r = _lib(), _cache(), _rows()
    ref, rows = ctypes.byref(c), ctypes.byref(r)
    for f in (lib.lx_kv_write, lib.lx_kv_read):
        for layer, dtype, k, v in ((-1, 0, P, P), (2, 0, P, P), (0, 3, P, P), (0, -1, P, P), (0, 0, None, P),
                                   (0, 0, P, None), (0, 0, P + 1, P), (0, 2, P, P + 2)):
            assert f(ref, layer, rows, dtype, k, 128, 64, v, 128, 64, None) == 1

    def att(layer=0, heads=4, dtype=0, q=P, out=P, lse=P, scale=0.1, chunk=1, left=-1, max_len=0):
        return lib.lx_kv_attention(ref, layer, rows, heads, dtype, q, 256, 64, out, 256, 64, lse, scale, chunk, left,
                                   max_len, None)

    for bad in (dict(layer=2), dict(layer=-1), dict(heads=3), dict(heads=0), dict(dtype=2), dict(q=None),
                dict(out=None), dict(q=P + 1), dict(lse=P + 2), dict(scale=float("nan")), dict(scale=float("inf")),
                dict(chunk=-1), dict(chunk=0, left=0), dict(max_len=-1)):
        assert att(**bad) == 1, bad
    # no row: nothing to do, and nothing is enqueued (there is no GPU to enqueue on here)
    none = _rows(n=2, total=0, max_rows=0)
    assert lib.lx_kv_write(ref, 0, ctypes.byref(none), 0, P, 128, 64, P, 128, 64, None) == 0
    assert lib.lx_kv_attention(ref, 0, ctypes.byref(none), 2, 0, P, 128, 64, P, 128, 64, None, 0.1, 1, -1, 0, None) == 0


def test_oracle_quantiser():
    """Every value is within half a step of what it is held as, the ends are
    reached, and a value halfway between two codes goes to the even one."""
    rng = np.random.default_rng(3)
    for scale in (1.0, 1e-30, 1e30, 2.0 ** -130):
        x = (rng.standard_normal(32) * scale).astype(np.float32)
        codes, s, m = ko.quantise_group(x)
        held = codes * np.float64(s) + np.float64(m)
        assert np.abs(held - x.astype(np.float64)).max() <= 0.5 * float(s)
        assert m <= x.min() and float(m) + 15 * float(s) >= x.max()
    codes, s, m = ko.quantise_group(np.array([0, 15, 0.5, 1.5, 2.5, 14.5], np.float32))
    assert (s, m) == (1, 0) and codes.tolist() == [0, 15, 0, 2, 2, 14]
    assert ko.quantise_group(np.full(32, 3.0, np.float32))[0].max() == 0
    assert ko.quantise_group(np.array([1, np.inf], np.float32))[0] is None
    assert ko.quantise_group(np.array([-3e38, 3e38], np.float32))[0] is None


def test_oracle_quantiser_in_bulk_is_the_exact_one():
    rng = np.random.default_rng(4)
    x = rng.standard_normal((300, 32)).astype(np.float32)
    x[100:200] = ((x[100:200].view(np.uint32) >> 16) << 16).view(np.float32)  # bf16: ties
    x[200:220] *= np.exp(rng.uniform(-30, 30, (20, 32))).astype(np.float32)
    x[220] = 1.5
    x[221, 3] = np.nan
    got, steps = ko.quantise(x, 32), ko.steps(x, 32)
    for i, row in enumerate(x):
        codes, s, m = ko.quantise_group(row)
        want = np.full(32, np.nan, np.float32) if codes is None else (codes * float(s) + float(m)).astype(np.float32)
        assert np.array_equal(got[i], want, equal_nan=True) and np.array_equal(steps[i, 0], s, equal_nan=True)
