"""Python host side of the paged key/value cache held in 4 bits: a ctypes
binding of the C ABI (include/larynx_kv.h) over device pointers, beside
``flow.op_attention``, which takes dense keys and values.

``KVCache`` describes a cache on the caller's device buffers and calls the
operators on it: ``extend`` reserves pages for new tokens, ``write`` quantises
rows into them, ``read`` returns their values, ``attention`` attends to them,
``fork``, ``copy``, ``free`` and ``compact`` handle the pages.  Every call but
``status`` is asynchronous on ``stream``.  Shares liblarynx_flow.so with the
Flow decoder; there is no CPU fallback.
"""

from __future__ import annotations

import ctypes

from .flow import ERRORS, LX_OK, load_library

KV_EXPORTS = ("lx_kv_pool_bytes", "lx_kv_scratch_ints", "lx_kv_reset", "lx_kv_status", "lx_kv_extend", "lx_kv_write",
              "lx_kv_read", "lx_kv_attention", "lx_kv_fork", "lx_kv_copy", "lx_kv_free", "lx_kv_compact")

DTYPES = {"bf16": 0, "fp16": 1, "fp32": 2}

FULL, SLOT, WIDTH, PAGE, ROWS, STUCK = 1, 2, 4, 8, 16, 32  # bits of the error word
REFUSED = -2 ** 31  # start of an entry that extend did not serve


class KVError(RuntimeError):
    pass


class LxKvCache(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_int32) for n in ("device", "n_layers", "n_pages", "n_seq", "max_pages", "kv_heads",
                                               "head_dim", "group", "page")] +
                [(n, ctypes.c_void_p) for n in ("pool", "table", "lengths", "refs", "scratch", "error")])


class LxKvRows(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_int32) for n in ("n", "total", "max_rows")] +
                [(n, ctypes.c_void_p) for n in ("seqs", "row0", "start")])


def _declare(lib):
    if getattr(lib, "_kv_declared", False):
        return lib
    vp, i32, i64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64
    cache, rows = ctypes.POINTER(LxKvCache), ctypes.POINTER(LxKvRows)
    for name in ("lx_kv_pool_bytes", "lx_kv_scratch_ints"):
        getattr(lib, name).argtypes = [cache]
        getattr(lib, name).restype = ctypes.c_size_t
    lib.lx_kv_reset.argtypes = [cache, vp]
    lib.lx_kv_status.argtypes = [cache, ctypes.POINTER(i32), vp]
    lib.lx_kv_extend.argtypes = [cache, i32, vp, vp, vp, vp]
    for name in ("lx_kv_write", "lx_kv_read"):
        getattr(lib, name).argtypes = [cache, i32, rows, i32, vp, i64, i64, vp, i64, i64, vp]
    lib.lx_kv_attention.argtypes = [cache, i32, rows, i32, i32, vp, i64, i64, vp, i64, i64, vp, ctypes.c_float, i32,
                                    i32, i32, vp]
    for name in ("lx_kv_fork", "lx_kv_copy", "lx_kv_free"):
        getattr(lib, name).argtypes = [cache, i32, vp, vp, vp]
    lib.lx_kv_compact.argtypes = [cache, vp, vp]
    for name in KV_EXPORTS[2:]:
        getattr(lib, name).restype = ctypes.c_int
    lib._kv_declared = True
    return lib


def pool_bytes(n_layers: int, n_pages: int, kv_heads: int, head_dim: int, group: int, page: int) -> int:
    """Bytes of the pool of a cache of this geometry (0 when it is not valid)."""
    c = LxKvCache(0, n_layers, n_pages, 1, 1, kv_heads, head_dim, group, page)
    return int(_declare(load_library()).lx_kv_pool_bytes(ctypes.byref(c)))


def scratch_ints(n_pages: int, n_seq: int, max_pages: int) -> int:
    """32-bit words of scratch that a cache needs (0 when the sizes are not valid)."""
    c = LxKvCache(0, 1, n_pages, n_seq, max_pages, 1, 64, 64, 16)
    return int(_declare(load_library()).lx_kv_scratch_ints(ctypes.byref(c)))


class KVCache:
    """A cache on the caller's device buffers (pointers; include/larynx_kv.h
    has their layouts).  The buffers have to outlive it."""

    def __init__(self, n_layers: int, n_pages: int, n_seq: int, max_pages: int, kv_heads: int, head_dim: int,
                 group: int, page: int, pool_ptr: int, table_ptr: int, lengths_ptr: int, refs_ptr: int,
                 scratch_ptr: int, error_ptr: int, device: int = 0):
        self._lib = _declare(load_library())
        self._c = LxKvCache(device, n_layers, n_pages, n_seq, max_pages, kv_heads, head_dim, group, page, pool_ptr,
                            table_ptr, lengths_ptr, refs_ptr, scratch_ptr, error_ptr)
        self._ref = ctypes.byref(self._c)
        if not self._lib.lx_kv_pool_bytes(self._ref):
            raise KVError("KVCache: geometry not supported (head_dim 64 or 128, group 32 or 64, page 16, 32, 64 or "
                          "128, counts positive)")

    def _check(self, rc: int, what: str) -> None:
        if rc != LX_OK:
            raise KVError(f"lx_kv_{what} failed: {ERRORS.get(rc, rc)}")

    @staticmethod
    def rows(n: int, total: int, max_rows: int, seqs: int = 0, row0: int = 0, start: int = 0) -> LxKvRows:
        """The rows of a batch (device pointers, 0 = the default of lx_kv_rows)."""
        return LxKvRows(n, total, max_rows, seqs or None, row0 or None, start or None)

    def reset(self, stream: int = 0) -> None:
        """Empty the cache (lengths, tables, refs, error; not the pool)."""
        self._check(self._lib.lx_kv_reset(self._ref, stream or None), "reset")

    def status(self, stream: int = 0) -> int:
        """Wait for the stream; the error bits since the last call (FULL, SLOT, WIDTH, PAGE, ROWS, STUCK)."""
        bits = ctypes.c_int32(0)
        self._check(self._lib.lx_kv_status(self._ref, ctypes.byref(bits), stream or None), "status")
        return bits.value

    def extend(self, n: int, seqs_ptr: int, counts_ptr: int, start_ptr: int, stream: int = 0) -> None:
        """Grow sequences; start gets their old lengths, REFUSED where the pool did not suffice."""
        self._check(self._lib.lx_kv_extend(self._ref, n, seqs_ptr, counts_ptr, start_ptr, stream or None), "extend")

    def _strides(self, strides):
        return (self._c.kv_heads * self._c.head_dim, self._c.head_dim) if strides is None else strides

    def write(self, layer: int, rows: LxKvRows, dtype: str, k_ptr: int, v_ptr: int, k_strides=None, v_strides=None,
              stream: int = 0) -> None:
        """Quantise rows [total, kv_heads, head_dim] into a layer; strides are (row, head) in elements."""
        ks, vs = self._strides(k_strides), self._strides(v_strides)
        self._check(self._lib.lx_kv_write(self._ref, layer, ctypes.byref(rows), DTYPES[dtype], k_ptr, ks[0], ks[1],
                                          v_ptr, vs[0], vs[1], stream or None), "write")

    def read(self, layer: int, rows: LxKvRows, dtype: str, k_ptr: int, v_ptr: int, k_strides=None, v_strides=None,
             stream: int = 0) -> None:
        """The values of rows of a layer, into [total, kv_heads, head_dim]."""
        ks, vs = self._strides(k_strides), self._strides(v_strides)
        self._check(self._lib.lx_kv_read(self._ref, layer, ctypes.byref(rows), DTYPES[dtype], k_ptr, ks[0], ks[1],
                                         v_ptr, vs[0], vs[1], stream or None), "read")

    def attention(self, layer: int, rows: LxKvRows, q_heads: int, dtype: str, q_ptr: int, out_ptr: int, lse: int = 0,
                  scale: float = 0.125, chunk: int = 0, left: int = -1, max_len: int = 0, q_strides=None,
                  out_strides=None, stream: int = 0) -> None:
        """Attention of rows [total, q_heads, head_dim] over a layer; chunk 0 = full, 1 = causal, n = block-causal."""
        d = self._c.head_dim
        qs = (q_heads * d, d) if q_strides is None else q_strides
        os = (q_heads * d, d) if out_strides is None else out_strides
        self._check(self._lib.lx_kv_attention(self._ref, layer, ctypes.byref(rows), q_heads, DTYPES[dtype], q_ptr,
                                              qs[0], qs[1], out_ptr, os[0], os[1], lse or None, scale, chunk, left,
                                              max_len, stream or None), "attention")

    def fork(self, n: int, src_ptr: int, dst_ptr: int, stream: int = 0) -> None:
        """dst[i] (empty) shares the pages of src[i]."""
        self._check(self._lib.lx_kv_fork(self._ref, n, src_ptr, dst_ptr, stream or None), "fork")

    def copy(self, n: int, src_ptr: int, dst_ptr: int, stream: int = 0) -> None:
        """dst[i] (empty) becomes a copy of src[i] on fresh pages."""
        self._check(self._lib.lx_kv_copy(self._ref, n, src_ptr, dst_ptr, stream or None), "copy")

    def free(self, n: int, seqs_ptr: int, keep_ptr: int, stream: int = 0) -> None:
        """Cut sequences to their first keep[i] tokens."""
        self._check(self._lib.lx_kv_free(self._ref, n, seqs_ptr, keep_ptr, stream or None), "free")

    def compact(self, used_ptr: int, stream: int = 0) -> None:
        """Move the used pages to the lowest ids; used gets their count."""
        self._check(self._lib.lx_kv_compact(self._ref, used_ptr, stream or None), "compact")
