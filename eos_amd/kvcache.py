"""Paged key-value cache and the attention over it (libeoship): what a
decoder-type embedder or reranker keeps between its calls, stored as f16 or
bf16, as 8-bit codes (``q8``) or as 4-bit Hadamard TurboQuant codes (``tq4``).
The counterpart of the kv_cache capability that the reference's CUDA backend
advertises (runtime/backend/backend.go:1428-1431).

Rows and pools are device memory: anything with ``ptr`` (its address) and
``nbytes``, as :class:`~eos_amd.runtime.DeviceBuffer` has them. Calls enqueue
on the runtime's stream and do not wait.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _lib
from .runtime import DeviceBuffer, Runtime

FORMATS = {"f16": 0, "bf16": 1, "q8": 2, "tq4": 3}
DTYPES = {"f16": 0, "bf16": 1, "f32": 2}


def gaussian_codebook() -> np.ndarray:
    """The 8 magnitudes of the 16-level quantizer with the least squared error
    for a normal variable (its published table, rounded to f16)."""
    return np.array([0.1284, 0.3881, 0.6568, 0.9424, 1.2562, 1.6181, 2.0690, 2.7326],
                    np.float16).astype(np.float32)


def _desc(fmt: str, kv_heads: int, head_dim: int, page_tokens: int, pages: int):
    if fmt not in FORMATS:
        raise ValueError(f"format must be one of {sorted(FORMATS)}, got {fmt!r}")
    return _lib.EosHipKVDesc(format=FORMATS[fmt], kv_heads=int(kv_heads), head_dim=int(head_dim),
                             page_tokens=int(page_tokens), pages=int(pages))


def kv_bytes(fmt: str, kv_heads: int, head_dim: int, page_tokens: int, pages: int):
    """(bytes of the K pool and of the V pool, bytes of each scale pool)."""
    pool, scale = C.c_int64(), C.c_int64()
    d = _desc(fmt, kv_heads, head_dim, page_tokens, pages)
    _lib.call("eoship_kv_bytes", C.byref(d), C.byref(pool), C.byref(scale))
    return pool.value, scale.value


def check_batch(fmt: str, kv_heads: int, head_dim: int, page_tokens: int, pages: int, page_table,
                lengths, offsets=None, rows: int | None = None, writes: bool = False,
                window: int = 0) -> None:
    """Checks a batch's host arrays (page ids, lengths, offsets; with
    ``writes`` also that no page is written twice) before they are uploaded.
    With a ``window``, attention's own, pages in front of every row's window may
    be gone; 1 asks for the pages of the rows themselves only."""
    table = np.ascontiguousarray(page_table, np.int32)
    if table.ndim != 2:
        raise ValueError("page_table must be [batch, pages]")
    lens = np.ascontiguousarray(lengths, np.int32)
    batch = table.shape[0]
    if lens.shape != (batch,):
        raise ValueError("lengths must be [batch]")
    off = None
    if offsets is not None:
        off = np.ascontiguousarray(offsets, np.int32)
        if off.shape != (batch + 1,):
            raise ValueError("offsets must be [batch + 1]")
    if rows is None:
        rows = batch if off is None else int(off[-1])
    d = _desc(fmt, kv_heads, head_dim, page_tokens, pages)
    _lib.call("eoship_kv_check_batch_window", C.byref(d), table.ctypes.data_as(C.c_void_p),
              C.c_int32(table.shape[1]), C.c_int32(batch), lens.ctypes.data_as(C.c_void_p),
              off.ctypes.data_as(C.c_void_p) if off is not None else None, C.c_int64(rows),
              C.c_int32(int(window)), C.c_int32(int(writes)))


def _address(buf):
    if buf is None:
        return None
    p = buf.ptr
    return p.value if isinstance(p, C.c_void_p) else p


class KVBatch:
    """A batch of sequences and the rows of a call: page ids i32
    [batch, table_stride], lengths i32 [batch] with the call's rows included,
    and row ranges i32 [batch + 1] (``offsets`` None: one row a sequence, the
    form for decoding). All on the device."""

    def __init__(self, page_table, table_stride: int, batch: int, lengths, offsets=None,
                 rows: int | None = None):
        if rows is None:
            if offsets is not None:
                raise ValueError("rows is needed with offsets")
            rows = batch
        self._keep = (page_table, lengths, offsets)
        self.batch, self.rows = int(batch), int(rows)
        for buf, need in ((page_table, 4 * self.batch * int(table_stride)),
                          (lengths, 4 * self.batch), (offsets, 4 * (self.batch + 1))):
            if buf is not None and buf.nbytes < need:
                raise ValueError("a batch array is smaller than its batch")
        self.c = _lib.EosHipKVBatch(_address(page_table), int(table_stride), self.batch,
                                    _address(lengths), _address(offsets), self.rows)


class KVCache:
    """A paged cache over the caller's pools (or its own, where none are
    given). ``codebook`` (8 magnitudes) and ``signs`` (+-1, [head_dim]) are
    tq4's tables; without them a normal codebook and signs drawn from ``seed``.
    """

    def __init__(self, rt: Runtime, fmt: str, kv_heads: int, head_dim: int, page_tokens: int,
                 pages: int, k=None, v=None, k_scale=None, v_scale=None, codebook=None, signs=None,
                 seed: int = 0):
        self.rt = rt
        self.handle = C.c_void_p()
        self.fmt, self.kv_heads, self.head_dim = fmt, int(kv_heads), int(head_dim)
        self.page_tokens, self.pages = int(page_tokens), int(pages)
        pool, scale = kv_bytes(fmt, kv_heads, head_dim, page_tokens, pages)
        self._own = []
        bufs = []
        for buf, need in ((k, pool), (v, pool), (k_scale, scale), (v_scale, scale)):
            if buf is None and need:
                buf = DeviceBuffer(rt, need)
                self._own.append(buf)
            if need and buf.nbytes < need:
                raise ValueError("a pool is smaller than its pages")
            bufs.append(buf if need else None)
        self.k, self.v, self.k_scale, self.v_scale = bufs
        d = _desc(fmt, kv_heads, head_dim, page_tokens, pages)
        d.d_k, d.d_v, d.d_k_scale, d.d_v_scale = (_address(b) for b in bufs)
        if fmt == "tq4":
            cb = gaussian_codebook() if codebook is None else codebook
            if signs is None:
                signs = np.random.default_rng(seed).choice([-1.0, 1.0], self.head_dim)
            self.codebook = np.ascontiguousarray(cb, np.float32)
            self.signs = np.ascontiguousarray(signs, np.float32)
            if self.codebook.shape != (8,) or self.signs.shape != (self.head_dim,):
                raise ValueError("codebook [8] and signs [head_dim] required")
            d.codebook = self.codebook.ctypes.data
            d.signs = self.signs.ctypes.data
        _lib.call("eoship_kv_bind", rt.handle, C.byref(d), C.byref(self.handle))

    def release(self) -> None:
        if self.handle and self.rt.handle:
            _lib.call("eoship_kv_release", self.rt.handle, self.handle)
            for b in self._own:
                b.free()
        self.handle, self._own = C.c_void_p(), []

    def __del__(self):
        try:
            self.release()
        except Exception:
            pass

    def _rows(self, batch: KVBatch, width: int, dtype: str, *bufs):
        """Strides of (buffer, stride) pairs, the buffers' sizes checked."""
        if dtype not in DTYPES:
            raise ValueError(f"dtype must be one of {sorted(DTYPES)}, got {dtype!r}")
        size = 4 if dtype == "f32" else 2
        out = []
        for buf, stride in bufs:
            stride = width if stride is None else int(stride)
            if batch.rows and buf.nbytes < ((batch.rows - 1) * stride + width) * size:
                raise ValueError("a row buffer is smaller than the batch's rows")
            out.append(stride)
        return out

    def append(self, batch: KVBatch, k, v, dtype: str, k_stride: int | None = None,
               v_stride: int | None = None) -> None:
        """Writes rows of keys and values [rows, kv_heads, head_dim] (``dtype``
        f16 or bf16, strides in elements between rows) at the sequences' last
        positions."""
        ks, vs = self._rows(batch, self.kv_heads * self.head_dim, dtype, (k, k_stride),
                            (v, v_stride))
        _lib.call("eoship_kv_append_device", self.rt.handle, self.handle, C.byref(batch.c), k.ptr,
                  ks, v.ptr, vs, DTYPES[dtype])

    def read(self, batch: KVBatch, k, v, dtype: str, k_stride: int | None = None,
             v_stride: int | None = None) -> None:
        """The values at the sequences' last positions into rows of ``dtype``
        (f16, bf16 or f32)."""
        ks, vs = self._rows(batch, self.kv_heads * self.head_dim, dtype, (k, k_stride),
                            (v, v_stride))
        _lib.call("eoship_kv_read_device", self.rt.handle, self.handle, C.byref(batch.c), k.ptr,
                  ks, v.ptr, vs, DTYPES[dtype])

    def attend(self, batch: KVBatch, q, heads: int, out, dtype: str, scale: float | None = None,
               window: int = 0, q_stride: int | None = None, out_stride: int | None = None,
               lse=None) -> None:
        """Attention of the rows' queries [rows, heads, head_dim] over the
        cached positions up to their own (the last ``window`` of them where it
        is positive): ``out`` [rows, heads, head_dim] and, if given, ``lse``
        f32 [rows, heads]. ``scale`` None: 1 / sqrt(head_dim)."""
        qs, os_ = self._rows(batch, int(heads) * self.head_dim, dtype, (q, q_stride),
                             (out, out_stride))
        if lse is not None and lse.nbytes < batch.rows * int(heads) * 4:
            raise ValueError("lse is smaller than the batch's rows")
        _lib.call("eoship_kv_attention_device", self.rt.handle, self.handle, C.byref(batch.c),
                  q.ptr, qs, int(heads), DTYPES[dtype],
                  self.head_dim ** -0.5 if scale is None else float(scale), int(window), out.ptr,
                  os_, lse.ptr if lse is not None else None)

    def status(self) -> int:
        """0 where every page id, length and offset of the calls since the last
        look was in range (bit 0: a page id, 1: a length, 2: an offset); waits."""
        st = C.c_int32()
        _lib.call("eoship_kv_status", self.rt.handle, self.handle, C.byref(st))
        return st.value
