"""Rotary positions of queries and keys (libeoship): heads turned by the
positions that a paged cache's batch gives them, in pairs or halves, a part of
the head or all of it, with frequencies stretched for long contexts. The
reference turns whole rows by pairs (ropeRows,
runtime/backend/tensor_ops.go:1936-1965).

Rows are device memory, as :mod:`eos_amd.kvcache` takes them. Calls enqueue on
the runtime's stream and do not wait.
"""
from __future__ import annotations

import ctypes as C
import math

import numpy as np

from . import _lib
from .kvcache import KVBatch
from .runtime import Runtime

DTYPES = {"f16": 0, "bf16": 1, "f32": 2}
LAYOUTS = {"pairs": 0, "halves": 1}


def frequencies(rotary_dim: int, base: float = 10000.0, scaling: str | None = None,
                stretch: float = 1.0, original: int = 0, low: float = 1.0,
                high: float = 32.0):
    """(frequencies f64 [rotary_dim / 2], factor) of base^(-2 i / rotary_dim),
    for a context ``stretch`` times the ``original`` number of positions:

    - ``None``: as they are;
    - ``"linear"``: all divided by ``stretch``;
    - ``"base"``: a larger base, so that the lowest frequency is divided by
      ``stretch`` and the highest stays;
    - ``"ramp"``: frequencies that turn less than ``low`` times in the original
      context are divided, those that turn more than ``high`` times stay, by the
      logarithm of the turns (their index) in between; values grow by
      0.1 ln(stretch) + 1;
    - ``"wavelength"``: the same borders, by the turns themselves in between,
      and no growth.
    """
    r = int(rotary_dim)
    if r < 2 or r % 2:
        raise ValueError("rotary_dim must be even and positive")
    if not (base > 1 and stretch >= 1):
        raise ValueError("base must be above 1 and stretch at least 1")
    i = np.arange(0, r, 2, dtype=np.float64) / r
    f = base ** -i
    if scaling is None:
        return f, 1.0
    if scaling == "linear":
        return f / stretch, 1.0
    if scaling == "base":
        if r == 2:
            return f, 1.0
        return (base * stretch ** (r / (r - 2))) ** -i, 1.0
    if scaling not in ("ramp", "wavelength"):
        raise ValueError(f"unknown scaling {scaling!r}")
    if original < 1 or not 0 < low < high:
        raise ValueError("original and 0 < low < high are needed")
    turns = original * f / (2 * math.pi)
    if scaling == "wavelength":
        stay = np.clip((turns - low) / (high - low), 0.0, 1.0)
        return f * (stay + (1 - stay) / stretch), 1.0
    # the (real) index at which a frequency turns so often
    index = lambda n: r * math.log(original / (n * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    first, last = max(math.floor(index(high)), 0), min(math.ceil(index(low)), r - 1)
    stay = 1 - np.clip((np.arange(r // 2) - first) / max(last - first, 1e-3), 0.0, 1.0)
    return f * (stay + (1 - stay) / stretch), 0.1 * math.log(stretch) + 1.0


class Rotary:
    """Frequencies bound for a runtime: ``freq`` f64 [rotary_dim / 2], radians
    a position; values behind the first rotary_dim of a head stay."""

    def __init__(self, rt: Runtime, head_dim: int, freq, layout: str = "halves",
                 factor: float = 1.0):
        if layout not in LAYOUTS:
            raise ValueError(f"layout must be one of {sorted(LAYOUTS)}, got {layout!r}")
        self.rt, self.head_dim = rt, int(head_dim)
        self.handle = C.c_void_p()
        freq = np.ascontiguousarray(freq, np.float64)
        if freq.ndim != 1:
            raise ValueError("freq must be [rotary_dim / 2]")
        d = _lib.EosHipRotaryDesc(head_dim=self.head_dim, rotary_dim=2 * len(freq),
                                  layout=LAYOUTS[layout], factor=float(factor),
                                  frequencies=freq.ctypes.data)
        _lib.call("eoship_rotary_bind", rt.handle, C.byref(d), C.byref(self.handle))

    def release(self) -> None:
        if self.handle and self.rt.handle:
            _lib.call("eoship_rotary_release", self.rt.handle, self.handle)
        self.handle = C.c_void_p()

    def __del__(self):
        try:
            self.release()
        except Exception:
            pass

    def _rows(self, buf, rows: int, width: int, size: int, stride) -> int:
        stride = width if stride is None else int(stride)
        if rows and buf.nbytes < ((rows - 1) * stride + width) * size:
            raise ValueError("a row buffer is smaller than its rows")
        return stride

    def apply(self, where, dtype: str, q=None, heads: int = 0, k=None, kv_heads: int = 0,
              q_out=None, k_out=None, q_stride: int | None = None, k_stride: int | None = None,
              q_out_stride: int | None = None, k_out_stride: int | None = None,
              inverse: bool = False) -> None:
        """Turns queries [rows, heads, head_dim] and keys [rows, kv_heads,
        head_dim] by the positions of ``where``: a :class:`KVBatch`, or a pair
        (positions i32 [rows] on the device, rows). Without ``q_out`` or
        ``k_out`` in place. ``inverse``: back again, the gradient's direction."""
        if dtype not in DTYPES:
            raise ValueError(f"dtype must be one of {sorted(DTYPES)}, got {dtype!r}")
        size, heads, kv_heads = 4 if dtype == "f32" else 2, int(heads), int(kv_heads)
        if isinstance(where, KVBatch):
            batch, positions, rows = C.byref(where.c), None, where.rows
        else:
            positions, rows = where[0], int(where[1])
            if positions.nbytes < 4 * rows:
                raise ValueError("positions are fewer than rows")
            batch, positions = None, positions.ptr
        qp = qop = kp = kop = None
        qs = qos = ks = kos = 0
        if q is None:
            heads = 0
        else:
            qs = self._rows(q, rows, heads * self.head_dim, size, q_stride)
            qop, qos = q.ptr, qs
            if q_out is not None:
                qop, qos = q_out.ptr, self._rows(q_out, rows, heads * self.head_dim, size, q_out_stride)
            qp = q.ptr
        if k is None:
            kv_heads = 0
        else:
            ks = self._rows(k, rows, kv_heads * self.head_dim, size, k_stride)
            kop, kos = k.ptr, ks
            if k_out is not None:
                kop, kos = k_out.ptr, self._rows(k_out, rows, kv_heads * self.head_dim, size, k_out_stride)
            kp = k.ptr
        _lib.call("eoship_rotary_device", self.rt.handle, self.handle, batch, positions, rows,
                  1 if inverse else 0, DTYPES[dtype], qp, qs, heads, qop, qos, kp, ks, kv_heads, kop,
                  kos)
