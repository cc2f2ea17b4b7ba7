"""Rows in microscaled 4-bit floating point (MXFP4) and linear layers over
weights held so (libeoship): blocks of 32 values with a power-of-two scale, the
form that gfx950's matrix units multiply directly. Beside the q8 encoder's
products for models that are served from 4 bits (the reference stores q4
weights too, runtime/weight_file.go:315-333, and unpacks them at load).

Rows, codes and scales are device memory: anything with ``ptr`` (its address)
and ``nbytes``, as :class:`~eos_amd.runtime.DeviceBuffer` has them. Calls
enqueue on the runtime's stream and do not wait.
"""
from __future__ import annotations

import ctypes as C

from . import _lib
from .runtime import DeviceBuffer, Runtime

DTYPES = {"f16": 0, "bf16": 1, "f32": 2}
_SIZES = {"f16": 2, "bf16": 2, "f32": 4}


def mx_bytes(rows: int, k: int):
    """(bytes of the codes, bytes of the scales) of rows of k values."""
    codes, scales = C.c_int64(), C.c_int64()
    _lib.call("eoship_mx_bytes", int(rows), int(k), C.byref(codes), C.byref(scales))
    return codes.value, scales.value


def _stride(buf, rows: int, width: int, dtype: str, stride, name: str) -> int:
    if dtype not in DTYPES:
        raise ValueError(f"dtype must be one of {sorted(DTYPES)}, got {dtype!r}")
    stride = width if stride is None else int(stride)
    if rows > 0 and buf.nbytes < ((rows - 1) * stride + width) * _SIZES[dtype]:
        raise ValueError(f"{name} is smaller than its rows")
    return stride


def _held(codes, scales, rows: int, k: int) -> None:
    blocks = rows * -(-k // 32)
    if codes.nbytes < 16 * blocks or scales.nbytes < blocks:
        raise ValueError("codes or scales are smaller than their rows")


def quantize(rt: Runtime, x, rows: int, k: int, dtype: str, codes, scales,
             x_stride: int | None = None) -> None:
    """Rows x [rows, k] into codes u8 [rows, ceil(k / 32), 16] and scales u8
    [rows, ceil(k / 32)]."""
    rows, k = int(rows), int(k)
    stride = _stride(x, rows, k, dtype, x_stride, "x")
    _held(codes, scales, rows, k)
    _lib.call("eoship_mx_quantize_device", rt.handle, x.ptr, stride, DTYPES[dtype], rows, k,
              codes.ptr, scales.ptr)


def dequantize(rt: Runtime, codes, scales, rows: int, k: int, out, dtype: str,
               out_stride: int | None = None) -> None:
    """The values that codes and scales stand for into rows out [rows, k]."""
    rows, k = int(rows), int(k)
    stride = _stride(out, rows, k, dtype, out_stride, "out")
    _held(codes, scales, rows, k)
    _lib.call("eoship_mx_dequantize_device", rt.handle, codes.ptr, scales.ptr, rows, k, out.ptr,
              stride, DTYPES[dtype])


class MXLinear:
    """A linear layer of n outputs over k inputs, its weights [n, k] given as
    codes and scales and laid out anew on the device (the given ones are not
    needed afterwards). ``bias``: f32 [n]."""

    def __init__(self, rt: Runtime, codes, scales, n: int, k: int, bias=None):
        self.rt, self.n, self.k = rt, int(n), int(k)
        self.handle = C.c_void_p()
        _held(codes, scales, self.n, self.k)
        if bias is not None and bias.nbytes < 4 * self.n:
            raise ValueError("bias is smaller than [n]")
        _lib.call("eoship_mx_bind", rt.handle, codes.ptr, scales.ptr, self.n, self.k,
                  bias.ptr if bias is not None else None, C.byref(self.handle))

    @classmethod
    def from_rows(cls, rt: Runtime, w, n: int, k: int, dtype: str, w_stride: int | None = None,
                  bias=None) -> "MXLinear":
        """A layer of weights that are still f16, bf16 or f32 rows."""
        codes, scales = (DeviceBuffer(rt, b) for b in mx_bytes(n, k))
        quantize(rt, w, n, k, dtype, codes, scales, w_stride)
        layer = cls(rt, codes, scales, n, k, bias)
        codes.free()
        scales.free()
        return layer

    def release(self) -> None:
        if self.handle and self.rt.handle:
            _lib.call("eoship_mx_release", self.rt.handle, self.handle)
        self.handle = C.c_void_p()

    def __del__(self):
        try:
            self.release()
        except Exception:
            pass

    def apply(self, x, rows: int, dtype: str, out, out_dtype: str | None = None,
              x_stride: int | None = None, out_stride: int | None = None, x_scales=None) -> None:
        """out [rows, n] = Q(x) W^T + bias for rows x [rows, k] of ``dtype``
        (quantised within the call), or for codes x with ``x_scales``
        (``dtype`` "mxfp4"). ``out_dtype`` None: x's."""
        rows = int(rows)
        if dtype == "mxfp4":
            if x_scales is None:
                raise ValueError("x_scales is needed with codes")
            _held(x, x_scales, rows, self.k)
            kind, xs, scales = 3, 0, x_scales.ptr
        else:
            xs, scales = _stride(x, rows, self.k, dtype, x_stride, "x"), None
            kind = DTYPES[dtype]
        out_dtype = dtype if out_dtype is None else out_dtype
        os_ = _stride(out, rows, self.n, out_dtype, out_stride, "out")
        _lib.call("eoship_mx_linear_device", self.rt.handle, self.handle, x.ptr, xs, kind, scales,
                  rows, out.ptr, os_, DTYPES[out_dtype])
