"""MXFP4 rows and layers on the host: sizes, refusals, and the reference's own
properties (no GPU call)."""
import ctypes as C

import numpy as np
import pytest

import mx_reference as ref
from eos_amd import _lib, microscale
from eos_amd._lib import EosHipError


@pytest.mark.parametrize("rows,k,blocks", [(1, 1, 1), (3, 32, 1), (3, 33, 2), (7, 4096, 128), (0, 5, 1)])
def test_sizes(rows, k, blocks):
    assert microscale.mx_bytes(rows, k) == (16 * rows * blocks, rows * blocks)


@pytest.mark.parametrize("rows,k,what", [(-1, 32, "rows"), (2 ** 31, 32, "rows"), (1, 0, "k must"),
                                         (1, 2 ** 24 + 1, "k must")])
def test_sizes_refused(rows, k, what):
    with pytest.raises(EosHipError, match=what):
        microscale.mx_bytes(rows, k)


def _quantize(rt=None, x=4096, stride=32, dtype=1, rows=2, k=32, codes=4096, scales=4096):
    _lib.call("eoship_mx_quantize_device", rt, x, stride, dtype, rows, k, codes, scales)


def _dequantize(rt=None, codes=4096, scales=4096, rows=2, k=32, out=4096, stride=32, dtype=1):
    _lib.call("eoship_mx_dequantize_device", rt, codes, scales, rows, k, out, stride, dtype)


@pytest.mark.parametrize("call", [_quantize, _dequantize])
@pytest.mark.parametrize("kw,what", [
    (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(k=0), "k must"),
    (dict(rows=-1), "rows"), (dict(rows=2 ** 31), "rows"), (dict(), "NULL runtime")])
def test_rows_refused(call, kw, what):
    with pytest.raises(EosHipError, match=what):
        call(**kw)


@pytest.mark.parametrize("kw,what", [
    (dict(n=0), "n must"), (dict(n=2 ** 24 + 1), "n must"), (dict(k=0), "k must"),
    (dict(codes=None), "NULL codes"), (dict(scales=None), "NULL codes"),
    (dict(codes=4104), "16-byte"), (dict(bias=4098), "4-byte"), (dict(), "NULL argument")])
def test_bind_refused(kw, what):
    a = dict(codes=4096, scales=4096, n=4, k=32, bias=None) | kw
    out = C.c_void_p(1)
    with pytest.raises(EosHipError, match=what):
        _lib.call("eoship_mx_bind", None, a["codes"], a["scales"], a["n"], a["k"], a["bias"],
                  C.byref(out))
    assert not out


def test_linear_and_release_refuse_null():
    with pytest.raises(EosHipError, match="NULL"):
        _lib.call("eoship_mx_linear_device", None, None, 4096, 32, 1, None, 1, 4096, 32, 1)
    _lib.call("eoship_mx_release", None, None)
    with pytest.raises(ValueError, match="dtype"):
        microscale.quantize(None, None, 0, 32, "i8", None, None)


class _Buf:
    def __init__(self, nbytes):
        self.nbytes, self.ptr = nbytes, C.c_void_p(4096)


class _Rt:
    handle = None


def test_wrapper_checks_sizes():
    with pytest.raises(ValueError, match="x is smaller"):
        microscale.quantize(_Rt, _Buf(127), 2, 32, "bf16", _Buf(32), _Buf(2))
    with pytest.raises(ValueError, match="codes or scales"):
        microscale.quantize(_Rt, _Buf(128), 2, 32, "bf16", _Buf(31), _Buf(2))
    with pytest.raises(ValueError, match="out is smaller"):
        microscale.dequantize(_Rt, _Buf(32), _Buf(2), 2, 32, _Buf(64 + 79), "bf16", 40)
    with pytest.raises(ValueError, match="bias"):
        microscale.MXLinear(_Rt, _Buf(32), _Buf(2), 2, 32, bias=_Buf(7))


def test_reference_rounds_to_the_nearest_level():
    rng = np.random.default_rng(0)
    x = rng.normal(size=(50, 70)) * np.exp(rng.normal(size=(50, 1)) * 20)
    codes, scales = ref.quantize(x)
    v = ref.values(codes, scales, 70)
    for r in range(50):
        for b in range(3):
            s = 2.0 ** (int(scales[r, b]) - 127)
            blk, got = x[r, 32 * b:32 * b + 32], v[r, 32 * b:32 * b + 32]
            assert 4 <= np.abs(blk).max() / s < 8
            near = np.abs(np.abs(blk[:, None]) / s - ref.LEVELS).min(1)
            np.testing.assert_allclose(np.abs(np.abs(blk) - np.abs(got)) / s, near, rtol=0, atol=1e-12)
            assert (np.sign(got) * np.sign(blk) >= 0).all()
    # ties go to the even code, beyond the last level to it
    t = np.array([[.25, .75, 1.25, 1.75, 2.5, 3.5, 5.0, 5.01, 7.9, -.75, -5.0, 4.0]])
    codes, scales = ref.quantize(t)
    np.testing.assert_array_equal(ref.values(codes, scales, 12),
                                  [[0, 1, 1, 2, 2, 4, 4, 6, 6, -1, -4, 4]])
    assert scales[0, 0] == 127
