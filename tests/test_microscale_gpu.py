"""MXFP4 rows and linear layers on the GPU against their 64-bit restatement:
codes and scales bit for bit, products within the f32 sums' bound."""
import numpy as np
import pytest

import mx_reference as ref
from eos_amd import microscale
from eos_amd._lib import EosHipError
from eos_amd.microscale import MXLinear
from eos_amd.runtime import DeviceBuffer, Runtime

pytestmark = pytest.mark.gpu


def _case(name):
    print(f"[case] {name}", flush=True)


def _rows(rng, rows, k, dtype, spread=1.0):
    """Rows of a type, in a wider array whose gaps hold NaN."""
    x = rng.normal(size=(rows, k)) * np.exp(spread * rng.normal(size=(rows, k)))
    stride = -(-k // 8) * 8 + 16
    b = ref.to_bits(np.full((rows, stride), np.nan), dtype)
    b[:, :k] = ref.to_bits(x, dtype)
    return b, stride, ref.from_bits(b[:, :k], dtype)


def _tight(b, stride, k):
    """The array without what lies behind its last row."""
    return np.ascontiguousarray(b).reshape(-1)[:(b.shape[0] - 1) * stride + k]


def _quantize(rt, b, stride, rows, k, dtype):
    x = DeviceBuffer.from_array(rt, _tight(b, stride, k))
    blocks = -(-k // 32)
    codes = DeviceBuffer.from_array(rt, np.full(rows * blocks * 16 + 32, 0xa5, np.uint8))
    scales = DeviceBuffer.from_array(rt, np.full(rows * blocks + 32, 0xa5, np.uint8))
    microscale.quantize(rt, x, rows, k, dtype, codes, scales, stride)
    return codes, scales


def _take(buf, rows, width):
    """(rows, what lies behind them)"""
    a = buf.download(np.uint8, (buf.nbytes,))
    return a[:rows * width].reshape(rows, width), a[rows * width:]


SHAPES = [(1, 1), (1, 31), (2, 32), (5, 33), (3, 100), (64, 128), (17, 1000), (130, 4096), (1, 16384),
          (1000, 40)]


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,k", SHAPES)
def test_quantize_and_back(rt, dtype, rows, k):
    _case(f"quantize {dtype} {rows} x {k}")
    rng = np.random.default_rng(rows * 7 + k)
    b, stride, x = _rows(rng, rows, k, dtype)
    codes, scales = _quantize(rt, b, stride, rows, k, dtype)
    blocks = -(-k // 32)
    (c, c_rest), (s, s_rest) = _take(codes, rows, blocks * 16), _take(scales, rows, blocks)
    want_c, want_s = ref.quantize(x)
    np.testing.assert_array_equal(s, want_s)
    np.testing.assert_array_equal(ref.values(c, s, blocks * 32), ref.values(want_c, want_s, blocks * 32))
    assert (c_rest == 0xa5).all() and (s_rest == 0xa5).all()
    for out in ("f16", "bf16", "f32"):
        gap = ref.to_bits(np.full((rows, stride), 777.0), out)
        buf = DeviceBuffer.from_array(rt, gap)
        microscale.dequantize(rt, codes, scales, rows, k, buf, out, stride)
        got = buf.download(gap.dtype, gap.shape)
        np.testing.assert_array_equal(
            ref.from_bits(got[:, :k], out),
            ref.from_bits(ref.to_bits(ref.values(c, s, k), out), out))
        np.testing.assert_array_equal(got[:, k:], gap[:, k:])


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_quantize_edges(rt, dtype):
    """Ties, saturation, zeros, the ends of the types and of the scale, values
    that are not finite."""
    _case(f"edges {dtype}")
    ties = [.25, .75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.75, 4.0, 0.125, -0.0]
    rows = []
    low, high = {"f16": (-14, 12), "bf16": (-126, 124), "f32": (-126, 124)}[dtype]
    for e in (low, low + 5, -3, 0, 7, high):
        for sign in (1, -1):
            r = np.zeros(32)
            r[:13] = np.array(ties) * sign * 2.0 ** e
            r[13] = 4.0 * 2.0 ** e
            rows.append(r)
    tiny = {"f16": 2.0 ** -24, "bf16": 2.0 ** -133, "f32": 2.0 ** -149}[dtype]
    rows.append(np.zeros(32))
    rows.append(np.full(32, -0.0))
    rows.append(np.arange(32) * tiny)
    rows.append(np.arange(32) * tiny * 17)
    rows.append(np.where(np.arange(32) % 5 == 0, {"f16": 65504.0, "bf16": 2.0 ** 127 * 1.9921875,
                                                  "f32": 3.4028234e38}[dtype], 1.0))
    for bad in (np.inf, -np.inf, np.nan):
        r = np.ones(32)
        r[31 if bad == np.inf else 3] = bad
        rows.append(r)
    x = np.array(rows)
    x = np.concatenate([x, x[::-1]], 1)  # two blocks a row
    b = ref.to_bits(x, dtype)
    x = ref.from_bits(b, dtype)
    n = len(x)
    codes, scales = _quantize(rt, b, 64, n, 64, dtype)
    (c, _), (s, _) = _take(codes, n, 32), _take(scales, n, 2)
    want_c, want_s = ref.quantize(x)
    np.testing.assert_array_equal(s, want_s)
    np.testing.assert_array_equal(ref.values(c, s, 64), ref.values(want_c, want_s, 64))
    out = DeviceBuffer(rt, n * 64 * 4)
    microscale.dequantize(rt, codes, scales, n, 64, out, "f32")
    np.testing.assert_array_equal(out.download(np.float32, (n, 64)).astype(np.float64),
                                  ref.values(c, s, 64))


def test_every_code_and_scale_comes_back(rt):
    """All 256 scale bytes times all codes, to every type."""
    c = np.tile((np.arange(16) | ((np.arange(16) * 7 + 3) % 16) << 4).astype(np.uint8), (256, 1))
    s = np.arange(256, dtype=np.uint8).reshape(256, 1)
    codes, scales = DeviceBuffer.from_array(rt, c), DeviceBuffer.from_array(rt, s)
    for out in ("f32", "bf16", "f16"):
        buf = DeviceBuffer(rt, 256 * 32 * 4)
        microscale.dequantize(rt, codes, scales, 256, 32, buf, out)
        got = ref.from_bits(buf.download(ref.np_dtype(out), (256, 32)), out)
        with np.errstate(over="ignore"):
            want = ref.from_bits(ref.to_bits(ref.values(c, s, 32).astype(np.float32), out), out)
        np.testing.assert_array_equal(got, want)


# ------------------------------------------------------------------- layers


class Layer:
    def __init__(self, rt, rng, n, k, bias=True, w=None):
        w = rng.normal(size=(n, k)) / np.sqrt(k) * np.exp(rng.normal(size=(n, 1))) if w is None else w
        self.codes, self.scales = ref.quantize(w)
        self.w, self.n, self.k = ref.values(self.codes, self.scales, k), n, k
        self.bias = rng.normal(size=n).astype(np.float32) if bias else None
        up = lambda a: DeviceBuffer.from_array(rt, a)  # noqa: E731
        self.layer = MXLinear(rt, up(self.codes), up(self.scales), n, k,
                              up(self.bias) if bias else None)


def _apply(rt, layer, b, stride, rows, dtype, out, scales=None):
    """The layer's rows, in an array whose gaps have to stay."""
    n = layer.n
    ostride = -(-n // 8) * 8 + 8
    gap = ref.to_bits(np.full((rows, ostride), 777.0), out)
    buf = DeviceBuffer.from_array(rt, gap)
    if dtype == "mxfp4":
        layer.layer.apply(DeviceBuffer.from_array(rt, b), rows, dtype, buf, out, out_stride=ostride,
                          x_scales=DeviceBuffer.from_array(rt, scales))
    else:
        x = DeviceBuffer.from_array(rt, _tight(b, stride, layer.k))
        layer.layer.apply(x, rows, dtype, buf, out, x_stride=stride, out_stride=ostride)
    got = buf.download(gap.dtype, gap.shape)
    np.testing.assert_array_equal(got[:, n:], gap[:, n:])
    return ref.from_bits(got[:, :n], out)


def _check(got, want, tol):
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], tol[bad][:5])


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 33, 48, 64, 65, 130, 300])
@pytest.mark.parametrize("n,k", [(1, 1), (3, 31), (16, 32), (17, 100), (100, 129), (64, 512),
                                 (257, 1000), (1000, 640), (24, 4111)])
def test_linear(rt, rows, n, k):
    i = rows + n + k
    dtype, out = ("f16", "bf16", "f32")[i % 3], ("bf16", "f32", "f16", "f32")[i % 4]
    _case(f"linear {dtype} -> {out} {rows} x {k} x {n}")
    rng = np.random.default_rng(i)
    layer = Layer(rt, rng, n, k, bias=i % 2 == 0)
    b, stride, x = _rows(rng, rows, k, dtype, 0.5)
    codes, scales = ref.quantize(x)
    want, tol = ref.linear(ref.values(codes, scales, k), layer.w, layer.bias, out)
    got = _apply(rt, layer, b, stride, rows, dtype, out)
    _check(got, want, tol)
    again = _apply(rt, layer, codes, 0, rows, "mxfp4", out, scales)
    _check(again, want, tol)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("out", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows", [1, 40, 200])
def test_linear_types(rt, dtype, out, rows):
    _case(f"types {dtype} -> {out} {rows}")
    rng = np.random.default_rng(5)
    layer = Layer(rt, rng, 200, 384)
    b, stride, x = _rows(rng, rows, 384, dtype)
    want, tol = ref.linear(ref.values(*ref.quantize(x), 384), layer.w, layer.bias, out)
    _check(_apply(rt, layer, b, stride, rows, dtype, out), want, tol)


@pytest.mark.parametrize("rows,n,k", [(8, 6144, 4096), (70, 4096, 2048), (1024, 1024, 1024),
                                      (777, 1531, 1000), (2500, 520, 256), (513, 2050, 768)])
def test_linear_larger(rt, rows, n, k):
    _case(f"larger {rows} x {k} x {n}")
    rng = np.random.default_rng(rows)
    layer = Layer(rt, rng, n, k, bias=False)
    b, stride, x = _rows(rng, rows, k, "bf16", 0.5)
    want, tol = ref.linear(ref.values(*ref.quantize(x), k), layer.w, None, "f32")
    _check(_apply(rt, layer, b, stride, rows, "bf16", "f32"), want, tol)


@pytest.mark.parametrize("rows", [5, 20, 100, 300])
def test_linear_values_not_finite_stay_in_their_rows(rt, rows):
    """A block that stands for NaN makes its row, or its output, NaN and no other."""
    _case(f"nan {rows}")
    rng = np.random.default_rng(2)
    k, n = 300, 90
    w = rng.normal(size=(n, k))
    w[7, 40], w[60, 299] = np.inf, np.nan
    layer = Layer(rt, rng, n, k, w=w)
    b, stride, _ = _rows(rng, rows, k, "bf16")
    b[3, 299] = 0x7f80
    b[rows - 1, 0] = 0x7fc0
    x = ref.from_bits(b[:, :k], "bf16")
    want, tol = ref.linear(ref.values(*ref.quantize(x), k), layer.w, layer.bias, "f32")
    got = _apply(rt, layer, b, stride, rows, "bf16", "f32")
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    assert np.isnan(got[3]).all() and np.isnan(got[:, 7]).all() and not np.isnan(got[0, 0])
    ok = ~np.isnan(want)
    _check(got[ok], want[ok], tol[ok])


@pytest.mark.parametrize("rows", [4, 150])
def test_linear_scales_at_their_ends(rt, rows):
    """Scale bytes of 0 and 254 against each other, zero blocks beside large ones."""
    _case(f"scale ends {rows}")
    rng = np.random.default_rng(3)
    k, n = 256, 40
    w = rng.normal(size=(n, k)) * 2.0 ** np.repeat(rng.integers(90, 120, (n, 8)), 32, 1)
    layer = Layer(rt, rng, n, k, bias=False, w=w)
    x = rng.normal(size=(rows, k)) * 2.0 ** np.repeat(rng.integers(-125, -100, (rows, 8)), 32, 1)
    x[0] = 0.0
    x[1, :64] = 2.0 ** -133  # a bf16 subnormal: scale byte 0
    b = ref.to_bits(x, "bf16")
    x = ref.from_bits(b, "bf16")
    want, tol = ref.linear(ref.values(*ref.quantize(x), k), layer.w, None, "f32")
    got = _apply(rt, layer, b, k, rows, "bf16", "f32")
    _check(got, want, tol)
    assert (got[0] == 0).all()


def _filled(rt, nbytes, byte):
    from eos_amd import _lib
    buf = DeviceBuffer(rt, nbytes)
    _lib.call("eoship_memset", rt.handle, buf.ptr, byte, nbytes)
    return buf


@pytest.mark.parametrize("rows", [1, 20, 65])
def test_weights_beyond_four_gigabytes(rt, rows):
    """131,077 weights rows of 65,536 ones, some rows others; sums of whole numbers."""
    _case(f"large weights {rows}")
    n, k = 131077, 65536
    codes, scales = _filled(rt, n * k // 2, 0x22), _filled(rt, n * k // 32, 127)  # 1.0, 1.0
    want = np.full(n, float(k))
    for i, (byte, value) in {0: (0x44, 2.0), 77777: (0xAA, -1.0), 131071: (0x11, 0.5),
                             131072: (0x22, 1.0), n - 1: (0x66, 4.0)}.items():
        codes.view(i * k // 2, k // 2).upload(np.full(k // 2, byte, np.uint8))
        want[i] = value * k
    layer = MXLinear(rt, codes, scales, n, k)
    codes.free()
    scales.free()
    x = np.ones((rows, k), np.float16)
    x[rows // 2] = -1.5
    out = DeviceBuffer(rt, rows * (n + 3) * 4)
    layer.apply(DeviceBuffer.from_array(rt, x), rows, "f16", out, "f32", out_stride=n + 3)
    got = out.download(np.float32, (rows, n + 3))[:, :n]
    for r in range(rows):
        np.testing.assert_array_equal(got[r], want * float(x[r, 0]))
    layer.release()


def test_rows_beyond_four_gigabytes(rt):
    """2^21 + 35 rows of 4,096 codes; their last rows differ."""
    _case("large rows")
    rows, k, n = (1 << 21) + 35, 4096, 8
    x, xs = _filled(rt, rows * k // 2, 0x22), _filled(rt, rows * k // 32, 127)
    want = np.full(rows, float(k))
    for i, (byte, value) in {5: (0x44, 2.0), 1 << 20: (0xAA, -1.0), rows - 35: (0x11, 0.5),
                             rows - 1: (0x66, 4.0)}.items():
        x.view(i * k // 2, k // 2).upload(np.full(k // 2, byte, np.uint8))
        want[i] = value * k
    w = np.ones((n, k))
    w[3] = 0.0
    c, s = ref.quantize(w)
    layer = MXLinear(rt, DeviceBuffer.from_array(rt, c), DeviceBuffer.from_array(rt, s), n, k)
    out = DeviceBuffer(rt, rows * n * 4)
    layer.apply(x, rows, "mxfp4", out, "f32", x_scales=xs)
    got = out.download(np.float32, (rows, n))
    for j in range(n):
        np.testing.assert_array_equal(got[:, j], want * (j != 3))
    back = DeviceBuffer(rt, rows * k * 2)  # 17 GB: offsets of rows beyond 32 bits
    microscale.dequantize(rt, x, xs, rows, k, back, "bf16")
    again, ags = _filled(rt, rows * k // 2, 0), _filled(rt, rows * k // 32, 0)
    microscale.quantize(rt, back, rows, k, "bf16", again, ags)
    for i in (0, 5, 1 << 20, rows - 35, rows - 2, rows - 1):
        got = back.view(i * k * 2, k * 2).download(np.uint16, (k,))
        np.testing.assert_array_equal(ref.from_bits(got, "bf16"), want[i] / k)
        c = again.view(i * k // 2, k // 2).download(np.uint8, (1, k // 2))
        s = ags.view(i * k // 32, k // 32).download(np.uint8, (1, k // 32))
        np.testing.assert_array_equal(ref.values(c, s, k)[0], want[i] / k)
    for b in (x, xs, out, back, again, ags):
        b.free()


def test_linear_of_no_rows_and_after_the_weights_are_gone(rt):
    rng = np.random.default_rng(4)
    w = rng.normal(size=(33, 70)).astype(np.float32)
    dev = DeviceBuffer.from_array(rt, np.pad(w, ((0, 0), (0, 2))))
    layer = MXLinear.from_rows(rt, dev, 33, 70, "f32", 72)
    dev.upload(np.zeros((33, 72), np.float32))
    dev.free()
    out = DeviceBuffer.from_array(rt, np.full((2, 40), 5.0, np.float32))
    x = rng.normal(size=(2, 72)).astype(np.float32)
    buf = DeviceBuffer.from_array(rt, x)
    layer.apply(buf, 0, "f32", out, out_stride=40, x_stride=72)
    assert (out.download(np.float32, (2, 40)) == 5.0).all()
    layer.apply(buf, 2, "f32", out, out_stride=40, x_stride=72)
    got = out.download(np.float32, (2, 40))
    want, tol = ref.linear(ref.values(*ref.quantize(x[:, :70].astype(np.float64)), 70),
                           ref.values(*ref.quantize(w.astype(np.float64)), 70), None, "f32")
    _check(got[:, :33], want, tol)
    layer.release()
    layer.release()


def test_equal_calls_give_equal_results(rt):
    """No sum depends on the order in which workgroups end."""
    rng = np.random.default_rng(6)
    for rows, n, k in ((1, 640, 8192), (20, 512, 4096), (200, 300, 2048)):
        layer = Layer(rt, rng, n, k)
        b, stride, _ = _rows(rng, rows, k, "bf16")
        first = _apply(rt, layer, b, stride, rows, "bf16", "f32")
        for _ in range(3):
            np.testing.assert_array_equal(_apply(rt, layer, b, stride, rows, "bf16", "f32"), first)


def test_two_runtimes_and_refusals(rt):
    rng = np.random.default_rng(7)
    layer = Layer(rt, rng, 48, 64)
    buf = DeviceBuffer(rt, 1 << 16)
    with Runtime(0) as other:
        with pytest.raises(EosHipError, match="another runtime"):
            MXLinear.apply(_Other(layer.layer, other), buf, 1, "bf16", buf)
        mine = Layer(other, rng, 48, 64)
        b, stride, x = _rows(rng, 9, 64, "f16")
        for t in (layer, mine):
            want, tol = ref.linear(ref.values(*ref.quantize(x), 64), t.w, t.bias, "f32")
            _check(_apply(t.layer.rt, t, b, stride, 9, "f16", "f32"), want, tol)
        mine.layer.release()
    for kw, what in ((dict(x_stride=60), "stride of x"), (dict(x_stride=68), "stride of x"),
                     (dict(out_stride=40), "stride of out"), (dict(out_stride=52), "stride of out")):
        with pytest.raises(EosHipError, match=what):
            layer.layer.apply(buf, 2, "bf16", buf, **kw)
    with pytest.raises(EosHipError, match="x is not 16-byte"):
        layer.layer.apply(buf.view(2, 4096), 2, "bf16", buf)
    with pytest.raises(EosHipError, match="out is not 16-byte"):
        layer.layer.apply(buf, 2, "bf16", buf.view(8, 4096))
    with pytest.raises(ValueError, match="x_scales"):
        layer.layer.apply(buf, 2, "mxfp4", buf, "bf16")
    with pytest.raises(EosHipError, match="rows"):
        layer.layer.apply(buf, -1, "bf16", buf)


class _Other:
    def __init__(self, layer, rt):
        self.handle, self.rt, self.n, self.k = layer.handle, rt, layer.n, layer.k
