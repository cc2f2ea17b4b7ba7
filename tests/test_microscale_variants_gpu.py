"""Every kernel that a linear layer of MXFP4 weights takes, on values that differ
along all axes, against 64 bits; which one a call took is read from its launches."""
import numpy as np
import pytest

import mx_reference as ref
from eos_amd.microscale import MXLinear
from eos_amd.runtime import DeviceBuffer

pytestmark = pytest.mark.gpu

TYPES = ("f16", "bf16", "f32")


def _codes(rng, rows, k):
    """Random codes and scales of rows of k values, zeros behind them."""
    blocks = -(-k // 32)
    c = rng.integers(0, 256, (rows, blocks, 16), np.uint8)
    left = k - 32 * (blocks - 1)
    c[:, -1, (left + 1) // 2:] = 0
    if left % 2:
        c[:, -1, left // 2] &= 15
    return c.reshape(rows, blocks * 16), rng.integers(112, 124, (rows, blocks)).astype(np.uint8)


def _sample(rng, n, most):
    """Places along an axis: its ends, both sides of tiles' borders, others."""
    if n <= most:
        return np.arange(n)
    edges = [i for b in (32, 64, 128, 256, n - n % 32, n - n % 64, n - n % 256, n) for i in (b - 1, b)]
    at = np.concatenate([[0, 1], edges, rng.integers(0, n, most - 20)])
    return np.unique(at[(at >= 0) & (at < n)])


def _layer(rt, rng, n, k, bias):
    c, s = _codes(rng, n, k)
    b = rng.normal(size=n).astype(np.float32) if bias else None
    up = lambda a: DeviceBuffer.from_array(rt, a)  # noqa: E731
    return MXLinear(rt, up(c), up(s), n, k, up(b) if bias else None), c, s, b


def _run(rt, rng, kernel, rows, n, k, dtype, out, bias, most=220):
    print(f"[case] {kernel}: {dtype} -> {out} {rows} x {k} x {n} bias {bias}", flush=True)
    layer, wc, ws, b = _layer(rt, rng, n, k, bias)
    ostride = -(-n // 8) * 8 + 8
    gap = ref.to_bits(np.full((rows, ostride), 777.0), out)
    buf = DeviceBuffer.from_array(rt, gap)
    if dtype == "mxfp4":
        xc, xs = _codes(rng, rows, k)
        args = dict(x=DeviceBuffer.from_array(rt, xc), x_scales=DeviceBuffer.from_array(rt, xs))
    else:
        stride = -(-k // 8) * 8 + 8
        x = ref.to_bits(np.full((rows, stride), np.nan), dtype)
        v = rng.normal(size=(rows, k)) * np.exp(0.5 * rng.normal(size=(rows, k)))
        x[:, :k] = ref.to_bits(v, dtype)
        xc, xs = ref.quantize(ref.from_bits(x[:, :k], dtype))
        args = dict(x=DeviceBuffer.from_array(rt, x), x_stride=stride)
    rt.profile(True)
    rt.profile_reset()
    layer.apply(rows=rows, dtype=dtype, out=buf, out_dtype=out, out_stride=ostride, **args)
    rt.sync()
    taken = rt.profile_read(kernel)[0]
    rt.profile(False)
    rt.profile_reset()
    assert taken == 1, f"{kernel} was not taken"
    got = buf.download(gap.dtype, gap.shape)
    np.testing.assert_array_equal(got[:, n:], gap[:, n:])
    got = ref.from_bits(got[:, :n], out)
    # whole rows, then whole columns, unless one of them is everything
    some = _sample(rng, n, 4 * most)
    parts = [(np.arange(rows), np.arange(n) if n * k < 1e7 else some)]
    if rows > most:
        parts = [(_sample(rng, rows, most), np.arange(n)), (np.arange(rows), some)]
    for r, c in parts:
        w = ref.values(wc[c], ws[c], k)
        want, tol = ref.linear(ref.values(xc[r], xs[r], k), w, None if b is None else b[c], out)
        bad = ~(np.abs(got[np.ix_(r, c)] - want) <= tol)
        assert not bad.any(), (np.argwhere(bad)[:5], int(bad.sum()), got[np.ix_(r, c)][bad][:5], want[bad][:5])
    layer.release()


# k in quads of 256 values: less than one, one, two, three, an odd number, and
# ones whose last quad, step or block is ragged.
DEPTHS = [40, 256, 512, 700, 768, 1280, 1311]


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("tile,rows,n", [(64, 300, 517), (128, 701, 3010), (256, 2907, 2950)])
@pytest.mark.parametrize("k", DEPTHS)
def test_tiles(rt, tile, rows, n, k, out):
    i = TYPES.index(out)
    rng = np.random.default_rng(tile + k + i)
    dtype = ("bf16", "mxfp4", "f16", "f32")[(i + DEPTHS.index(k)) % 4]
    _run(rt, rng, f"eos_mx_product_{tile}_{out}", rows, n, k, dtype, out, (i + k) % 2 == 0)


@pytest.mark.parametrize("tile,rows,n,k,out", [(128, 70001, 300, 40, "f16"), (128, 70001, 300, 700, "f32"),
                                               (256, 200, 65501, 40, "f32"), (256, 200, 65501, 700, "bf16"),
                                               (128, 2048, 10240, 256, "bf16")])
def test_tiles_along_one_axis(rt, tile, rows, n, k, out):
    """One column of tiles, or a row: how they are dealt to the XCDs; three turns of
    tiles of 128 where two of 256 would do."""
    _run(rt, np.random.default_rng(k), f"eos_mx_product_{tile}_{out}", rows, n, k, "bf16", out, True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 3, 4, 5, 9, 16])
@pytest.mark.parametrize("wide", [1, 2, 4])
def test_few_rows(rt, dtype, rows, wide):
    """n on both sides of 16 and 32 outputs for each CU, all of K in one turn of
    the wavefronts or in more."""
    cus = rt.info()["compute_units"]
    n = {1: 16 * cus - 7, 2: 16 * cus + 5, 4: 32 * cus + 9}[wide]
    rng = np.random.default_rng(rows + wide)
    form, most = ("4", 2) if rows <= 4 else ("16", 4)
    for i, k in enumerate((100, 1111, 4400)):
        out = TYPES[(rows + i) % 3]
        _run(rt, rng, f"eos_mx_few_{dtype}_{form}_{min(wide, most)}", rows, n, k, dtype, out, i == 1)


@pytest.mark.parametrize("rows", [1, 4, 16])
@pytest.mark.parametrize("wide", [1, 2])
def test_few_rows_of_codes(rt, rows, wide):
    cus = rt.info()["compute_units"]
    n = {1: 16 * cus - 7, 2: 32 * cus + 9}[wide]
    rng = np.random.default_rng(rows + wide)
    for i, k in enumerate((31, 1111, 4400)):
        _run(rt, rng, f"eos_mx_few_codes_16_{wide}", rows, n, k, "mxfp4", TYPES[i], i == 1)


@pytest.mark.parametrize("rows", [17, 32, 33, 48, 49, 64])
@pytest.mark.parametrize("wide", [1, 2])
def test_rows_laid_out(rt, rows, wide):
    cus = rt.info()["compute_units"]
    n = {1: 16 * cus, 2: 16 * cus + 5}[wide]
    rng = np.random.default_rng(rows + wide)
    for i, k in enumerate((100, 1111, 4400)):
        dtype = ("bf16", "mxfp4", "f32", "f16")[(rows + i) % 4]
        _run(rt, rng, f"eos_mx_few_laid_{-(-rows // 16) * 16}_{wide}", rows, n, k, dtype, TYPES[i], i == 1)
