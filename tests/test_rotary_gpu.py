"""Rotary positions on the GPU against the formula in 64 bits."""
import numpy as np
import pytest

from eos_amd._lib import EosHipError
from eos_amd.kvcache import KVBatch
from eos_amd.rotary import Rotary, frequencies
from eos_amd.runtime import DeviceBuffer, Runtime
from mx_reference import STEP, U, from_bits, np_dtype, to_bits

pytestmark = pytest.mark.gpu


def _case(name):
    print(f"[case] {name}", flush=True)


def _turned(x, pos, freq, layout, factor, inverse=False):
    """x f64 [rows, heads, d] -> (turned, bound before the last rounding): an angle
    is off by 2^-51 of itself (f64) and by f32's roundings of what is left within
    a turn, a function by 4 steps, and three products and a sum follow."""
    r = 2 * len(freq)
    a, b = (slice(0, r, 2), slice(1, r, 2)) if layout == "pairs" else (slice(0, r // 2), slice(r // 2, r))
    ang = pos[:, None].astype(np.longdouble) * freq.astype(np.longdouble)
    if inverse:
        ang = -ang
    c, s = (f(ang).astype(np.float64)[:, None] * factor for f in (np.cos, np.sin))
    y, e = x.copy(), np.zeros_like(x)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    size = abs(factor) * (np.abs(x[..., a]) + np.abs(x[..., b]))
    e[..., a] = e[..., b] = size * (np.abs(ang).astype(np.float64)[:, None] * 2.0 ** -51 + 20 * 2.0 ** -24)
    return y, e


def _check(got, want, e, dtype):
    tol = e + U[dtype] * (np.abs(want) + e) + np.where(e > 0, STEP[dtype] / 2, 0)
    bad = ~(np.abs(got - want) <= tol * (e > 0))
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5])


class Rows:
    """Packed rows q | k | v of one projection, and arrays of their own."""

    def __init__(self, rt, rng, rows, heads, kvh, d, dtype):
        self.shape = (rows, heads, kvh, d)
        self.dtype, self.width = dtype, (heads + 2 * kvh) * d + 8
        self.bits = to_bits(rng.normal(size=(rows, self.width)), dtype)
        self.size = self.bits.itemsize
        self.dev = DeviceBuffer.from_array(rt, self.bits)

    def part(self, dev, which):
        _, heads, _, d = self.shape
        at = (heads * d if which == "k" else 0) * self.size
        return dev.view(at, dev.nbytes - at)

    def values(self, bits, which):
        rows, heads, kvh, d = self.shape
        at, n = (heads * d, kvh) if which == "k" else (0, heads)
        return from_bits(bits[:, at:at + n * d], self.dtype).reshape(rows, n, d)


# (head_dim, rotary_dim): whole, parts, odd parts
DIMS = [(64, 64), (128, 128), (128, 32), (80, 80), (96, 48), (256, 256), (128, 122), (40, 10), (8, 2),
        (1024, 1024), (512, 256), (32, 4)]


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("layout", ["pairs", "halves"])
@pytest.mark.parametrize("d,r", DIMS)
def test_batches_of_ragged_sequences(rt, dtype, layout, d, r):
    """Rows at the ends of sequences of every kind, padding and rows behind the
    last sequence left alone, out of place and in place."""
    _case(f"{dtype} {layout} {d}/{r}")
    rng = np.random.default_rng(d + r)
    n = np.array([1, 0, 5, 3, 17, 2, 1])
    lens = np.array([1, 9, 5, 40000, 1000003, 1, 1 << 29])  # the sixth: one row of padding
    off = np.concatenate([[0], n.cumsum()])
    rows, heads, kvh = int(off[-1]) + 4, 3, 1
    pos = np.full(rows, -1, np.int64)
    for b in range(len(n)):
        pos[off[b]:off[b + 1]] = lens[b] - n[b] + np.arange(n[b])
    x = Rows(rt, rng, rows, heads, kvh, d, dtype)
    freq, factor = frequencies(r, scaling="linear", stretch=2)[0], 1.25
    rot = Rotary(rt, d, freq, layout, factor)
    i32 = lambda a: DeviceBuffer.from_array(rt, np.asarray(a, np.int32))  # noqa: E731
    batch = KVBatch(None, 0, len(n), i32(lens), i32(off), rows)
    out = {w: DeviceBuffer.from_array(rt, to_bits(np.full((rows, m * d + 8), 776.0), dtype))
           for w, m in (("q", heads), ("k", kvh))}
    for inverse in (False, True):
        rot.apply(batch, dtype, x.part(x.dev, "q"), heads, x.part(x.dev, "k"), kvh, out["q"],
                  out["k"], x.width, x.width, heads * d + 8, kvh * d + 8, inverse)
        for w, m in (("q", heads), ("k", kvh)):
            got = from_bits(out[w].download(np_dtype(dtype), (rows, m * d + 8)), dtype)
            assert (got[:, m * d:] == 776).all() and (got[pos < 0] == 776).all()
            live = pos >= 0
            want, e = _turned(x.values(x.bits, w)[live], pos[live], freq, layout, factor, inverse)
            _check(got[live, :m * d].reshape(want.shape), want, e, dtype)
    # in place: what is neither query nor key stays
    rot.apply(batch, dtype, x.part(x.dev, "q"), heads, x.part(x.dev, "k"), kvh, q_stride=x.width,
              k_stride=x.width)
    got = x.dev.download(np_dtype(dtype), x.bits.shape)
    np.testing.assert_array_equal(got[:, (heads + kvh) * d:], x.bits[:, (heads + kvh) * d:])
    np.testing.assert_array_equal(got[pos < 0], x.bits[pos < 0])
    for w in "qk":
        want, e = _turned(x.values(x.bits, w)[live], pos[live], freq, layout, factor)
        _check(x.values(got, w)[live], want, e, dtype)


@pytest.mark.parametrize("layout", ["pairs", "halves"])
@pytest.mark.parametrize("rows", [1, 3, 64, 1500, 9000])
def test_positions_given(rt, layout, rows):
    """Positions in any order, twice the same, negative; queries or keys alone."""
    _case(f"positions {layout} {rows}")
    rng = np.random.default_rng(rows)
    d, heads = 64, 2
    pos = rng.integers(0, 200000, rows)
    pos[rng.random(rows) < 0.1] = -1
    if rows > 2:
        pos[1] = pos[2] = 77
    x = Rows(rt, rng, rows, heads, heads, d, "f32")
    rot = Rotary(rt, d, frequencies(d)[0], layout)
    where = (DeviceBuffer.from_array(rt, pos.astype(np.int32)), rows)
    live = pos >= 0
    got = x.bits
    for w in "qk":
        rot.apply(where, "f32", **({"q": x.part(x.dev, "q"), "heads": heads, "q_stride": x.width}
                                   if w == "q" else
                                   {"k": x.part(x.dev, "k"), "kv_heads": heads, "k_stride": x.width}))
        before, got = got, x.dev.download(np.float32, x.bits.shape)
        want, e = _turned(x.values(x.bits, w)[live], pos[live], frequencies(d)[0], layout, 1.0)
        _check(x.values(got, w)[live], want, e, "f32")
        np.testing.assert_array_equal(got[~live], x.bits[~live])
        other = "k" if w == "q" else "q"
        np.testing.assert_array_equal(x.values(got, other), x.values(before, other))


@pytest.mark.parametrize("batch", [1, 2, 63, 64, 65, 130, 4100])
def test_rows_find_their_sequences(rt, batch):
    """Batches around the search's widths, with empty sequences and long ones."""
    _case(f"batch {batch}")
    rng = np.random.default_rng(batch)
    n = rng.integers(0, 4, batch)
    n[rng.integers(0, batch)] = 60
    lens = n + rng.integers(0, 1000, batch)
    off = np.concatenate([[0], n.cumsum()])
    rows, d = int(off[-1]), 8
    pos = np.concatenate([lens[b] - n[b] + np.arange(n[b]) for b in range(batch)])
    x = Rows(rt, rng, rows, 1, 1, d, "f32")
    freq = frequencies(d)[0]
    i32 = lambda a: DeviceBuffer.from_array(rt, np.asarray(a, np.int32))  # noqa: E731
    Rotary(rt, d, freq).apply(KVBatch(None, 0, batch, i32(lens), i32(off), rows), "f32",
                              x.part(x.dev, "q"), 1, q_stride=x.width)
    want, e = _turned(x.values(x.bits, "q"), pos, freq, "halves", 1.0)
    _check(x.values(x.dev.download(np.float32, x.bits.shape), "q"), want, e, "f32")


def test_decoding_form_and_damaged_batches(rt):
    """One row a sequence without offsets; offsets and lengths out of range
    touch nothing."""
    rng = np.random.default_rng(1)
    d, rows = 32, 5
    x = Rows(rt, rng, rows, 2, 1, d, "bf16")
    freq = frequencies(d)[0]
    rot = Rotary(rt, d, freq)
    i32 = lambda a: DeviceBuffer.from_array(rt, np.asarray(a, np.int32))  # noqa: E731
    q = x.part(x.dev, "q")
    rot.apply(KVBatch(None, 0, 5, i32([0, 3, -2, -7, -9]), i32([0, -3, 9, 2, 2, 1000]), 5), "bf16", q,
              2, q_stride=x.width)
    lens = np.array([7, 0, 1, -5, 100000])
    rot.apply(KVBatch(None, 0, 5, i32(lens)), "bf16", q, 2, q_stride=x.width)
    got = x.dev.download(np.uint16, x.bits.shape)
    live = lens > 0
    np.testing.assert_array_equal(got[~live], x.bits[~live])
    want, e = _turned(x.values(x.bits, "q")[live], lens[live] - 1, freq, "halves", 1.0)
    _check(x.values(got, "q")[live], want, e, "bf16")


def test_inverse_is_the_gradient(rt):
    """<g, turned(x)> has the gradient inverse(g); also by differences."""
    rng = np.random.default_rng(9)
    d, r, rows, heads = 16, 12, 6, 2
    for layout in ("pairs", "halves"):
        rot = Rotary(rt, d, frequencies(r)[0], layout, 1.5)
        pos = DeviceBuffer.from_array(rt, np.array([0, 1, 5, 100, 7, 3], np.int32))

        def run(a, inverse=False):
            b = DeviceBuffer.from_array(rt, a.astype(np.float32))
            rot.apply((pos, rows), "f32", b, heads, inverse=inverse)
            return b.download(np.float32, a.shape).astype(np.float64)

        x, g = rng.normal(size=(2, rows, heads * d)).astype(np.float32)
        grad = run(g, True)
        for _ in range(20):
            v = rng.normal(size=x.shape).astype(np.float32)
            # linear: a difference is exact but for the f32 roundings
            got = (g.astype(np.float64) * (run(x + v) - run(x))).sum()
            size = (np.abs(g) * 1.5 * 4 * (np.abs(x) + np.abs(v))).sum() * 2
            assert abs(got - (grad * v).sum()) <= size * 2.0 ** -18


def test_large_strides_and_refusals(rt):
    rng = np.random.default_rng(3)
    d = 64
    freq = frequencies(d)[0]
    rot = Rotary(rt, d, freq)
    # rows 64 MB apart: offsets beyond 32 bits
    stride, rows = 1 << 24, 70
    far = DeviceBuffer(rt, ((rows - 1) * stride + d) * 4)
    x = rng.normal(size=(rows, d)).astype(np.float32)
    for i in range(rows):
        far.view(i * stride * 4, d * 4).upload(x[i])
    pos = np.arange(rows) * 11
    where = (DeviceBuffer.from_array(rt, pos.astype(np.int32)), rows)
    rot.apply(where, "f32", far, 1, q_stride=stride)
    got = np.stack([far.view(i * stride * 4, d * 4).download(np.float32, (d,)) for i in range(rows)])
    want, e = _turned(x.astype(np.float64)[:, None], pos, freq, "halves", 1.0)
    _check(got.astype(np.float64)[:, None], want, e, "f32")
    far.free()
    buf = DeviceBuffer(rt, 1 << 16)
    for kw, what in ((dict(q_stride=60), "stride of q"), (dict(q_stride=68), "stride of q"),
                     (dict(q_out=buf, q_out_stride=8), "stride of q_out"),
                     (dict(q_out=buf, q_stride=64, q_out_stride=72), "in place"),
                     (dict(q=buf.view(8, 4096)), "16-byte"), (dict(heads=-1), "heads")):
        with pytest.raises(EosHipError, match=what):
            rot.apply((buf, 2), "f32", **(dict(q=buf, heads=1) | kw))
    with pytest.raises(EosHipError, match="heads"):
        rot.apply((buf, 2), "f32")
    with pytest.raises(EosHipError, match="one row"):
        rot.apply(KVBatch(None, 0, 2, buf, None, 3), "f32", buf, 1)
    with pytest.raises(ValueError, match="dtype"):
        rot.apply((buf, 2), "i8", buf, 1)
    with pytest.raises(ValueError, match="smaller"):
        rot.apply((buf, 2), "f32", buf.view(0, 508), 1)
    with Runtime(0) as other:
        mine = Rotary(other, d, freq)
        mine.rt = rt
        with pytest.raises(EosHipError, match="another runtime"):
            mine.apply((buf, 2), "f32", buf, 1)
        mine.rt = other
        mine.release()
