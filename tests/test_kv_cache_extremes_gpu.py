"""The paged key-value cache at the ends of its ranges: the most heads, the
longest sequences, the widest strides."""
import numpy as np
import pytest

import kv_bounds
import kv_reference as ref
from eos_amd.kvcache import KVBatch, KVCache
from eos_amd.runtime import DeviceBuffer
from test_kv_cache_gpu import World, _attend, _case, _check, _io

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["f16", "q8"])
@pytest.mark.parametrize("rows,stride", [(1, None), (1, 4000), (3, None), (3, 4000)])
def test_the_most_heads_of_one_key_head(rt, fmt, rows, stride):
    """65,535 heads on one: 4,096 tiles of 16 rows (or 1,536 of 128)."""
    _case(f"65535 heads {fmt} rows={rows} stride={stride}")
    heads, d = 65535, 32
    w = World(rt, fmt, 1, d, 16, np.array([70]), np.array([rows]), seed=3, stride=stride)
    w.fill()
    q64, out, lse = _attend(w, heads, _io(fmt))
    assert w.cache.status() == 0
    some = np.r_[0:40, 16380:16390, 32760:32776, 65520:65535]
    want, wl, tol, ltol = kv_bounds.attention(w.plan, q64[:, some], len(some), _io(fmt), d ** -0.5)
    assert (np.abs(out[:, some] - want) <= tol).all()
    assert (np.abs(lse[:, some] - wl) <= ltol).all()
    assert np.isfinite(out).all() and np.isfinite(lse).all()


@pytest.mark.parametrize("fmt", ["bf16", "q8"])
@pytest.mark.parametrize("batch,rows", [(2, 1), (1, 9), (1, 400)])
def test_the_most_key_heads(rt, fmt, batch, rows):
    """1,024 key-value heads, pages of 256 tokens."""
    _case(f"1024 key heads {fmt} batch={batch} rows={rows}")
    w = World(rt, fmt, 1024, 32, 256, np.full(batch, max(rows, 20)), np.full(batch, rows), seed=4, spare=1)
    w.fill()
    if rows == 400:
        q64, out, lse = _attend(w, 1024, _io(fmt))
        some = [0, 1, 511, 1022, 1023]
        for h in some:                               # one head at a time, as a cache of its own
            pool = ref.Pool(fmt, 1, 32, 256, w.pool.pages)
            for name, a in w.pool.arrays().items():
                setattr(pool, name, np.ascontiguousarray(a.reshape(w.pool.pages, 1024, -1)[:, h]).reshape(-1))
            plan = ref.Plan(pool, w.plan.lengths, w.plan.n, 4)
            plan.table = w.plan.table
            want, wl, tol, ltol = kv_bounds.attention(plan, q64[:, h:h + 1], 1, _io(fmt), 32 ** -0.5)
            assert (np.abs(out[:, h:h + 1] - want) <= tol).all()
            assert (np.abs(lse[:, h:h + 1] - wl) <= ltol).all()
        return
    _check(w, 1024, _io(fmt))


@pytest.mark.parametrize("fmt", ["bf16", "q8"])
def test_the_longest_sequence(rt, fmt):
    """2^30 tokens, every page of the table the same one: the row's position, its
    page and the ends of its splits stand next to the largest."""
    _case(f"2^30 tokens {fmt}")
    d, p, n = 32, 256, 2 ** 30
    w = World(rt, fmt, 1, d, p, np.array([p]), np.array([1]), seed=5, spare=1)
    w.fill()
    page = int(w.plan.table[0, 0])
    table = DeviceBuffer.from_array(rt, np.full(n // p, page, np.int32))
    buf = lambda a: DeviceBuffer.from_array(rt, np.asarray(a, np.int32))  # noqa: E731
    batch = KVBatch(table, n // p, 1, buf([n]))
    io = _io(fmt)
    row = ref.to_rows(w.rng.normal(size=(1, d)).astype(np.float32), io)
    dev = DeviceBuffer.from_array(rt, row)
    w.cache.append(batch, dev, dev, io)
    back = [DeviceBuffer(rt, d * 4) for _ in range(2)]
    w.cache.read(batch, *back, "f32")
    for name, a in w.pools().items():
        setattr(w.pool, name, a)
    k, v = (x[page, 0] for x in w.pool.values())
    for b, x in zip(back, (k, v)):
        np.testing.assert_allclose(b.download(np.float32, d), x[p - 1], rtol=2.0 ** -22)
    q = np.zeros((1, 2, d), np.float32)
    q[0, 1] = w.rng.normal(size=d)
    out, lse = DeviceBuffer(rt, 2 * d * 2), DeviceBuffer(rt, 8)
    bits = ref.to_rows(q, io)
    w.cache.attend(batch, DeviceBuffer.from_array(rt, bits), 2, out, io, lse=lse)
    assert w.cache.status() == 0
    got = ref.from_rows(out.download(np.uint16 if io == "bf16" else np.float16, (2, d)), io)
    s = ref.from_rows(bits, io).astype(np.float64)[0] @ k.T * d ** -0.5
    e = np.exp(s)
    want = (e @ v) / e.sum(1, keepdims=True)
    # A lane adds up 2^30 / (512 * 16) weights one by one in f32, a step's products
    # likewise: 2^17 * 2^-24, beside the weights' and the output's roundings.
    tol = (2 * 2.0 ** -7 + 3 * 2.0 ** -8) * np.abs(v).max()
    assert (np.abs(got - want) <= tol).all()
    assert (np.abs(lse.download(np.float32, 2) - np.log(e.sum(1) * (n // p))) <= 2.0 ** -6).all()


def test_wide_strides(rt):
    """Rows 2^21 elements apart: the last one lies past 2^31 bytes."""
    _case("wide strides")
    stride, rows, d = 1 << 21, 600, 64
    cache = KVCache(rt, "f16", 1, d, 16, 38)
    big = DeviceBuffer(rt, ((rows - 1) * stride + 2 * d) * 2)
    x = np.random.default_rng(6).normal(size=(rows, 2 * d)).astype(np.float16)
    for i in range(rows):
        big.view(2 * i * stride, 4 * d).upload(x[i])
    v = big.view(2 * d, big.nbytes - 2 * d)
    buf = lambda a: DeviceBuffer.from_array(rt, np.asarray(a, np.int32))  # noqa: E731
    batch = KVBatch(buf(np.arange(38)), 38, 1, buf([rows]), buf([0, rows]), rows)
    cache.append(batch, big, v, "f16", stride, stride)
    out = [DeviceBuffer(rt, rows * d * 2) for _ in range(2)]
    cache.read(batch, *out, "f16")
    for b, want in zip(out, (x[:, :d], x[:, d:])):
        np.testing.assert_array_equal(b.download(np.float16, (rows, d)), want)
    # attention over the same rows as queries, its output as far apart
    cache.attend(batch, big, 1, v, "f16", q_stride=stride, out_stride=stride)
    near = DeviceBuffer(rt, rows * d * 2)
    cache.attend(batch, DeviceBuffer.from_array(rt, np.ascontiguousarray(x[:, :d])), 1, near, "f16")
    want = near.download(np.uint16, (rows, d))
    for i in (0, 1, 511, 512, 599):
        np.testing.assert_array_equal(v.view(2 * i * stride, 2 * d).download(np.uint16, d), want[i])
    assert cache.status() == 0
    cache.release()
