"""Append and read of one row a sequence (no offsets): the kernels of a decoding
step against the plain restatement, and against the form with offsets."""
import numpy as np
import pytest

import kv_reference as ref
from eos_amd.runtime import DeviceBuffer, Runtime
from test_kv_cache_gpu import FORMATS, World, _case, _io, put_rows

pytestmark = pytest.mark.gpu

SHAPES = [(32, 3, 16), (64, 2, 32), (128, 1, 64), (256, 2, 16)]


def _step(rt, fmt, d, kvh, p, seed):
    """Sequences whose one row stands at the start, inside and at the end of a
    group of 8 and of a page; one without tokens: its row is padding."""
    lengths = np.array([1, 2, 8, 9, 0, p - 1, p, p + 1, 2 * p, 13, 0, 3 * p + 5, 24])
    return World(rt, fmt, kvh, d, p, lengths, np.ones_like(lengths), seed=seed)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d,kvh,p", SHAPES)
def test_single_rows_are_written_to_their_slots_only(rt, fmt, d, kvh, p):
    _case(f"append one row each {fmt} d={d} kvh={kvh} p={p}")
    w = _step(rt, fmt, d, kvh, p, seed=d)
    io = _io(fmt, d // 32)
    stride = 2 * kvh * d + 8
    x = w.rng.normal(size=(w.plan.rows, stride)).astype(np.float32) * 3
    x *= np.exp(w.rng.normal(size=x.shape))
    x[1] = 0.0
    bits = ref.to_rows(x, io)
    dev = DeviceBuffer.from_array(rt, bits)
    assert w.batch.c.d_offsets is None
    w.cache.append(w.batch, dev, dev.view(kvh * d * 2, dev.nbytes - kvh * d * 2), io, stride, stride)
    got = w.pools()
    assert w.cache.status() == 0
    rows = ref.from_rows(bits, io)
    where = list(w.plan.slots())
    assert len(where) == (w.plan.lengths > 0).sum()
    live, slots = [s[0] for s in where], [(s[3], s[4]) for s in where]
    if fmt != "tq4":
        for name, col in (("k", 0), ("v", kvh * d)):
            put_rows(w.pool, name, rows[:, col:col + kvh * d].reshape(-1, kvh, d)[live], slots)
        for name, a in w.pool.arrays().items():
            np.testing.assert_array_equal(got[name], a, err_msg=name)
        return
    # 4 bits: scales within a step of f32, codes equal but at a threshold nearer
    # than the rotation's f32 sums; every other slot as it was.
    old = [np.copy(a) for a in w.pool.views()]
    for name in got:
        setattr(w.pool, name, got[name])
    new = w.pool.views()
    for name, col, codes, scales in (("k", 0, 0, 2), ("v", kvh * d, 1, 3)):
        r = rows[:, col:col + kvh * d].reshape(-1, kvh, d)
        want, ws, near = w.pool.quantize(r)
        for row, _, _, page, slot in where:
            at = (page, slice(None), slot) if name == "k" else (page, slice(None), slot // 8,
                                                                slice(None), slot % 8)
            assert (near[row] | (new[codes][at] == want[row])).all()
            assert near[row].mean() < 0.01 or not r[row].any()
            s = new[scales][page, :, slot]
            assert (np.abs(s - ws[row]) <= 2 * ref.U["f32"] * ws[row]).all()
            new[codes][at] = old[codes][at]
            new[scales][page, :, slot] = old[scales][page, :, slot]
    for a, b in zip(new, old):
        np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("d,kvh,p", SHAPES)
def test_single_rows_read_back(rt, fmt, dtype, d, kvh, p):
    _case(f"read one row each {fmt} -> {dtype} d={d}")
    w = _step(rt, fmt, d, kvh, p, seed=d + 1)
    w.fill()
    size = 4 if dtype == "f32" else 2
    stride = kvh * d + 16
    mark = np.full(w.plan.rows * stride * size, 0x5A, np.uint8)
    outs = [DeviceBuffer.from_array(rt, mark) for _ in range(2)]
    w.cache.read(w.batch, outs[0], outs[1], dtype, stride, stride)
    assert w.cache.status() == 0
    t = {"f16": np.float16, "bf16": np.uint16, "f32": np.float32}[dtype]
    for buf, vals in zip(outs, w.pool.values()):
        raw = buf.download(np.uint8, mark.shape)
        got = raw.view(t).reshape(w.plan.rows, stride)
        touched = np.zeros(got.shape, bool)
        for row, _, _, page, slot in w.plan.slots():
            v = vals[page, :, slot].reshape(-1)
            touched[row, :kvh * d] = True
            y = ref.from_rows(got[row, :kvh * d], dtype).astype(np.float64)
            # A product's and the output's rounding; tq4: the transform's log2(d)
            # additions over the sum of magnitudes, and three factors.
            tol = (ref.U[dtype] + 2 * ref.U["f32"]) * np.abs(v)
            if fmt == "tq4":
                s = (w.pool.k_scale if buf is outs[0] else w.pool.v_scale).reshape(-1, kvh, p)[page, :, slot]
                tol = tol + np.repeat(s, d) * (np.log2(d) + 4) * ref.U["f32"] * np.sqrt(d) * 2.74
            assert (np.abs(y - v) <= tol + 2.0 ** -25).all()
        assert (raw.reshape(w.plan.rows, stride, size)[~touched] == 0x5A).all()


@pytest.mark.parametrize("fmt,io", [("q8", "f16"), ("q8", "bf16"), ("tq4", "f16"), ("tq4", "bf16")])
@pytest.mark.parametrize("d", [32, 64, 128, 256])
def test_a_row_is_the_same_by_either_form(rt, fmt, io, d):
    """Rows written, and read, one a sequence and by row ranges: scales, q8's codes
    and values bit by bit, tq4's codes but at a threshold nearer than the rotation's
    f32 sums, which the two forms add up in their own orders."""
    n, p = (1 << 20) // d, 16
    _case(f"both forms {fmt} {io} d={d} rows={n}")
    rng = np.random.default_rng(d)
    lengths = rng.integers(1, p + 1, n)
    w = World(rt, fmt, 1, d, p, lengths, np.ones(n, int), seed=1, spare=0)
    # (of many sizes in one row, so that f32 sums of them are rounded)
    x = rng.normal(size=(n, 2 * d)) * np.exp(2 * rng.normal(size=(n, 2 * d)))
    bits = ref.to_rows(np.clip(x, -6e4, 6e4).astype(np.float32), io)
    dx = DeviceBuffer.from_array(rt, bits)
    dv = dx.view(d * 2, dx.nbytes - d * 2)
    pools = []
    for one_each in (True, False):
        w.upload()
        batch = w.on_device(w.plan, one_each=one_each)
        assert (batch.c.d_offsets is None) == one_each
        w.cache.append(batch, dx, dv, io, 2 * d, 2 * d)
        pools.append(w.pools())
    for name in pools[0]:
        if fmt == "q8" or "scale" in name:
            np.testing.assert_array_equal(pools[0][name], pools[1][name], err_msg=name)
    if fmt == "tq4":
        codes = []
        for got in pools:
            for name in got:
                setattr(w.pool, name, got[name])
            codes.append(w.pool.views()[:2])
        where = list(w.plan.slots())
        row, page, slot = (np.array([s[i] for s in where]) for i in (0, 3, 4))
        rows = ref.from_rows(bits, io)
        for (a, b), col, at in zip(zip(*codes), (0, d), ((page, 0, slot), (page, 0, slot // 8, slice(None), slot % 8))):
            turned = a[at] != b[at]
            odd = np.nonzero(turned.any(-1))[0]
            assert len(odd) <= n * d * 1e-5
            near = w.pool.quantize(rows[row[odd], col:col + d].reshape(-1, 1, d))[2][:, 0]
            assert (near | ~turned[odd]).all()
            a[at] = b[at]
            np.testing.assert_array_equal(a, b)          # every other slot
    values = []
    for one_each in (True, False):
        out = [DeviceBuffer(rt, n * d * 4) for _ in range(2)]
        w.cache.read(w.on_device(w.plan, one_each=one_each), *out, "f32")
        values.append([o.download(np.uint32, (n, d)) for o in out])
    for a, b in zip(*values):
        np.testing.assert_array_equal(a, b)


def test_caches_of_one_runtime_and_of_several():
    """The kernels are loaded with a runtime's first cache: two caches of one
    runtime, one bound after the first is gone, and two runtimes at once."""
    _case("kernels loaded with the first cache")
    runtimes = [Runtime(0), Runtime(0)]
    try:
        for r in (runtimes[0], runtimes[0], runtimes[1], runtimes[0]):
            worlds = [_step(r, fmt, 64, 2, 16, seed=7) for fmt in ("f16", "tq4")]
            for w in worlds:
                w.fill()
                out = [DeviceBuffer(r, w.plan.rows * 128 * 4) for _ in range(2)]
                w.cache.read(w.batch, *out, "f32")
                assert w.cache.status() == 0
                k = out[0].download(np.float32, (w.plan.rows, 128)).reshape(-1, 2, 64)
                for row, _, _, page, slot in w.plan.slots():
                    want = w.pool.values()[0][page, :, slot]
                    assert np.abs(k[row] - want).max() <= 2.0 ** -18 * np.abs(want).max()
                w.cache.release()
    finally:
        for r in runtimes:
            r.close()


@pytest.mark.parametrize("fmt", FORMATS)
def test_prompts_then_tokens_are_stored_as_given(rt, fmt):
    """Prompts by row ranges, then tokens one a sequence into the same pages and
    half-filled groups: what the cache holds is every row's own."""
    _case(f"stored prompt and tokens {fmt}")
    kvh, d, p, io = 2, 64, 16, _io(fmt)
    prompt, steps = np.array([21, 9]), 20
    total = prompt + steps
    w = World(rt, fmt, kvh, d, p, total, np.array([1, 1]), seed=12, spare=1)
    given = np.zeros((2, w.pool.pages, p, kvh, d), np.float32)      # K and V by page and slot
    there = np.zeros((w.pool.pages, p), bool)

    def call(lengths, n):
        plan = ref.Plan(w.pool, total, n, 12)
        plan.lengths = np.asarray(lengths, np.int32)
        np.testing.assert_array_equal(plan.table, w.plan.table)
        bits = [ref.to_rows(w.rng.normal(size=(plan.rows, kvh * d)).astype(np.float32) * 2, io) for _ in "kv"]
        w.cache.append(w.on_device(plan), *(DeviceBuffer.from_array(rt, b) for b in bits), io)
        for row, _, _, page, slot in plan.slots():
            assert not there[page, slot]
            there[page, slot] = True
            for a, b in zip(given, bits):
                a[page, slot] = ref.from_rows(b[row], io).reshape(kvh, d)
    call(prompt, prompt)
    for i in range(1, steps + 1):
        call(prompt + i, np.array([1, 1]))
    assert w.cache.status() == 0 and there.sum() == total.sum()
    got = w.pools()
    page, slot = np.nonzero(there)
    if fmt != "tq4":
        for name, a in zip("kv", given):
            put_rows(w.pool, name, a[page, slot], list(zip(page, slot)))
        for name, a in w.pool.arrays().items():
            np.testing.assert_array_equal(got[name], a, err_msg=name)
        return
    for name in got:
        setattr(w.pool, name, got[name])
    k, v, ks, vs = w.pool.views()
    for codes, scales, a in ((k.swapaxes(1, 2)[page, slot], ks, given[0]),
                             (v.swapaxes(-1, -2).reshape(w.pool.pages, kvh, p, d).swapaxes(1, 2)[page, slot], vs,
                              given[1])):
        want, s, near = w.pool.quantize(a[page, slot])
        assert (near | (codes == want)).all()
        assert (np.abs(scales.swapaxes(1, 2)[page, slot] - s) <= 2 * ref.U["f32"] * s).all()
