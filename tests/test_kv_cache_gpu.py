"""The paged key-value cache on the GPU against its plain restatement
(kv_reference): pools byte for byte, values read back, and attention within
bounds derived from the kernels' roundings."""
import numpy as np
import pytest

import kv_reference as ref
from eos_amd._lib import EosHipError
from eos_amd.kvcache import KVBatch, KVCache, gaussian_codebook
from eos_amd.runtime import DeviceBuffer, Runtime

pytestmark = pytest.mark.gpu


def _case(name):
    print(f"[case] {name}", flush=True)


class World:
    """A pool and a plan on the host and on the device."""

    def __init__(self, rt, fmt, kvh, d, p, lengths, n, seed=0, spare=3, **plan):
        self.rt, self.rng = rt, np.random.default_rng(seed + 1)
        pages = int((-(-np.maximum(lengths, 0) // p)).sum()) + spare
        signs = self.rng.choice([-1.0, 1.0], d)
        self.pool = ref.Pool(fmt, kvh, d, p, pages, seed, gaussian_codebook(), signs)
        self.plan = ref.Plan(self.pool, lengths, n, seed, **plan)
        self.upload()

    def upload(self):
        dev = {k: DeviceBuffer.from_array(self.rt, a) for k, a in self.pool.arrays().items()}
        tq4 = self.pool.fmt == "tq4"
        self.cache = KVCache(self.rt, self.pool.fmt, self.pool.kvh, self.pool.d, self.pool.p,
                             self.pool.pages, codebook=self.pool.codebook if tq4 else None,
                             signs=self.pool.signs if tq4 else None, **dev)
        self.dev = dev
        self.batch = self.on_device(self.plan)

    def on_device(self, plan, one_each=None):
        if one_each is None:
            one_each = plan.rows == len(plan.n) and (plan.n == 1).all()
        buf = lambda a: DeviceBuffer.from_array(self.rt, a)  # noqa: E731
        return KVBatch(buf(plan.table), plan.stride, len(plan.n), buf(plan.lengths),
                       None if one_each else buf(plan.offsets), plan.rows)

    def pools(self):
        return {k: b.download(self.pool.arrays()[k].dtype, self.pool.arrays()[k].shape)
                for k, b in self.dev.items()}

    def fill(self, values=None):
        """Every slot a token: random rows, quantized as the cache does."""
        pool = self.pool
        rows = self.rng.normal(size=(2, pool.pages * pool.p, pool.kvh, pool.d)).astype(np.float32)
        if values is not None:
            rows = values(rows)
        for name, r in zip("kv", rows):
            put_rows(pool, name, r)
        self.upload()


def put_rows(pool, name, rows, where=None):
    """Rows f32 [n, H, d] into the pool's slots (page, slot) `where` (all)."""
    if where is None:
        where = [(i // pool.p, i % pool.p) for i in range(pool.pages * pool.p)]
    page, slot = np.array(where).T
    k, v, ks, vs = pool.views()
    if pool.fmt in ("f16", "bf16"):
        code, scale = ref.to_rows(rows, pool.fmt).view(np.uint16), None
    else:
        code, scale = pool.quantize(rows)[:2]
    if name == "k":
        k[page, :, slot] = code
    else:
        v[page, :, slot // 8, :, slot % 8] = code
    if scale is not None:
        (ks if name == "k" else vs)[page, :, slot] = scale
    pool.put(k, v)


FORMATS = ["f16", "bf16", "q8", "tq4"]


def _io(fmt, i=0):
    return fmt if fmt in ("f16", "bf16") else ("f16", "bf16")[i % 2]


# ------------------------------------------------------------ append, read


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d,kvh,p", [(32, 3, 16), (64, 2, 32), (128, 1, 64), (256, 2, 16)])
def test_append_writes_only_its_slots(rt, fmt, d, kvh, p):
    _case(f"append {fmt} d={d} kvh={kvh} p={p}")
    # whole groups, groups begun and ended in the middle, one token, none,
    # padding rows in front of position 0, rows behind the last sequence
    lengths = np.array([40, 1, 17, 0, 5, 2 * p, p + 3, 9])
    n = np.array([40, 1, 3, 2, 8, 16, p + 3, 0])
    w = World(rt, fmt, kvh, d, p, lengths, n, seed=d, extra_rows=4)
    io = _io(fmt, d // 32)
    stride = 2 * kvh * d + 8
    x = w.rng.normal(size=(w.plan.rows, stride)).astype(np.float32) * 3
    x *= np.exp(w.rng.normal(size=x.shape))
    x[1] = 0.0                                 # a row of zeros
    bits = ref.to_rows(x, io)
    dev = DeviceBuffer.from_array(rt, bits)
    before = w.pools()
    w.cache.append(w.batch, dev, dev.view(kvh * d * 2, dev.nbytes - kvh * d * 2), io, stride, stride)
    got = w.pools()
    assert w.cache.status() == 0
    rows = ref.from_rows(bits, io)
    for name, a in w.pool.arrays().items():
        np.testing.assert_array_equal(before[name], a)
    for name, col in (("k", 0), ("v", kvh * d)):
        r = rows[:, col:col + kvh * d].reshape(-1, kvh, d)
        where = list(w.plan.slots())
        live, slots = [s[0] for s in where], [(s[3], s[4]) for s in where]
        if fmt == "tq4":
            continue
        put_rows(w.pool, name, r[live], slots)
    if fmt != "tq4":
        for name, a in w.pool.arrays().items():
            np.testing.assert_array_equal(got[name], a, err_msg=name)
        return
    # 4 bits: scales within a step of f32, codes equal but where f32 may
    # decide a border the other way; every other slot as it was.
    old = [np.copy(a) for a in w.pool.views()]
    for name in got:
        setattr(w.pool, name, got[name])
    new = w.pool.views()
    for name, col, codes, scales in (("k", 0, 0, 2), ("v", kvh * d, 1, 3)):
        r = rows[:, col:col + kvh * d].reshape(-1, kvh, d)
        want, ws, near = w.pool.quantize(r)
        for row, _, _, page, slot in w.plan.slots():
            at = (page, slice(None), slot) if name == "k" else (page, slice(None), slot // 8,
                                                                slice(None), slot % 8)
            c = new[codes][at]
            assert (near[row] | (c == want[row])).all()
            assert near[row].mean() < 0.01 or not r[row].any()
            s = new[scales][page, :, slot]
            assert (np.abs(s - ws[row]) <= 2 * ref.U["f32"] * ws[row]).all()
            new[codes][at] = old[codes][at]
            new[scales][page, :, slot] = old[scales][page, :, slot]
    for a, b in zip(new, old):
        np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("fmt", ["q8", "tq4"])
def test_append_rows_beyond_the_scales(rt, fmt):
    """NaN, infinities and scales outside [2^-60, 2^40]."""
    _case(f"append edge rows {fmt}")
    d = 64
    w = World(rt, fmt, 1, d, 16, np.array([8]), np.array([8]))
    x = w.rng.normal(size=(8, d)).astype(np.float32)
    x[0, 3] = np.nan
    x[1, 5] = np.inf
    x[2, 7] = -np.inf
    x[3] *= np.float32(2.0 ** -70)
    x[4] *= np.float32(2.0 ** 60)
    x[5] = 0.0
    x[6] *= np.float32(2.0 ** -50)
    dev = DeviceBuffer.from_array(rt, ref.to_bf16(x))
    w.cache.append(w.batch, dev, dev, "bf16")
    out = [DeviceBuffer(rt, 8 * d * 4) for _ in range(2)]
    w.cache.read(w.batch, *out, "f32")
    for b in out:
        y = b.download(np.float32, (8, d))
        assert np.isnan(y[[0, 1, 2, 4]]).all()
        assert (y[[3, 5]] == 0).all()
        for i in (6, 7):
            r = ref.from_bf16(ref.to_bf16(x[i]))
            # q8: half a step of 1 / 127; tq4: a level's half gap (or what lies past the last)
            assert np.abs(y[i] - r).max() <= (np.abs(r).max() / 254 * 1.01 if fmt == "q8"
                                              else np.sqrt((r * r).sum()) * 0.2)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_read_gives_the_values(rt, fmt, dtype):
    d, kvh, p = {"f16": (128, 2, 16), "bf16": (256, 1, 32), "f32": (64, 3, 64)}[dtype]
    _case(f"read {fmt} -> {dtype} d={d}")
    lengths, n = np.array([70, 1, 0, 33, 9]), np.array([70, 1, 3, 5, 0])
    w = World(rt, fmt, kvh, d, p, lengths, n, seed=5, extra_rows=2)
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
            # One product and the output's rounding; tq4: the transform's log2(d)
            # additions over the sum of magnitudes, and three factors.
            tol = (ref.U[dtype] + 2 * ref.U["f32"]) * np.abs(v)
            if fmt == "tq4":
                s = (w.pool.k_scale if buf is outs[0] else w.pool.v_scale).reshape(-1, kvh, p)[page, :, slot]
                tol = tol + np.repeat(s, d) * (np.log2(d) + 4) * ref.U["f32"] * np.sqrt(d) * 2.74
            assert (np.abs(y - v) <= tol + 2.0 ** -25).all()
        assert (raw.reshape(w.plan.rows, stride, size)[~touched] == 0x5A).all()


# --------------------------------------------------------------- attention


def _attend(w, heads, dtype, window=0, scale=None, q=None, plan=None, batch=None, pad=0, qmul=1.0):
    plan, batch = plan or w.plan, batch or w.batch
    d = w.pool.d
    if q is None:
        q = w.rng.normal(size=(plan.rows, heads, d)).astype(np.float32) * np.float32(qmul)
    stride = heads * d + pad
    qrows = np.zeros((plan.rows, stride), np.float32)
    qrows[:, :heads * d] = q.reshape(plan.rows, -1)
    bits = ref.to_rows(qrows, dtype)
    dq = DeviceBuffer.from_array(w.rt, bits)
    mark = np.full((plan.rows, stride), 0x5A5A, np.uint16)
    do = DeviceBuffer.from_array(w.rt, mark)
    dl = DeviceBuffer.from_array(w.rt, np.full((plan.rows, heads), 7.0, np.float32))
    w.cache.attend(batch, dq, heads, do, dtype, scale=scale, window=window, q_stride=stride,
                   out_stride=stride, lse=dl)
    raw = do.download(np.uint16, mark.shape)
    assert (raw[:, heads * d:] == 0x5A5A).all() and (raw[plan.used:] == 0x5A5A).all()
    lse = dl.download(np.float32, (plan.rows, heads))
    assert (lse[plan.used:] == 7.0).all()
    out = raw[:, :heads * d].reshape(plan.rows, heads, d)
    out = ref.from_bf16(out) if dtype == "bf16" else np.ascontiguousarray(out).view(np.float16).astype(np.float32)
    q64 = ref.from_rows(bits, dtype)[:, :heads * d].reshape(plan.rows, heads, d).astype(np.float64)
    return q64, out, lse


def _check(w, heads, dtype, window=0, scale=None, plan=None, batch=None, q=None, pad=0, qmul=1.0):
    plan = plan or w.plan
    q64, out, lse = _attend(w, heads, dtype, window, scale, q, plan, batch, pad, qmul)
    sc = w.pool.d ** -0.5 if scale is None else scale
    want, wl, tol, ltol = ref.attention(plan, w.pool.values(), q64, heads, dtype, sc, window)
    u = plan.used
    over = np.abs(out[:u] - want[:u]) - tol[:u]
    assert not (over > 0).any(), (float(over.max()), float(np.abs(out[:u] - want[:u]).max()))
    fine = np.isfinite(wl[:u])
    np.testing.assert_array_equal(fine, np.isfinite(lse[:u]))
    assert (np.abs(lse[:u][fine] - wl[:u][fine]) <= ltol[:u][fine]).all()
    assert (lse[:u][~fine] == -np.inf).all() and (out[:u][~fine] == 0).all()
    assert w.cache.status() == 0
    return out[:u], want[:u]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d,kvh,group,p", [(32, 2, 3, 16), (64, 3, 1, 32), (128, 2, 4, 64),
                                           (128, 1, 20, 16), (256, 1, 7, 128)])
def test_single_token_rows(rt, fmt, d, kvh, group, p):
    _case(f"decode {fmt} d={d} kvh={kvh} group={group} p={p}")
    lengths = np.array([0, 1, 2, 15, 16, 17, 31, 33, 64, 127, 128, 129, 300, 511])
    w = World(rt, fmt, kvh, d, p, lengths, np.ones_like(lengths), seed=d + group)
    w.fill()
    _check(w, kvh * group, _io(fmt, group), pad=8)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("length,stride", [(1, 200), (700, 11), (4099, 130)])
def test_single_token_split_over_the_length(rt, fmt, length, stride):
    """One sequence, a table far wider than it or just wide enough."""
    _case(f"decode split {fmt} {length}")
    w = World(rt, fmt, 1, 64, 64, np.array([length]), np.array([1]), seed=3, stride=stride)
    w.fill()
    _check(w, 2, _io(fmt), pad=0)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d,kvh,group,p,window", [(32, 2, 3, 16, 0), (64, 3, 1, 32, 0),
                                                  (128, 2, 4, 64, 700), (128, 1, 35, 16, 0),
                                                  (256, 1, 7, 128, 0)])
def test_single_token_rows_of_many_lengths(rt, fmt, d, kvh, group, p, window):
    """A wide page table: the workgroups take equal shares of all keys, which
    begin and end inside sequences."""
    _case(f"decode shares {fmt} d={d} kvh={kvh} group={group} p={p} window={window}")
    lengths = np.array([0, 3000, 1, 129, 0, 4096, 2, 511, 128, 1500, 0])
    w = World(rt, fmt, kvh, d, p, lengths, np.ones_like(lengths), seed=d + group, stride=200000 // p)
    w.fill()
    _check(w, kvh * group, _io(fmt, group), window=window, pad=8)


@pytest.mark.parametrize("fmt", ["q8", "bf16"])
@pytest.mark.parametrize("batch", [2, 65, 256, 257, 300, 512, 513, 1024, 1025])
def test_single_token_rows_of_many_sequences(rt, fmt, batch):
    _case(f"decode batch {batch} {fmt}")
    lengths = np.random.default_rng(batch).integers(0, 40, batch)
    lengths[-1] = 300
    w = World(rt, fmt, 1, 32, 16, lengths, np.ones_like(lengths), seed=batch, stride=40000 // batch)
    w.fill()
    _check(w, 2, _io(fmt))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d,kvh,group,p,window", [(64, 2, 1, 16, 0), (128, 1, 5, 32, 0),
                                                  (32, 1, 16, 16, 19), (256, 1, 3, 64, 70),
                                                  (128, 2, 4, 16, 1), (64, 1, 20, 16, 0)])
@pytest.mark.parametrize("wide", [False, True])
def test_prompt_rows(rt, fmt, d, kvh, group, p, window, wide):
    """Few keys in the page table, and (wide) room for many: the second goes by
    128 query rows a workgroup where a sequence has rows enough, the first by 16."""
    _case(f"prompt {fmt} d={d} group={group} p={p} window={window} wide={wide}")
    lengths = np.array([37, 1, 150, 64, 3, 0, 131])
    n = np.array([37, 1, 5, 33, 4, 0, 20])      # whole prompts, behind a prefix, a padding row
    if wide:
        lengths, n = lengths * 3, n * 3
        lengths[1], n[1] = 1, 2
    w = World(rt, fmt, kvh, d, p, lengths, n, seed=d, extra_rows=3, stride=4096 // p if wide else None)
    w.fill()
    _check(w, kvh * group, _io(fmt, group), window=window, pad=16)


@pytest.mark.parametrize("fmt", FORMATS)
def test_windows_on_single_tokens(rt, fmt):
    _case(f"decode window {fmt}")
    lengths = np.array([1, 5, 64, 200, 333])
    for window in (1, 33, 128, 1000):
        w = World(rt, fmt, 1, 64, 16, lengths, np.ones_like(lengths), seed=window)
        w.fill()
        # pages wholly in front of the window may be gone
        for b, t in enumerate(lengths):
            w.plan.table[b, :max(0, t - window) // 16] = -1
        vals = w.pool.values()
        w.batch = w.on_device(w.plan)
        q64, out, lse = _attend(w, 4, _io(fmt), window)
        assert w.cache.status() == 0
        w.plan.table[w.plan.table < 0] = 0
        want, wl, tol, ltol = ref.attention(w.plan, vals, q64, 4, _io(fmt), 64 ** -0.5, window)
        assert (np.abs(out - want) <= tol).all() and (np.abs(lse - wl) <= ltol).all()


@pytest.mark.parametrize("rows", [False, True])
def test_widest_windows(rt, rows):
    """Windows of any width up to the type's largest, also beside padding rows
    whose positions are negative, as without one."""
    _case(f"widest windows rows={rows}")
    lengths = np.array([3, 40, 90])
    n = np.array([5, 40, 7]) if rows else np.ones(3, int)
    w = World(rt, "bf16", 1, 64, 16, lengths, n, seed=1)
    w.fill()
    q = w.rng.normal(size=(w.plan.rows, 3, 64)).astype(np.float32)
    want = _attend(w, 3, "bf16", q=q)[1:]
    for window in (96, 2 ** 30, 2 ** 31 - 1):
        got = _attend(w, 3, "bf16", window, q=q)[1:]
        np.testing.assert_array_equal(got[0], want[0])
        np.testing.assert_array_equal(got[1], want[1])
    w.cache.status()


@pytest.mark.parametrize("fmt", FORMATS)
def test_peaked_and_growing_scores(rt, fmt):
    """The largest score last, far above the others, and V rows whose size grows
    and shrinks by 2^12: the running reference has to move late."""
    _case(f"peaked {fmt}")
    lengths = np.array([600, 257])
    w = World(rt, fmt, 1, 64, 32, lengths, np.ones_like(lengths), seed=8, shuffle=False)

    def rows(r):
        ramp = np.linspace(0, 1, r.shape[1], dtype=np.float32)[:, None, None]
        r[0] = r[0] * 0.3 + ramp * 6
        r[1] *= np.float32(2) ** np.rint(12 * np.sin(9 * ramp))
        return r
    w.fill(rows)
    q = np.ones((2, 3, 64), np.float32) * np.array([1.0, -1.0, 0.01], np.float32)[None, :, None]
    _check(w, 3, _io(fmt), q=q)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
def test_scales(rt, fmt, scale):
    _case(f"scale {fmt} {scale}")
    lengths = np.array([90, 14])
    w = World(rt, fmt, 2, 32, 16, lengths, np.ones_like(lengths), seed=4)
    w.fill()
    _check(w, 4, _io(fmt), scale=scale)


@pytest.mark.parametrize("fmt", FORMATS)
def test_zero_rows_in_the_cache(rt, fmt):
    """V rows of zeros (scale 0) with the largest weights, and all of them zero."""
    _case(f"zero V {fmt}")
    lengths = np.array([70, 70])
    w = World(rt, fmt, 1, 64, 16, lengths, np.ones_like(lengths), seed=4, shuffle=False)

    def rows(r):
        r[0, 5] = 4.0                # the first sequence's sixth token takes the weight
        r[1, 5] = 0.0
        r[1, 80:] = 0.0              # the second sequence's are all zero
        r[1, :80] *= np.float32(1e-4)
        return r
    w.fill(rows)
    out, _ = _check(w, 2, _io(fmt), q=np.full((2, 2, 64), 0.5, np.float32))
    assert (out[1] == 0).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_what_lies_behind_a_sequence_does_not_reach_it(rt, fmt):
    """Unwritten slots hold NaN: behind the last token, in front of a window,
    and in pages that no table row names."""
    _case(f"NaN slots {fmt}")
    lengths = np.array([37, 3, 130])
    n = np.array([5, 3, 2])
    for stride in (None, 200):                  # 16 and 128 query rows a workgroup
        _nan_slots(rt, fmt, lengths, n, stride)


def _nan_slots(rt, fmt, lengths, n, stride):
    heads = 2 if stride is None else 128
    w = World(rt, fmt, 1, 64, 16, lengths, n, seed=6, stride=stride)
    w.fill()
    clean = [_attend(w, heads, _io(fmt), window, q=np.ones((10, heads, 64), np.float32))[1:] for window in (0, 9)]
    used = set()
    for b, t in enumerate(lengths):
        used |= {(int(w.plan.table[b, i // 16]), i % 16) for i in range(t)}
    free = [(pg, s) for pg in range(w.pool.pages) for s in range(16) if (pg, s) not in used]
    for name in "kv":
        bad = np.full((len(free), 1, 64), np.nan, np.float32)
        bad[::2] = np.inf
        put_rows(w.pool, name, bad, free)
    w.upload()
    q = np.ones((10, heads, 64), np.float32)
    for window, want in zip((0, 9), clean):
        got = _attend(w, heads, _io(fmt), window, q=q)[1:]
        np.testing.assert_array_equal(got[0], want[0])
        np.testing.assert_array_equal(got[1], want[1])
    # ... and what a window has passed
    passed = [(int(w.plan.table[2, i // 16]), i % 16) for i in range(130 - 2 - 9 + 1)]
    for name in "kv":
        put_rows(w.pool, name, np.full((len(passed), 1, 64), np.nan, np.float32), passed)
    w.upload()
    got = _attend(w, heads, _io(fmt), 9, q=q)[1:]
    np.testing.assert_array_equal(got[0], clean[1][0])


@pytest.mark.parametrize("fmt", FORMATS)
def test_a_later_token_does_not_reach_earlier_rows(rt, fmt):
    """NaN and infinities in a token of the prompt: rows before it are as
    without it, rows from it on are NaN or follow the infinity."""
    _case(f"NaN token {fmt}")
    for stride, heads in ((None, 2), (200, 2), (200, 11)):   # 16 and 128 query rows a workgroup
        _nan_token(rt, fmt, stride, heads)


def _nan_token(rt, fmt, stride, heads):
    n = 40
    w = World(rt, fmt, 1, 64, 16, np.array([n]), np.array([n]), seed=6, shuffle=False, spare=0,
              stride=stride)
    w.fill()
    q = w.rng.normal(size=(n, heads, 64)).astype(np.float32)
    clean = _attend(w, heads, _io(fmt), q=q)[1]
    bad = np.ones((1, 1, 64), np.float32)
    bad[0, 0, 7] = np.nan
    put_rows(w.pool, "v", bad, [(1, 4)])          # token 20
    bad[0, 0, 7] = np.inf
    put_rows(w.pool, "v", bad, [(1, 14)])         # token 30
    w.upload()
    got = _attend(w, heads, _io(fmt), q=q)[1]
    vals = w.pool.values()
    q64 = ref.from_rows(ref.to_rows(q, _io(fmt)), _io(fmt)).astype(np.float64)
    with np.errstate(all="ignore"):
        want, _, tol, _ = ref.attention(w.plan, vals, q64, heads, _io(fmt), 64 ** -0.5)
    assert (np.abs(got[:20] - want[:20]) <= tol[:20]).all()
    assert (np.abs(got[:20] - clean[:20]) <= 2 * tol[:20]).all()
    np.testing.assert_array_equal(np.isnan(got[20:]), np.isnan(want[20:]))


def test_offsets_past_32_bits(rt):
    """Pools above 4 GiB, the sequence's pages at their end."""
    _case("large pools")
    kvh, d, p, pages = 8, 128, 64, 33500           # 131 KB a page: 4.4 GB a pool
    cache = KVCache(rt, "f16", kvh, d, p, pages)
    assert cache.k.nbytes > 2 ** 32
    rng = np.random.default_rng(1)
    n = 130
    table = np.array([[pages - 1, 2, pages - 2]], np.int32)
    plan = ref.Plan(ref.Pool("f16", kvh, d, p, 3), [n], [n])
    x = rng.normal(size=(2, n, kvh * d)).astype(np.float16)
    dk, dv = (DeviceBuffer.from_array(rt, a) for a in x)
    buf = lambda a: DeviceBuffer.from_array(rt, a)  # noqa: E731
    batch = KVBatch(buf(table), 3, 1, buf(plan.lengths), buf(plan.offsets), n)
    cache.append(batch, dk, dv, "f16")
    ok, ov = DeviceBuffer(rt, x[0].nbytes), DeviceBuffer(rt, x[0].nbytes)
    cache.read(batch, ok, ov, "f16")
    np.testing.assert_array_equal(ok.download(np.float16, x[0].shape), x[0])
    np.testing.assert_array_equal(ov.download(np.float16, x[0].shape), x[1])
    q = rng.normal(size=(n, kvh, d)).astype(np.float16)
    dq, do = buf(q), DeviceBuffer(rt, q.nbytes)
    cache.attend(batch, dq, kvh, do, "f16")
    out = do.download(np.float16, q.shape).astype(np.float64)
    k, v = (a.reshape(n, kvh, d).astype(np.float64) for a in x)
    s = np.einsum("qhd,khd->hqk", q.astype(np.float64), k) * d ** -0.5
    s[:, ~np.tri(n, dtype=bool)] = -np.inf
    w = np.exp(s - s.max(-1, keepdims=True))
    want = np.einsum("hqk,khd->qhd", w / w.sum(-1, keepdims=True), v)
    # weights and output rounded to f16, scores' f32 sums far below that
    assert np.abs(out - want).max() <= 4 * ref.U["f16"] * np.abs(v).max()
    assert cache.status() == 0
    cache.release()


def test_out_of_range_is_reported_and_masked(rt):
    """Page ids, lengths and offsets out of range set their status bit; sound
    sequences of the same batch are as without them."""
    _case("bad batches")
    for fmt in FORMATS:
        lengths = np.array([40, 40, 40])
        w = World(rt, fmt, 1, 64, 16, lengths, np.array([2, 2, 2]), seed=2)
        w.fill()
        q = w.rng.normal(size=(6, 2, 64)).astype(np.float32)
        clean = _attend(w, 2, _io(fmt), q=q)[1]

        def run(plan):
            return _attend(w, 2, _io(fmt), q=q, plan=plan, batch=w.on_device(plan))[1]
        for what, bit in (("page", 1), ("negative page", 1), ("length", 2), ("negative length", 2),
                          ("offset", 4)):
            plan = ref.Plan(w.pool, lengths, np.array([2, 2, 2]), 2)
            np.testing.assert_array_equal(plan.table, w.plan.table)
            if what == "page":
                plan.table[1, 1] = w.pool.pages
            elif what == "negative page":
                plan.table[1, 0] = -5
            elif what == "length":
                plan.lengths[1] = 1000
            elif what == "negative length":
                plan.lengths[1] = -3
            else:
                plan.offsets[:] = [0, 2, 2000000, 6]
            got = run(plan)
            assert w.cache.status() == bit, (fmt, what)
            np.testing.assert_array_equal(got[:2], clean[:2])
            if what != "offset":
                np.testing.assert_array_equal(got[4:], clean[4:])
            if what == "negative length":
                assert (got[2:4] == 0).all()
            assert w.cache.status() == 0
            # the writes and reads of the same batch: nothing outside is touched
            before = w.pools()
            dev = DeviceBuffer(rt, 6 * 64 * 2)
            batch = w.on_device(plan)
            w.cache.read(batch, dev, dev, _io(fmt))
            w.cache.append(batch, dev, dev, _io(fmt))
            w.cache.status()
            after = w.pools()
            for name in before:
                a, b = before[name].reshape(w.pool.pages, -1), after[name].reshape(w.pool.pages, -1)
                touched = set(np.nonzero((a != b).any(1))[0].tolist())
                assert touched <= {int(plan.table[b, 2]) for b in range(3)} - {-1}
            for name, b in w.dev.items():
                b.upload(before[name])


def test_out_of_range_single_tokens(rt):
    """The same for one row a sequence, with and without equal shares."""
    _case("bad batches, single tokens")
    for stride in (3, 20000):
        lengths = np.array([40, 40, 40])
        w = World(rt, "q8", 1, 64, 16, lengths, np.ones(3, int), seed=2, stride=stride)
        w.fill()
        q = w.rng.normal(size=(3, 2, 64)).astype(np.float32)
        clean = _attend(w, 2, "f16", q=q)[1]
        for what, bit in (("page", 1), ("length", 2), ("negative length", 2)):
            plan = ref.Plan(w.pool, lengths, np.ones(3, int), 2, stride=stride)
            if what == "page":
                plan.table[1, 1] = w.pool.pages
            else:
                plan.lengths[1] = 10 ** 9 if what == "length" else -3
            got = _attend(w, 2, "f16", q=q, plan=plan, batch=w.on_device(plan))[1]
            assert w.cache.status() & bit, (stride, what)
            np.testing.assert_array_equal(got[[0, 2]], clean[[0, 2]])
            if what == "negative length":
                assert (got[1] == 0).all()


def test_call_refusals(rt):
    _case("refusals")
    w = World(rt, "f16", 2, 64, 16, np.array([8, 8]), np.array([1, 1]))
    buf = DeviceBuffer(rt, 1 << 16)
    ok = dict(heads=4, out=buf, dtype="f16")
    w.cache.attend(w.batch, buf, **ok)
    for kw, what in ((dict(heads=3), "multiple of kv_heads"), (dict(dtype="bf16"), "holds f16"),
                     (dict(q_stride=4 * 64 + 4), "stride"), (dict(out_stride=64), "stride"),
                     (dict(window=-1), "window"), (dict(scale=float("nan")), "scale"),
                     (dict(out=buf.view(8, 4096)), "aligned")):
        with pytest.raises(EosHipError, match=what):
            w.cache.attend(w.batch, buf, **(ok | kw))
    with pytest.raises(EosHipError, match="f16 .0. or bf16"):
        w.cache.append(w.batch, buf, buf, "f32")
    with pytest.raises(EosHipError, match="holds f16"):
        w.cache.append(w.batch, buf, buf, "bf16")
    with pytest.raises(EosHipError, match="stride"):
        w.cache.read(w.batch, buf, buf, "f16", k_stride=132)
    with pytest.raises(ValueError, match="smaller"):
        w.cache.append(w.batch, DeviceBuffer(rt, 64), buf, "f16")
    batch = KVBatch(buf, 1, 2, buf)
    batch.c.rows = 3
    with pytest.raises(EosHipError, match="one row"):
        w.cache.attend(batch, buf, **ok)
    other = Runtime(0)
    try:
        w.cache.rt = other
        with pytest.raises(EosHipError, match="another runtime"):
            w.cache.attend(w.batch, buf, **ok)
    finally:
        w.cache.rt = rt
        other.close()
    empty = KVBatch(buf, 1, 0, buf)
    w.cache.attend(empty, buf, **ok)
    w.cache.append(empty, buf, buf, "f16")
    assert w.cache.status() == 0


# ------------------------------------------------------------ run together


@pytest.mark.parametrize("fmt", FORMATS)
def test_prompt_then_tokens(rt, fmt):
    """Two sequences as a model runs them: prompts appended and attended, then
    tokens one at a time, each call seeing what the earlier ones wrote; the
    cache's values against the rows, attention against those values."""
    _case(f"prompt then tokens {fmt}")
    kvh, d, p, heads, io = 2, 64, 16, 6, _io(fmt)
    prompt, steps = np.array([21, 9]), 20
    total = prompt + steps
    w = World(rt, fmt, kvh, d, p, total, np.array([1, 1]), seed=11, spare=1)
    table = w.plan.table
    outs, plans, qs = [], [], []
    width = (heads + 2 * kvh) * d

    def call(lengths, n):
        plan = ref.Plan(w.pool, total, n, 11)
        plan.lengths = np.asarray(lengths, np.int32)
        np.testing.assert_array_equal(plan.table, table)
        batch = w.on_device(plan)
        x = ref.to_rows(w.rng.normal(size=(plan.rows, width)).astype(np.float32), io)
        dev = DeviceBuffer.from_array(rt, x)     # one projection's output: q, k, v side by side
        k = dev.view(heads * d * 2, dev.nbytes - heads * d * 2)
        v = dev.view((heads + kvh) * d * 2, dev.nbytes - (heads + kvh) * d * 2)
        out = DeviceBuffer(rt, plan.rows * heads * d * 2)
        w.cache.append(batch, k, v, io, width, width)
        w.cache.attend(batch, dev, heads, out, io, q_stride=width)
        plans.append(plan)
        qs.append(ref.from_rows(x, io)[:, :heads * d].reshape(-1, heads, d).astype(np.float64))
        outs.append(out)
    call(prompt, prompt)
    for i in range(1, steps + 1):
        call(prompt + i, np.array([1, 1]))
    assert w.cache.status() == 0
    for name, a in w.pools().items():
        setattr(w.pool, name, a)
    vals = w.pool.values()
    for plan, q, out in zip(plans, qs, outs):
        raw = out.download(np.uint16, (plan.rows, heads, d))
        got = ref.from_bf16(raw) if io == "bf16" else raw.view(np.float16).astype(np.float32)
        want, _, tol, _ = ref.attention(plan, vals, q, heads, io, d ** -0.5)
        assert (np.abs(got - want) <= tol).all()


def test_two_runtimes_on_one_cache(rt):
    """A second stream binds the same pools; both attend at once, several
    times, with the results of one alone."""
    _case("two runtimes")
    lengths = np.array([700, 300, 900])
    w = World(rt, "q8", 2, 128, 32, lengths, np.ones_like(lengths), seed=9)
    w.fill()
    q = w.rng.normal(size=(3, 8, 128)).astype(np.float32)
    want = _attend(w, 8, "f16", q=q)[1]
    other = Runtime(0)
    again = KVCache(other, "q8", 2, 128, 32, w.pool.pages, **w.dev)
    dq = DeviceBuffer.from_array(rt, ref.to_rows(q, "f16"))
    outs = [DeviceBuffer(rt, 3 * 8 * 128 * 2) for _ in range(8)]
    rt.sync()
    for i, o in enumerate(outs):
        (w.cache if i % 2 else again).attend(w.batch, dq, 8, o, "f16")
    other.sync()
    for o in outs:
        np.testing.assert_array_equal(o.download(np.float16, (3, 8, 128)).astype(np.float32), want)
    again.release()
    other.close()
