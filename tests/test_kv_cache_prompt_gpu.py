"""The kernel of 128 query rows a workgroup in every format and width: which
kernel a call took is read from the launches, so that a test of it stays one."""
import numpy as np
import pytest

import kv_bounds
from test_kv_cache_gpu import FORMATS, World, _attend, _case, _io, put_rows

pytestmark = pytest.mark.gpu


def _launches(rt, call):
    """call()'s result, and the key-value cache kernels that it launched."""
    rt.profile(True)
    rt.profile_reset()
    try:
        out = call()
        rt.sync()
        names = [f"eos_kv_{k}_{f}_{d}" for k in ("split", "prompt", "stream", "stream_join", "join", "join_few")
                 for f in FORMATS for d in (32, 64, 128, 256)]
        return out, {n: rt.profile_read(n)[0] for n in names if rt.profile_read(n)[0]}
    finally:
        rt.profile(False)


def _check(w, heads, kernel, join, window=0, scale=None, pad=16):
    fmt, d, io = w.pool.fmt, w.pool.d, _io(w.pool.fmt, w.pool.d // 32)
    (q64, out, lse), ran = _launches(w.rt, lambda: _attend(w, heads, io, window, scale, pad=pad))
    want = {f"eos_kv_{kernel}_{fmt}_{d}": 1}
    if join:
        want[f"eos_kv_{join}_{fmt}_{d}"] = 1
    assert ran == want
    assert w.cache.status() == 0
    ref_out, ref_lse, tol, ltol = kv_bounds.attention(w.plan, q64, heads, io, d ** -0.5 if scale is None else scale,
                                                      window)
    u = w.plan.used
    over = np.abs(out[:u] - ref_out[:u]) - tol[:u]
    assert not (over > 0).any(), (float(over.max()), float(np.abs(out[:u] - ref_out[:u]).max()))
    fine = np.isfinite(ref_lse[:u])
    np.testing.assert_array_equal(fine, np.isfinite(lse[:u]))
    assert (np.abs(lse[:u][fine] - ref_lse[:u][fine]) <= ltol[:u][fine]).all()
    assert (out[:u][~fine] == 0).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("columns,join", [(1200, "join_few"), (5000, "join")])
@pytest.mark.parametrize("window", [0, 1100])
def test_prompts_in_splits(rt, fmt, d, columns, join, window):
    """Rows behind a prefix, a whole prompt, padding rows, in up to 8 splits and
    in more; with a window (which keeps the splits few) pages in front of it are
    gone and what stands in front of it in a page is NaN."""
    _case(f"prompt {fmt} d={d} columns={columns} window={window}")
    lengths = np.array([1190 if columns < 2000 or window else 2600, 70, 15, 0])
    n = np.array([70, 70, 20, 2])
    kvh, group = 2, 10
    w = World(rt, fmt, kvh, d, 16, lengths, n, seed=d, extra_rows=3, stride=columns // 16)
    w.fill()
    if window:
        first = int(lengths[0] - n[0] - window + 1)               # the first row's first key
        assert 16 < first < 32
        bad = np.full((first, kvh, d), np.nan, np.float32)
        bad[::2] = np.inf
        for name in "kv":
            put_rows(w.pool, name, bad, [(int(w.plan.table[0, i // 16]), i % 16) for i in range(first)])
        w.upload()
        gone = w.plan.table[0, 0]
        w.plan.table[0, 0] = -1
        w.batch = w.on_device(w.plan)
        w.plan.table[0, 0] = gone
    # (162 rows of 10 heads a group: about 400 query rows a sequence)
    assert w.plan.used * group // len(n) >= 384
    few = window > 0 or join == "join_few"
    _check(w, kvh * group, "prompt", "join_few" if few else "join", window)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("window", [0, 1, 40])
def test_prompts_of_one_split(rt, fmt, d, window):
    """Few keys under many rows: no splits, and the rows' outputs are finished by
    the kernel itself."""
    _case(f"prompt in one piece {fmt} d={d} window={window}")
    kvh, group = 4, 16
    w = World(rt, fmt, kvh, d, 16, np.array([230]), np.array([140]), seed=d + 1, extra_rows=1)
    w.fill()
    assert 140 * group // 16 * kvh > 512
    _check(w, kvh * group, "prompt", None, window)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
@pytest.mark.parametrize("columns", [256, 1200])
def test_prompts_of_any_scale(rt, fmt, scale, columns):
    _case(f"prompt scale {fmt} {scale} columns={columns}")
    kvh, group = 4, 16
    w = World(rt, fmt, kvh, 64, 16, np.array([230]), np.array([140]), seed=9, stride=columns // 16)
    w.fill()
    _check(w, kvh * group, "prompt", None if columns == 256 else "join_few", scale=scale)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,columns,kernel,join", [
    (1, 256, "split", None), (1, 1024, "split", "join_few"), (1, 8192, "split", "join"),
    (7, 256, "split", None), (7, 1024, "split", "join_few"), (7, 8192, "split", "join")])
def test_other_kernels_by_the_launches(rt, fmt, rows, columns, kernel, join):
    """16 query rows a workgroup: one split, few, many."""
    _case(f"{kernel} {fmt} rows={rows} columns={columns}")
    w = World(rt, fmt, 2, 64, 16, np.array([250]), np.array([rows]), seed=rows, stride=columns // 16)
    w.fill()
    _check(w, 2, kernel, join, pad=8)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("batch", [2, 256])
def test_equal_shares_by_the_launches(rt, fmt, batch):
    _case(f"stream {fmt} batch={batch}")
    lengths = np.random.default_rng(batch).integers(0, 60, batch)
    lengths[0] = 1000
    w = World(rt, fmt, 1, 64, 16, lengths, np.ones(batch, int), seed=batch, stride=400000 // batch // 16)
    w.fill()
    _check(w, 2, "stream", "stream_join", pad=8)
