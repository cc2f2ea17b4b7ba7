"""Attention over quantized caches whose V scales differ by many powers of two:
a row is as exact as the tokens that it attends, and weighs, let it be."""
import numpy as np
import pytest

import kv_bounds
from test_kv_cache_gpu import World, _attend, _case, _io

pytestmark = pytest.mark.gpu


def _check(w, heads, q):
    io = _io(w.pool.fmt)
    q64, out, lse = _attend(w, heads, io, q=q)
    assert w.cache.status() == 0
    want, wl, tol, ltol = kv_bounds.attention(w.plan, q64, heads, io, w.pool.d ** -0.5)
    over = np.abs(out - want) - tol
    at = np.unravel_index(over.argmax(), over.shape)
    assert over.max() <= 0, (at, float(out[at]), float(want[at]), float(tol[at]))
    assert (np.abs(lse - wl) <= ltol).all()


@pytest.mark.parametrize("fmt", ["q8", "tq4"])
@pytest.mark.parametrize("power", [12, 16, 24, 38])
@pytest.mark.parametrize("wide", [False, True])
def test_a_later_token_of_any_size_does_not_reach_earlier_rows(rt, fmt, power, wide):
    """A prompt whose token 44 has values 2^power times the others', by 16 and
    (wide: 384 query rows, room for many keys) by 128 query rows a workgroup."""
    _case(f"large token {fmt} 2^{power} wide={wide}")
    n, heads = 64, 6 if wide else 2
    w = World(rt, fmt, 1, 64, 16, np.array([n]), np.array([n]), seed=power, shuffle=False,
              stride=200 if wide else None)

    def rows(r):
        r[1, 44] *= np.float32(2.0 ** power)
        return r
    w.fill(rows)
    q = w.rng.normal(size=(n, heads, 64)).astype(np.float32)
    q64, out, lse = _attend(w, heads, "bf16", q=q)
    want, wl, tol, ltol = kv_bounds.attention(w.plan, q64, heads, "bf16", 64 ** -0.5)
    assert (np.abs(out[:44] - want[:44]) <= tol[:44]).all(), float((np.abs(out - want) / tol)[:44].max())
    assert (np.abs(out[44:] - want[44:]) <= tol[44:]).all()
    assert (np.abs(lse - wl) <= ltol).all()


@pytest.mark.parametrize("fmt", ["q8", "tq4"])
@pytest.mark.parametrize("power", [16, 24, 34])
@pytest.mark.parametrize("batch", [1, 3])
def test_a_large_token_of_no_weight_takes_nothing_from_the_others(rt, fmt, power, batch):
    """Single tokens: one key with a weight of about 2^-2 power below the others'
    and values 2^power times theirs (3: in equal shares of a wide table)."""
    _case(f"large light token {fmt} 2^{power} batch={batch}")
    w = World(rt, fmt, 1, 64, 16, np.full(batch, 200), np.ones(batch, int), seed=power, shuffle=False,
              stride=None if batch == 1 else 40000)

    def rows(r):
        for b in range(batch):
            r[0, 208 * b + 40] = np.float32(-2 * power * np.log(2) / 8)   # q . k / 8, q = 1
            r[1, 208 * b + 40] *= np.float32(2.0 ** power)
        return r
    w.fill(rows)
    q = np.ones((batch, 2, 64), np.float32)
    _check(w, 2, q)


@pytest.mark.parametrize("fmt", ["q8", "tq4"])
@pytest.mark.parametrize("zeros", [32, 128, 1500])
@pytest.mark.parametrize("rows,wide", [(1, False), (8, False), (64, True)])
def test_zero_rows_keep_their_weight_beside_large_ones(rt, fmt, zeros, rows, wide):
    """V rows of zeros first (within a wavefront's keys, and a split's), then
    rows of 2^30 and more: the zeros count in the weights' sum."""
    _case(f"zeros then large {fmt} {zeros} rows={rows} wide={wide}")
    n, heads = zeros + 100, 6 if wide else 2
    w = World(rt, fmt, 1, 64, 16, np.array([n]), np.array([rows]), seed=zeros, shuffle=False,
              stride=200 if wide else None)

    def values(r):
        r[1, :zeros] = 0.0
        r[1, zeros:] *= np.float32(2.0 ** 36)
        return r
    w.fill(values)
    q = w.rng.normal(size=(rows, heads, 64)).astype(np.float32)
    q64, out, lse = _attend(w, heads, "bf16", q=q)
    want, wl, tol, ltol = kv_bounds.attention(w.plan, q64, heads, "bf16", 64 ** -0.5)
    assert (np.abs(out - want) <= tol).all(), float((np.abs(out - want) / np.maximum(tol, 1e-30)).max())
    assert (np.abs(lse - wl) <= ltol).all(), float(np.abs(lse - wl).max())


@pytest.mark.parametrize("fmt", ["f16", "bf16", "q8", "tq4"])
@pytest.mark.parametrize("rows,wide", [(1, False), (8, False), (64, True)])
def test_values_that_grow_and_shrink(rt, fmt, rows, wide):
    """Scores that rise, V rows that swell and shrink by 2^12: a row's bound is
    what its own weights times values leave."""
    _case(f"growing {fmt} rows={rows} wide={wide}")
    n, heads = 600, 6
    w = World(rt, fmt, 1, 64, 16, np.array([n]), np.array([rows]), seed=8, shuffle=False,
              stride=200 if wide else None)

    def values(r):
        ramp = np.linspace(0, 1, r.shape[1], dtype=np.float32)[:, None, None]
        r[0] = r[0] * 0.3 + ramp * 6
        r[1] *= np.float32(2) ** np.rint(12 * np.sin(9 * ramp))
        return r
    w.fill(values)
    q = np.ones((rows, heads, 64), np.float32) * np.array([1.0, -1.0, 0.01, 0.3, -0.3, 0.0], np.float32)[:, None]
    q64, out, lse = _attend(w, heads, "bf16" if fmt == "bf16" else "f16", q=q)
    want, wl, tol, ltol = kv_bounds.attention(w.plan, q64, heads, "bf16" if fmt == "bf16" else "f16", 64 ** -0.5)
    assert (np.abs(out - want) <= tol).all(), float((np.abs(out - want) / tol).max())
    assert (np.abs(lse - wl) <= ltol).all()
