"""Attention beside pages that are not there."""
import numpy as np
import pytest

import kv_reference as ref
from test_kv_cache_gpu import World, _attend, _case, put_rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("stride,heads", [(None, 2), (200, 2)])
def test_odd_values_beside_a_missing_page(rt, fmt, d, stride, heads):
    """A page id out of range masks its own tokens; NaN and infinity in the
    valid pages around it still reach the rows that attend them (by 16 and by
    128 query rows a workgroup)."""
    _case(f"odd values beside a missing page {fmt} d={d} stride={stride}")
    n, rows = 192, 64
    w = World(rt, fmt, 1, d, 16, np.array([n]), np.array([rows]), seed=3, shuffle=False, stride=stride)
    w.fill()
    vals = [x[:, 0].reshape(-1, d)[:n].copy() for x in w.pool.values()]
    bad = np.ones((1, 1, d), np.float32)
    bad[0, 0, 7], bad[0, 0, 9] = np.nan, np.inf
    put_rows(w.pool, "v", bad, [(0, 5)])
    bad[0, 0, 7], bad[0, 0, 9] = 1.0, np.inf
    bad[0, 0, 11] = -np.inf
    put_rows(w.pool, "v", bad, [(2, 8)])
    w.upload()
    w.plan.table[0, 1] = w.pool.pages                  # tokens 16 .. 31
    q = w.rng.normal(size=(rows, heads, d)).astype(np.float32)
    q64, out, _ = _attend(w, heads, fmt, q=q, batch=w.on_device(w.plan))
    assert w.cache.status() == 1
    assert np.isnan(out[:, :, 7]).all()
    assert (out[:, :, 9] == np.inf).all() and (out[:, :, 11] == -np.inf).all()
    # every other dimension as the other keys give it
    k, v = vals
    v[5] = v[40] = 1.0
    fine = [i for i in range(d) if i not in (7, 9, 11)]
    for i in range(rows):
        see = np.r_[0:16, 32:n - rows + i + 1]
        s = (q64[i] @ k[see].T) * d ** -0.5
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        # weights and output rounded to 16 bits, sums and scores far below
        tol = 2.5 * ref.U[fmt] * (p @ np.abs(v[see])) + 2.0 ** -12 * p.max() + 2.0 ** -20
        assert (np.abs(out[i] - p @ v[see]) <= tol)[:, fine].all()
