"""Attention where scores, weights and values span wide ranges."""
import numpy as np
import pytest

import kv_bounds
from test_kv_cache_gpu import World, _attend, _case

pytestmark = pytest.mark.gpu

# One row a sequence (splits of the length, and equal shares of a wide table),
# 16 and 128 query rows a workgroup: batch, rows, heads, table columns.
FORMS = {"split": (1, 1, 2, None), "shares": (3, 1, 2, 40000), "rows16": (2, 5, 2, None),
         "rows128": (1, 64, 6, 200)}


def _world(rt, fmt, form, n, seed, rows, d=64):
    batch, r, heads, stride = FORMS[form]
    w = World(rt, fmt, 1, d, 16, np.full(batch, n), np.full(batch, r), seed=seed, shuffle=False,
              stride=stride, spare=0)
    each = -(-n // 16) * 16

    def values(x):
        for b in range(batch):
            rows(x[:, each * b:each * b + n])
        return x
    w.fill(values)
    return w, heads


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("fmt", ["f16", "bf16", "q8", "tq4"])
@pytest.mark.parametrize("sign", [1, -1])
def test_equal_scores_of_any_size(rt, fmt, form, sign):
    """Equal keys whose score is far beyond f32's whole numbers (and no power of
    two, so that its products are rounded): weights as equal as ever."""
    _case(f"far scores {fmt} {form} {sign}")
    size = 2.0 ** (14 if fmt == "f16" else 30)

    def rows(x):
        x[0] = 1.37 * size
        x[1] = 1.5
    w, heads = _world(rt, fmt, form, 90, 1, rows)
    io = "f16" if fmt == "f16" else "bf16"
    q = np.full((w.plan.rows, heads, 64), sign * 1.7 * size, np.float32)
    q64, out, lse = _attend(w, heads, io, q=q)
    k, v = (x[w.plan.table[0, 0], 0, 0] for x in w.pool.values())
    # equal weights of equal values: the output's rounding and the weights' (one
    # 16-bit value, in a bf16 cache 2^-8 off), sums in f32
    tol = (2.0 ** -8 + 2.0 ** -8 + 200 * 2.0 ** -24) * np.abs(v).max()
    assert (np.abs(out - v) <= tol).all(), (float(out.min()), float(out.max()))
    s = float(k @ q64[0, 0]) / 8
    assert (np.abs(lse - s) <= 2.0 ** -14 * abs(s)).all()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("fmt", ["bf16", "q8", "tq4"])
def test_scores_of_any_size_below_zero(rt, fmt, form):
    """Every key's score is -2^108 and less: the weights are as equal as ever."""
    _case(f"low scores {fmt} {form}")

    def rows(x):
        x[0] = -2.0 ** 39                   # (scales of tq4 end at 2^40)
        x[1] = 1.5
    w, heads = _world(rt, fmt, form, 90, 1, rows)
    q = np.full((w.plan.rows, heads, 64), 2.0 ** 66, np.float32)
    q64, out, lse = _attend(w, heads, "bf16", q=q)
    k, v = (x[w.plan.table[0, 0], 0, 0] for x in w.pool.values())
    # equal weights of equal values: the output's rounding, some f32 sums and the
    # weights' roundings (one 16-bit value each, its sum exact in f32)
    tol = (2.0 ** -8 + 2.0 ** -8 + 200 * 2.0 ** -24) * np.abs(v).max()
    assert (np.abs(out - v) <= tol).all(), (float(out.min()), float(out.max()))
    s = float(k @ q64[0, 0]) / 8
    assert np.isfinite(lse).all() and (np.abs(lse - s) <= 2.0 ** -14 * abs(s)).all()


@pytest.mark.parametrize("form", FORMS)
def test_small_weights_of_large_values(rt, form):
    """f16: 16 keys of weight 2^-26 and value 2^15 beside one of weight 1 and
    value 0: what they give is the whole of the row."""
    _case(f"small weights {form}")

    def rows(x):
        x[0] = 0.0
        x[0, 3] = 26 * np.log(2) / 8
        x[1] = 0.0
        x[1, 4:20] = 2.0 ** 15
    w, heads = _world(rt, "f16", form, 90, 2, rows)
    q = np.ones((w.plan.rows, heads, 64), np.float32)
    q64, out, lse = _attend(w, heads, "f16", q=q)
    want, wl, tol, ltol = kv_bounds.attention(w.plan, q64, heads, "f16", 64 ** -0.5)
    # (16 weights' smallest steps are 16 * 2^15 * 2^-31 = 2^-12, every rounding to 11
    # bits 2^-7 * 2^-11 and so little beside it; nothing summed would be 2^-7 off)
    assert want.min() > 2.0 ** -8 and tol.max() < 2.0 ** -11, (want.min(), tol.max())
    assert (np.abs(out - want) <= tol).all(), (float(out.min()), float(want.min()))
    assert (np.abs(lse - wl) <= ltol).all()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("fmt", ["bf16", "q8", "tq4"])
def test_a_factor_of_zero_levels_any_scores(rt, fmt, form):
    """scale 0: equal weights, however large the products q . k are."""
    _case(f"scale 0 {fmt} {form}")

    def rows(x):
        x[0] = np.where(np.arange(x.shape[1]) % 2, 2.0 ** 38, -2.0 ** 38)[:, None, None]
        x[1] = np.where(np.arange(x.shape[1]) % 2, 1.0, 3.0)[:, None, None]
    w, heads = _world(rt, fmt, form, 90, 1, rows)
    q = np.full((w.plan.rows, heads, 64), 2.0 ** 80, np.float32)
    q64, out, lse = _attend(w, heads, "bf16", scale=0.0, q=q)
    want, wl, _, _ = kv_bounds.attention(w.plan, q64, heads, "bf16", 0.0)
    # equal weights: the output's rounding, the weights' and f32 sums
    assert (np.abs(out - want) <= 3 * (2.0 ** -8 + 2.0 ** -8 + 200 * 2.0 ** -24)).all(), (out.min(), out.max())
    assert (np.abs(lse - wl) <= 2.0 ** -16).all()
