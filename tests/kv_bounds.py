"""Attention over the paged cache in 64 bits with a bound that a row's own
weights give: what a row does not attend, or hardly weighs, allows it nothing.

A weight times its V scale (the weight alone in a cache without scales) is
rounded to the matrix operand's 16 bits: by u = 2^-11 (f16) or 2^-8 (bf16) of
itself, in f16 at least by half the smallest step, 2^-25, where the largest
product of the row that a reference was taken from is at least 2^6."""
import numpy as np

import kv_reference as ref

U = ref.U


def attention(plan, q, heads, dtype, scale, window=0):
    """q f64 [rows, heads, d] -> (out, lse, bound on out's error, on lse's)."""
    pool = plan.pool
    d, group = pool.d, heads // pool.kvh
    tq4, quant = pool.fmt == "tq4", pool.fmt in ("q8", "tq4")
    with np.errstate(all="ignore"):
        vals = pool.values()
    back = ref.hadamard(d) / np.sqrt(d) if tq4 else np.eye(d)
    sg = pool.signs if tq4 else np.ones(d)
    up = U["bf16" if pool.fmt == "bf16" else "f16"]
    # tq4's rotated query (log2(d) f32 additions) is held in two f16 terms.
    uq = U["f16"] ** 2 + (np.log2(d) + 2) * U["f32"] if tq4 else 0.0
    out = np.zeros((plan.rows, heads, d))
    lse = np.full((plan.rows, heads), -np.inf)
    tol, ltol = np.zeros_like(out), np.zeros_like(lse)
    for b in range(len(plan.n)):
        k, v = plan.sequence(b, vals[0]), plan.sequence(b, vals[1])
        ka, va = np.abs((k * sg) @ back), np.abs((v * sg) @ back)
        for i in range(plan.n[b]):
            pos = int(plan.lengths[b]) - int(plan.n[b]) + i
            if pos < 0:
                continue
            lo = max(0, pos - window + 1) if window else 0
            row, n = int(plan.offsets[b]) + i, pos + 1 - lo
            for j in range(heads):
                h = j // group
                kh, vh, vah = k[h, lo:pos + 1], v[h, lo:pos + 1], va[h, lo:pos + 1]
                s = (kh @ q[row, j]) * scale
                top = s.max()
                p = np.exp(s - top)
                tot = p.sum()
                out[row, j] = (p @ vh) / tot
                lse[row, j] = top + np.log(tot)
                qa = np.abs((q[row, j] * sg) @ back)
                # A score: the query's rounding (its second term's smallest step,
                # 2^-25 of its largest), 2 d f32 additions and a few factors; the
                # exponential's argument is rounded in f32 beside the reference, which
                # lies within 64 + 41 of the scores (the exponent of a V scale).
                small = 2.0 ** -25 * qa.max() * ka[h, lo:pos + 1].sum(-1) * abs(scale) if tq4 else 0.0
                ds = (uq + (2 * d + 8) * U["f32"]) * ((ka[h, lo:pos + 1] @ qa) * abs(scale)) + small
                ds = ds + 8 * U["f32"] * (np.abs(s) + np.abs(top) + (110 if quant else 2))
                # Weight by weight: its score's error, its rounding, f32 sums.
                rel = up + 2 * (ds + ds.max()) + (n + 64) * 2 * U["f32"]
                e = ((p * rel) @ vah) / tot
                if pool.fmt != "bf16":
                    # operands below the f16 steps, times the largest value one stands for
                    if quant:
                        one = p * vah.max(-1)
                        if tq4:  # (a row may lack the largest magnitude)
                            one = p * np.sqrt((vah ** 2).mean(-1)) * 4.0
                        e = e + 2.0 ** -31 * n * one.max() / tot
                    else:
                        e = e + 2.0 ** -31 * vah.sum(0) * p.max() / tot
                if tq4:  # rotated back: every coordinate has a share of each error
                    e = np.full(d, np.sqrt((e * e).sum()))
                tol[row, j] = U[dtype] * (np.abs(out[row, j]) + e) + e + (2.0 ** -25 if dtype == "f16" else 0)
                ltol[row, j] = 2 * ds.max() + (n + 64) * 2 * U["f32"] + 4 * U["f32"] * (abs(lse[row, j]) + 110)
    return out, lse, tol, ltol
