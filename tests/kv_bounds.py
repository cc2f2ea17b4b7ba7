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
        pos = int(plan.lengths[b]) - int(plan.n[b]) + np.arange(plan.n[b])
        at = int(plan.offsets[b]) + np.nonzero(pos >= 0)[0]
        pos = pos[pos >= 0]
        if not len(pos):
            continue
        key = np.arange(int(plan.lengths[b]))
        see = key <= pos[:, None]
        if window:
            see &= key > pos[:, None] - window
        n = see.sum(1)
        k, v = (plan.sequence(b, x).copy() for x in vals)
        k[:, ~see.any(0)] = v[:, ~see.any(0)] = 0.0          # no row's: whatever stands there
        ka, va = np.abs((k * sg) @ back), np.abs((v * sg) @ back)
        for j in range(heads):
            h = j // group
            x = np.where(see, (q[at, j] @ k[h].T) * scale, -np.inf)
            top = x.max(1, keepdims=True)
            p = np.exp(x - top)
            tot = p.sum(1, keepdims=True)
            got = (p @ v[h]) / tot
            out[at, j], lse[at, j] = got, top[:, 0] + np.log(tot[:, 0])
            qa = np.abs((q[at, j] * sg) @ back)
            # A score: the query's rounding (its second term's smallest step, 2^-25
            # of its largest), 2 d f32 additions and a few factors; the exponential's
            # argument is rounded in f32 beside the reference, which lies within 64 +
            # 41 of the scores (the exponent of a V scale).
            ds = (uq + (2 * d + 8) * U["f32"]) * ((qa @ ka[h].T) * abs(scale))
            if tq4:
                ds += 2.0 ** -25 * qa.max(1, keepdims=True) * ka[h].sum(-1) * abs(scale)
            far = np.where(see, np.abs(x), 0)
            ds += 8 * U["f32"] * (far + np.abs(top) + (110 if quant else 2))
            ds = np.where(see, ds, 0)
            most = ds.max(1, keepdims=True)
            # Weight by weight: its score's error, its rounding, f32 sums.
            rel = up + 2 * (ds + most) + (n[:, None] + 64) * 2 * U["f32"]
            e = ((p * rel) @ va[h]) / tot
            if pool.fmt != "bf16":
                # operands below the f16 steps, times the largest value one stands for
                if quant:
                    big = va[h].max(-1)
                    if tq4:  # (a row may lack the largest magnitude)
                        big = np.sqrt((va[h] ** 2).mean(-1)) * 4.0
                    # (the reference counts a scale as 2^-64 at least: its exponent is
                    # taken upwards, codes go to 127)
                    big = np.maximum(big, 2.0 ** (-63 + 7))
                    e += 2.0 ** -31 * n[:, None] * (p * big).max(1, keepdims=True) / tot
                else:
                    e += 2.0 ** -31 * (see @ va[h]) / tot
            # weights, and products, below f32's range
            e += 2.0 ** -125 * ((see @ va[h]) / tot + 1)
            if tq4:  # rotated back: every coordinate has a share of each error
                e = np.repeat(np.sqrt((e * e).sum(1, keepdims=True)), d, 1)
            tol[at, j] = U[dtype] * (np.abs(got) + e) + e + (2.0 ** -25 if dtype == "f16" else 0)
            ltol[at, j] = 2 * most[:, 0] + (n + 64) * 2 * U["f32"] + 4 * U["f32"] * (np.abs(lse[at, j]) + 110)
    return out, lse, tol, ltol
