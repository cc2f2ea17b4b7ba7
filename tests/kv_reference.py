"""Plain restatement of the paged key-value cache in numpy: the pools' layout,
the storage formats and attention in 64 bits, with bounds on how far a result
in the kernels' arithmetic may be off.

A rounding is off by at most half a step, u = eps / 2 relative to the value:
2^-11 for f16, 2^-8 for bf16, 2^-24 for f32."""
import numpy as np

U = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}
BITS = {"f16": 16, "bf16": 16, "q8": 8, "tq4": 4}


def to_bf16(x):
    """f32 -> bf16 bits (u16), nearest even, NaN kept."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((u.astype(np.uint64) + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r).astype(np.uint16)


def from_bf16(b):
    return (np.asarray(b, np.uint16).astype(np.uint32) << 16).view(np.float32)


def to_rows(x, dtype):
    """f32 values -> the bits of rows of dtype."""
    if dtype == "bf16":
        return to_bf16(x)
    return np.asarray(x, np.float32).astype(np.float16 if dtype == "f16" else np.float32)


def from_rows(r, dtype):
    return from_bf16(r) if dtype == "bf16" else np.asarray(r, np.float32)


def hadamard(d):
    h = np.ones((1, 1))
    while h.shape[0] < d:
        h = np.block([[h, h], [h, -h]])
    return h


class Pool:
    """Pools on the host, as bytes and as the values they stand for."""

    def __init__(self, fmt, kvh, d, p, pages, seed=0, codebook=None, signs=None):
        self.fmt, self.kvh, self.d, self.p, self.pages = fmt, kvh, d, p, pages
        self.codebook, self.signs = codebook, signs
        rng = np.random.default_rng(seed)
        n = pages * kvh * p
        # Old content: any bytes (NaN and infinity among them) and scales.
        self.k = rng.integers(0, 256, n * d * BITS[fmt] // 8, dtype=np.uint8)
        self.v = rng.integers(0, 256, n * d * BITS[fmt] // 8, dtype=np.uint8)
        self.k_scale = np.exp(rng.normal(size=n)).astype(np.float32)
        self.v_scale = np.exp(rng.normal(size=n)).astype(np.float32)

    def arrays(self):
        a = {"k": self.k, "v": self.v}
        if self.fmt in ("q8", "tq4"):
            a |= {"k_scale": self.k_scale, "v_scale": self.v_scale}
        return a

    def views(self):
        """K [pages, H, P, d] and V [pages, H, P / 8, d, 8] codes, and scales
        [pages, H, P]; 4-bit codes unpacked (write back with put)."""
        pg, h, p, d = self.pages, self.kvh, self.p, self.d
        if self.fmt in ("f16", "bf16"):
            k, v = self.k.view(np.uint16), self.v.view(np.uint16)
        elif self.fmt == "q8":
            k, v = self.k.view(np.int8), self.v.view(np.int8)
        else:
            sh = 4 * np.arange(8, dtype=np.uint32)
            k = (self.k.view(np.uint32)[:, None] >> sh & 15).astype(np.uint8)
            v = (self.v.view(np.uint32)[:, None] >> sh & 15).astype(np.uint8)
        return (k.reshape(pg, h, p, d), v.reshape(pg, h, p // 8, d, 8),
                self.k_scale.reshape(pg, h, p), self.v_scale.reshape(pg, h, p))

    def put(self, k, v):
        if self.fmt != "tq4":
            return  # views() gave the arrays themselves
        sh = 4 * np.arange(8, dtype=np.uint32)
        pack = lambda c: (c.reshape(-1, 8).astype(np.uint32) << sh).sum(1).astype(np.uint32)  # noqa: E731
        self.k = pack(k).view(np.uint8)
        self.v = pack(v).view(np.uint8)

    def quantize(self, x):
        """Rows f32 [n, H, d] -> (codes, scales); tq4 in 64 bits."""
        f = np.float32
        if self.fmt == "q8":
            most = np.abs(x).max(-1)
            with np.errstate(all="ignore"):
                scale = (most / f(127)).astype(f)
                ok = (scale >= f(2.0 ** -60)) & (scale <= f(2.0 ** 40))
                inv = np.where(ok, f(127) / most, f(0)).astype(f)
                code = np.clip(np.rint(x * inv[..., None]), -127, 127)
            code = np.where(ok[..., None], code, 0).astype(np.int8)
            nan = ~(scale <= f(2.0 ** 40))
            return code, np.where(nan, f(np.nan), np.where(ok, scale, f(0)))
        x = x.astype(np.float64)
        with np.errstate(all="ignore"):
            w = (x * self.signs) @ hadamard(self.d)
            scale = np.sqrt((x * x).mean(-1)).astype(f)
        nan, none = ~(scale <= f(2.0 ** 40)), scale < f(2.0 ** -60)
        w[nan | none] = 0.0
        cb = self.codebook.astype(np.float64)
        norm = np.where(nan | none, 0, scale).astype(np.float64) * np.sqrt(self.d)
        edge = (cb[1:] + cb[:-1]) / 2 * norm[..., None, None]
        code = (np.abs(w)[..., None] > edge).sum(-1) + 8 * (w < 0)
        # How near the closest edge (or a sign's turn) is, for what f32 may decide otherwise:
        # log2(d) additions of the transform, one product and two roundings of the edge.
        tol = (np.log2(self.d) + 4) * 2.0 ** -24 * np.abs(x).sum(-1)[..., None] + 4 * 2.0 ** -24 * norm[..., None] * 3
        near = (np.abs(np.abs(w)[..., None] - edge).min(-1) <= tol) | (np.abs(w) <= tol)
        return code.astype(np.uint8), np.where(nan, f(np.nan), np.where(none, f(0), scale)), near

    def values(self):
        """What the pools stand for, f64: K, V [pages, H, P, d]."""
        k, v, ks, vs = self.views()
        v = v.swapaxes(-1, -2).reshape(self.pages, self.kvh, self.p, self.d)
        if self.fmt == "f16":
            return k.view(np.float16).astype(np.float64), np.ascontiguousarray(v).view(np.float16).astype(np.float64)
        if self.fmt == "bf16":
            return from_bf16(k).astype(np.float64), from_bf16(v).astype(np.float64)
        with np.errstate(all="ignore"):
            if self.fmt == "q8":
                return k * ks[..., None].astype(np.float64), v * vs[..., None].astype(np.float64)
            cb = np.concatenate([self.codebook, -self.codebook]).astype(np.float64)
            back = hadamard(self.d) * (self.signs / np.sqrt(self.d))
            return ((cb[k] * ks[..., None].astype(np.float64)) @ back,
                    (cb[v] * vs[..., None].astype(np.float64)) @ back)


class Plan:
    """Sequences over a pool: rows n[b] of a call at the end of lengths[b]."""

    def __init__(self, pool, lengths, n, seed=0, stride=None, extra_rows=0, shuffle=True):
        self.pool, self.lengths, self.n = pool, np.asarray(lengths, np.int32), np.asarray(n, np.int32)
        need = -(-np.maximum(self.lengths, 0) // pool.p)
        self.stride = int(stride or max(1, need.max()))
        rng = np.random.default_rng(seed)
        ids = rng.permutation(pool.pages) if shuffle else np.arange(pool.pages)
        assert need.sum() <= pool.pages
        self.table = np.full((len(n), self.stride), -1, np.int32)
        at = 0
        for b, k in enumerate(need):
            self.table[b, :k] = ids[at:at + k]
            at += k
        self.offsets = np.concatenate([[0], np.cumsum(self.n)]).astype(np.int32)
        self.used = int(self.offsets[-1])
        self.rows = self.used + extra_rows

    def slots(self):
        """(row, sequence, position, page, slot) of every row that has one."""
        for b in range(len(self.n)):
            for i in range(self.n[b]):
                pos = int(self.lengths[b]) - int(self.n[b]) + i
                if pos >= 0:
                    yield (int(self.offsets[b]) + i, b, pos, int(self.table[b, pos // self.pool.p]),
                           pos % self.pool.p)

    def sequence(self, b, values):
        """Values [H, len, d] of sequence b."""
        ids = self.table[b, :-(-max(int(self.lengths[b]), 0) // self.pool.p)]
        x = values[ids].swapaxes(0, 1)
        return x.reshape(self.pool.kvh, -1, self.pool.d)[:, :max(int(self.lengths[b]), 0)]


def attention(plan, values, q, heads, dtype, scale, window=0):
    """q f64 [rows, heads, d] -> (out, lse, bound on out's error, bound on lse's),
    for rows the plan has. `values`: the pool's K and V."""
    pool = plan.pool
    d, group = pool.d, heads // pool.kvh
    quant = pool.fmt in ("q8", "tq4")
    out = np.zeros((plan.rows, heads, d))
    lse = np.full((plan.rows, heads), -np.inf)
    tol, ltol = np.zeros_like(out), np.zeros_like(lse)
    up = U["bf16" if pool.fmt == "bf16" else "f16"]
    # Rounding of the query: a rotated one (log2(d) f32 additions) goes to two f16
    # terms, 2^-22; any other is exact.
    uq = U["f16"] ** 2 + (np.log2(d) + 2) * U["f32"] if pool.fmt == "tq4" else 0.0
    back = hadamard(d) * (1 / np.sqrt(d)) if pool.fmt == "tq4" else np.eye(d)
    sg = pool.signs if pool.fmt == "tq4" else np.ones(d)
    for b in range(len(plan.n)):
        k, v = plan.sequence(b, values[0]), plan.sequence(b, values[1])
        # Magnitudes in the space the kernels sum in.
        ka, va = np.abs((k * sg) @ back), np.abs((v * sg) @ back)
        for i in range(plan.n[b]):
            pos = int(plan.lengths[b]) - int(plan.n[b]) + i
            if pos < 0:
                continue
            lo = max(0, pos - window + 1) if window else 0
            row = int(plan.offsets[b]) + i
            for j in range(heads):
                h = j // group
                s = (k[h, lo:pos + 1] @ q[row, j]) * scale
                top = s.max()
                p = np.exp(s - top)
                tot = p.sum()
                out[row, j] = (p @ v[h, lo:pos + 1]) / tot
                lse[row, j] = top + np.log(tot)
                qa = np.abs((q[row, j] * sg) @ back)
                mag = (ka[h, lo:pos + 1] @ qa) * abs(scale)
                # Score: the query's rounding (its second term is not below f16's normal range
                # before 2^-25 of its largest), d f32 additions of two terms, a few f32 factors;
                # exponential and its argument.
                small = 2.0 ** -25 * qa.max() * ka[h, lo:pos + 1].sum(-1) * abs(scale) if uq else 0.0
                ds = (uq + (2 * d + 8) * U["f32"]) * mag + small + 8 * U["f32"] * (np.abs(s).max() + 2)
                dmax = float(np.max(ds))
                n = pos + 1 - lo
                # Weights: rounded to the operand's type (f16 below 2^-14: 2^-25 absolute, of a
                # largest weight of at least 1, times the largest scale), n f32 additions.
                rel = up + 2 * dmax + (n + 64) * 2 * U["f32"]
                mean = (p @ va[h, lo:pos + 1]) / tot
                low = 0.0 if pool.fmt == "bf16" else 2.0 ** -25 * n * (va[h, lo:pos + 1].max() * (4 if quant else 1))
                e = rel * mean + low
                if pool.fmt == "tq4":  # rotated back: every coordinate has a share of each error
                    e = np.full(d, np.sqrt((e * e).sum()) if d else 0.0)
                tol[row, j] = U[dtype] * (np.abs(out[row, j]) + e) + e + (2.0 ** -25 if dtype == "f16" else 0)
                ltol[row, j] = dmax + (n + 64) * 2 * U["f32"] + 4 * U["f32"] * abs(lse[row, j])
    return out, lse, tol, ltol
