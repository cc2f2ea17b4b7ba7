"""MXFP4 rows in 64 bits, from the format's definition."""
import numpy as np

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
U = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}
STEP = {"f16": 2.0 ** -24, "bf16": 2.0 ** -133, "f32": 2.0 ** -149}  # the smallest subnormal


def to_bits(x, dtype):
    """f64 or f32 values as rows of a type, rounded once to the nearest."""
    x = np.asarray(x, np.float32)
    if dtype == "f32":
        return x
    if dtype == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16)
    u = x.view(np.uint32)
    r = ((u.astype(np.uint64) + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), (u >> 16).astype(np.uint16) | 0x40, r)


def from_bits(b, dtype):
    if dtype == "bf16":
        return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return b.astype(np.float64)


def np_dtype(dtype):
    return {"f16": np.float16, "bf16": np.uint16, "f32": np.float32}[dtype]


def quantize(x):
    """Rows f64 [rows, k] -> codes u8 [rows, 16 blocks], scales u8 [rows, blocks]."""
    rows, k = x.shape
    blocks = -(-k // 32)
    p = np.zeros((rows, blocks * 32))
    p[:, :k] = x
    p = p.reshape(rows, blocks, 32)
    most = np.abs(p).max(-1)
    with np.errstate(all="ignore"):
        e = np.frexp(most)[1] - 3
    e = np.where(most > 0, np.clip(e, -127, 127), -127)
    bad = ~np.isfinite(p).all(-1)
    e = np.where(bad, 0, e)
    with np.errstate(all="ignore"):
        v = np.where(bad[..., None], 0.0, p) * 2.0 ** -e[..., None].astype(np.float64)
    a = np.abs(v)
    step = np.where(a < 2, 0.5, np.where(a < 4, 1.0, 2.0))
    a = np.minimum(np.rint(a / step) * step, 6.0)
    code = np.searchsorted(LEVELS, a) + 8 * np.signbit(v)
    code = np.where(bad[..., None], 0, code).astype(np.uint8)
    codes = (code[..., 0::2] | code[..., 1::2] << 4).reshape(rows, blocks * 16)
    return codes, np.where(bad, 255, e + 127).astype(np.uint8)


def values(codes, scales, k):
    """What codes and scales stand for, f64 [rows, k]."""
    rows, blocks = scales.shape
    c = codes.reshape(rows, blocks, 16)
    c = np.stack([c & 15, c >> 4], -1).reshape(rows, blocks, 32)
    v = np.where(c & 8, -1.0, 1.0) * LEVELS[c & 7]
    s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return (v * s[..., None]).reshape(rows, -1)[:, :k]


def linear(x, w, bias, out):
    """(x w^T + bias f64, bound on a result of type `out`): products are exact,
    of the k + 1 f32 additions each is off by less than a step of what it adds up."""
    with np.errstate(invalid="ignore"):
        y = x @ w.T
        size = np.abs(x) @ np.abs(w).T
    if bias is not None:
        y, size = y + bias, size + np.abs(bias)
    e = (x.shape[1] + 2) * 2.0 ** -23 * size + 2.0 ** -149
    return y, e + U[out] * (np.abs(y) + e) + STEP[out] / 2
