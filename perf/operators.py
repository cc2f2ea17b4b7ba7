"""The paged key-value cache and the attention over it, measured.

Three operators: rows of keys and values written into a paged cache in one of
four formats (f16, bf16, q8, tq4), the values of cached positions read back,
and attention of new rows over the cache (one row a sequence while decoding,
many for a prompt). `run` computes them in their plain form with elementary
torch operations, or through the package's entry points where `own` is true.

Cache memory, for `pages` pages of P tokens, H key-value heads and width d:
  K        [pages][H][P][d]         f16 / bf16 values, or q8 int8 codes
           [pages][H][P][d / 8]     tq4: int32 words, dimension 8 w + j at bits 4 j
  V        [pages][H][P / 8][d][8]  f16 / bf16 values, or q8 int8 codes: 8 tokens side by side
           [pages][H][P / 8][d]     tq4: int32 words, token 8 g + j at bits 4 j
  scales   [pages][H][P]            f32, one for K and one for V (q8, tq4)
q8 stands for code * scale. tq4 keeps a vector rotated: w = Hd (signs * x) / sqrt(d)
with Hd the Walsh-Hadamard matrix; a code is a sign (bit 3) and the index of
one of 8 magnitudes, and stands for +-magnitude * scale in the rotated space.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
# The 16-level quantizer of least squared error for a normal variable (8
# magnitudes; thresholds half way between them).
MAGNITUDES = [0.12841796875, 0.388427734375, 0.6572265625, 0.94287109375, 1.2568359375,
              1.6181640625, 2.068359375, 2.732421875]
TINY, HUGE = 2.0 ** -60, 2.0 ** 40  # scales kept as they are; below: zero, above: NaN


def listed():
    return [
        # Decoding: 16 sequences write one token each, 4-bit cache; the smallest call.
        dict(name="store_step", kind="store", fmt="tq4", io="bf16", kvh=8, dim=128, page=64,
             batch=16, rows=1, shortest=1, cached=4000, packed=True),
        # Prompts of ragged length written as 8-bit codes, heads of 64.
        dict(name="store_prompt", kind="store", fmt="q8", io="f16", kvh=12, dim=64, page=32,
             batch=8, rows=1021, shortest=77, cached=0, packed=True),
        # A long document ingested into the 4-bit cache.
        dict(name="store_long", kind="store", fmt="tq4", io="bf16", kvh=8, dim=128, page=64,
             batch=2, rows=16384, shortest=16384, cached=0, packed=False),
        # A short prefix taken out of an 8-bit cache.
        dict(name="restore_short", kind="restore", fmt="q8", io="f16", kvh=12, dim=64, page=16,
             batch=3, rows=205, shortest=31),
        # Long prefixes taken out of the 4-bit cache.
        dict(name="restore_long", kind="restore", fmt="tq4", io="bf16", kvh=8, dim=128, page=64,
             batch=4, rows=8192, shortest=4096),
        # One short conversation, plain f16, as many key-value heads as heads: latency.
        dict(name="decode_one", kind="attend", fmt="f16", io="f16", heads=12, kvh=12, dim=64,
             page=16, batch=1, rows=1, shortest=1, cached=776, least=776, window=0, packed=False),
        # A serving batch of ragged conversations in bf16, four heads to one.
        dict(name="decode_batch", kind="attend", fmt="bf16", io="bf16", heads=32, kvh=8, dim=128,
             page=32, batch=32, rows=1, shortest=1, cached=4095, least=64, window=0, packed=True),
        # One very long context, 8-bit.
        dict(name="decode_long", kind="attend", fmt="q8", io="bf16", heads=32, kvh=8, dim=128,
             page=64, batch=1, rows=1, shortest=1, cached=131071, least=131071, window=0,
             packed=False),
        # A large serving batch of long contexts, 4-bit.
        dict(name="decode_tq4", kind="attend", fmt="tq4", io="bf16", heads=32, kvh=8, dim=128,
             page=64, batch=64, rows=1, shortest=1, cached=16383, least=1024, window=0,
             packed=False),
        # A few drafted tokens a sequence checked at once against an 8-bit cache.
        dict(name="draft", kind="attend", fmt="q8", io="f16", heads=28, kvh=4, dim=128, page=64,
             batch=8, rows=5, shortest=2, cached=8000, least=500, window=0, packed=True),
        # Ragged short prompts, f16, heads of 64.
        dict(name="prompt_short", kind="attend", fmt="f16", io="f16", heads=12, kvh=12, dim=64,
             page=16, batch=16, rows=511, shortest=17, cached=0, least=0, window=0, packed=True),
        # Two long prompts, bf16: the largest.
        dict(name="prompt_long", kind="attend", fmt="bf16", io="bf16", heads=32, kvh=8, dim=128,
             page=64, batch=2, rows=8192, shortest=8192, cached=0, least=0, window=0,
             packed=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "restore", "attend", "attend", "attend", "attend"])
    fmt = rng.choice(["f16", "bf16", "q8", "q8", "tq4", "tq4"])
    io = fmt if fmt in ("f16", "bf16") else rng.choice(["f16", "bf16"])
    dim = rng.choice([32, 64, 64, 128, 128, 128, 256])
    page = rng.choice([16, 32, 64, 128, 256])
    kvh = rng.choice([1, 2, 3, 4, 8, 8, 12])
    batch = _log_int(rng, 1, 128)
    base = dict(kind=kind, fmt=fmt, io=io, kvh=kvh, dim=dim, page=page, batch=batch,
                packed=rng.random() < 0.5)
    elems = 64 * 8192 * 8 * 128  # the largest listed cache: K elements
    if kind != "attend":
        rows = _log_int(rng, 1, max(1, min(16384, 32768 * 8 * 128 // (batch * kvh * dim))))
        base.update(rows=rows, shortest=rng.randint(1, rows))
        if kind == "restore":
            base.pop("packed")
        else:
            base.update(cached=rng.choice([0, rng.randint(0, 3000)]))
        return base
    group = rng.choice([1, 1, 2, 3, 4, 4, 5, 7, 8, 16])
    heads = kvh * group
    if rng.random() < 0.6:  # decoding, now and then a few drafted rows
        rows = rng.choice([1, 1, 1, rng.randint(2, 9)])
        cached = _log_int(rng, 1, max(1, min(131072, elems // (batch * kvh * dim))))
        shortest = rng.randint(1, rows)
    else:  # prompts, some behind a cached prefix
        most = 2 * 32 * 8192 * 8192 // (batch * heads)
        rows = _log_int(rng, 10, max(10, min(8192, int(math.sqrt(most)))))
        cached = rng.choice([0, rng.randint(0, max(0, min(16384, most // rows - rows)))])
        shortest = rng.randint(1, rows)
    least = rng.randint(0, cached)
    window = rng.choice([0, 0, 0, rng.randint(1, rows + cached)])
    base.update(heads=heads, rows=rows, shortest=shortest, cached=cached, least=least,
                window=window)
    return base


# ------------------------------------------------------------------- sizes


def _spread(lo, hi, n, phase):
    """n whole numbers over [lo, hi], the last of them hi."""
    got = [lo + int((hi - lo + 1) * (((i + 1) * 0.6180339887498949 + phase) % 1.0)) for i in range(n)]
    return got[:-1] + [hi]


def _sizes(case):
    """New rows of each sequence, and its length once they are written."""
    rows = _spread(case["shortest"], case["rows"], case["batch"], 0.0)
    if case["kind"] == "restore":
        return rows, rows
    cached = _spread(case.get("least", 0), case["cached"], case["batch"], 0.37)
    return rows, [r + c for r, c in zip(rows, cached)]


def _keys(row_pos, window):
    """Keys that a row at this position attends."""
    return row_pos + 1 if window == 0 else min(row_pos + 1, window)


def work(case):
    rows, lens = _sizes(case)
    kvh, d, n = case["kvh"], case["dim"], sum(rows)
    bits = {"f16": 16, "bf16": 16, "q8": 8, "tq4": 4}[case["fmt"]]
    token = 2 * kvh * (d * bits // 8 + (4 if bits < 16 else 0))  # K and V of one position
    io = 2 * kvh * d * 2                                         # K and V of one row
    if case["kind"] == "store":
        return {"bytes": n * (io + token) + n * (token + io), "flops": 0}
    if case["kind"] == "restore":
        return {"bytes": n * (token + io), "flops": 0}
    w, h = case["window"], case["heads"]
    live = pairs = 0
    for r, t in zip(rows, lens):
        first = t - r
        live += t if w == 0 else min(t, w + r - 1)
        pairs += r * first + r * (r + 1) // 2 if w == 0 else sum(_keys(p, w) for p in range(first, t))
    return {"bytes": live * token + 2 * n * h * d * 2, "flops": 4 * d * h * pairs}


# ------------------------------------------------------------------ inputs


def _hadamard(d):
    h = torch.ones(1, 1, dtype=torch.float64)
    while h.shape[0] < d:
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
    return h


def _scales(shape, g, bits):
    """Scales as normal rows give them: 8-bit from the largest of a row, 4-bit its size."""
    s = torch.exp(0.3 * torch.randn(shape, generator=g, device=DEV))
    return s * (2.7 / 127.0) if bits == 8 else s


def _pool(fmt, pages, case, g):
    """A cache as earlier tokens left it."""
    kvh, p, d = case["kvh"], case["page"], case["dim"]
    ks, vs = (pages, kvh, p, d), (pages, kvh, p // 8, d, 8)
    if fmt in ("f16", "bf16"):
        dt = DTYPES[fmt]
        return {"k": torch.randn(ks, generator=g, device=DEV).to(dt),
                "v": torch.randn(vs, generator=g, device=DEV).to(dt)}
    sc = {n: _scales((pages, kvh, p), g, 8 if fmt == "q8" else 4) for n in ("k_scale", "v_scale")}
    if fmt == "q8":
        return {n: (47.0 * torch.randn(s, generator=g, device=DEV)).clamp_(-127, 127).to(torch.int8)
                for n, s in (("k", ks), ("v", vs))} | sc
    return {n: torch.randint(-2 ** 31, 2 ** 31, s, generator=g, device=DEV).to(torch.int32)
            for n, s in (("k", (pages, kvh, p, d // 8)), ("v", (pages, kvh, p // 8, d)))} | sc


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        _bind(s)
    return s


def _inputs(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    rows, lens = _sizes(case)
    kvh, p, d, io = case["kvh"], case["page"], case["dim"], DTYPES[case["io"]]
    batch, n = case["batch"], sum(rows)
    need = [-(-t // p) for t in lens]
    stride = max(need) + 1
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((batch, stride), -1, dtype=torch.int32)
    at = 0
    for b in range(batch):
        table[b, :need[b]] = torch.tensor(order[at:at + need[b]], dtype=torch.int32)
        at += need[b]
    offsets = [0]
    for r in rows:
        offsets.append(offsets[-1] + r)
    s = {"case": case, "rows": n, "most_rows": max(rows), "pages": pages,
         "table": table.to(DEV), "lengths": torch.tensor(lens, dtype=torch.int32, device=DEV),
         "offsets": torch.tensor(offsets, dtype=torch.int32, device=DEV),
         "mags": torch.tensor(MAGNITUDES, device=DEV),
         "signs": (torch.randint(0, 2, (d,), generator=g, device=DEV) * 2 - 1).float(),
         "had": _hadamard(d).to(DEV)}
    s["pool"] = _pool(case["fmt"], pages, case, g)
    heads = case.get("heads", 0)
    if case["kind"] == "store":
        # Rows with a few large channels, as keys have them.
        size = torch.exp(0.8 * torch.randn(2 * kvh * d, generator=g, device=DEV))
        x = (torch.randn(n, 2 * kvh * d, generator=g, device=DEV) * size).to(io)
        if not case["packed"]:
            s["k"], s["v"] = x[:, :kvh * d].contiguous(), x[:, kvh * d:].contiguous()
        else:  # slices of one projection's output
            s["k"], s["v"] = x[:, :kvh * d], x[:, kvh * d:]
    if case["kind"] in ("store", "restore"):
        s["k_out"] = torch.zeros(n, kvh * d, dtype=io, device=DEV)
        s["v_out"] = torch.zeros(n, kvh * d, dtype=io, device=DEV)
    if case["kind"] == "attend":
        q = torch.randn(n, (heads + 2 * kvh if case["packed"] else heads) * d, generator=g, device=DEV)
        # Most rows spread over many keys, some fix on a few.
        q *= torch.exp(0.5 * torch.randn(n, 1, generator=g, device=DEV))
        s["q"] = q.to(io)[:, :heads * d]
        s["out"] = torch.zeros(n, heads * d, dtype=io, device=DEV)
    return s


# --------------------------------------------------------- the package's calls

_rt = None


class _Dev:
    """A tensor's device memory, as the device entry points take it."""

    def __init__(self, t):
        import ctypes
        self.t, self.nbytes = t, t.untyped_storage().nbytes() - t.storage_offset() * t.element_size()
        self.ptr = ctypes.c_void_p(t.data_ptr())


def _bind(s):
    """The program's runtime, its cache over the pages and the batch's plan."""
    global _rt
    from eos_amd.kvcache import KVBatch, KVCache
    from eos_amd.runtime import Runtime
    if _rt is None:
        _rt = Runtime(0)
    case, tq4 = s["case"], s["case"]["fmt"] == "tq4"
    s["cache"] = KVCache(_rt, case["fmt"], case["kvh"], case["dim"], case["page"], s["pages"],
                         codebook=s["mags"].cpu().numpy() if tq4 else None,
                         signs=s["signs"].cpu().numpy() if tq4 else None,
                         **{n: _Dev(t) for n, t in s["pool"].items()})
    one_each = s["most_rows"] == 1
    s["plan"] = KVBatch(_Dev(s["table"]), s["table"].shape[1], case["batch"], _Dev(s["lengths"]),
                        None if one_each else _Dev(s["offsets"]), s["rows"])
    s["dev"] = {n: _Dev(s[n]) for n in ("k", "v", "q", "out", "k_out", "v_out") if n in s}


def _run_own(s):
    case, c, plan, dev = s["case"], s["cache"], s["plan"], s["dev"]
    if case["kind"] == "attend":
        c.attend(plan, dev["q"], case["heads"], dev["out"], case["io"], window=case["window"],
                 q_stride=s["q"].stride(0))
        return s["out"]
    if case["kind"] == "store":
        c.append(plan, dev["k"], dev["v"], case["io"], k_stride=s["k"].stride(0),
                 v_stride=s["v"].stride(0))
    c.read(plan, dev["k_out"], dev["v_out"], case["io"])
    return {"k": s["k_out"], "v": s["v_out"]}


# --------------------------------------------------------------- plain forms


def _places(s):
    """Page, place in the page and sequence of every row of the call."""
    p, off, lens = s["case"]["page"], s["offsets"].long(), s["lengths"].long()
    seq = torch.repeat_interleave(torch.arange(len(lens), device=DEV), off[1:] - off[:-1],
                                  output_size=s["rows"])
    pos = torch.arange(s["rows"], device=DEV) - off[seq + 1] + lens[seq]
    return s["table"][seq, pos // p].long(), pos % p, seq, pos


def _kept(scale):
    """A scale as the cache keeps it."""
    scale = torch.where(scale < TINY, torch.zeros_like(scale), scale)
    return torch.where(scale <= HUGE, scale, torch.full_like(scale, math.nan))


def _nibbles(x):
    """4-bit codes [..., 8] -> int32 words."""
    shifts = 4 * torch.arange(8, device=DEV)
    words = (x.long() << shifts).sum(-1)
    return (words - ((words >> 31) << 32)).to(torch.int32)


def _codes(words):
    return (words.unsqueeze(-1) >> (4 * torch.arange(8, device=DEV, dtype=torch.int32))) & 15


def _quantize(s, x):
    """Rows f32 [n, H, d] -> codes [n, H, d] and scales [n, H]."""
    if s["case"]["fmt"] == "q8":
        most = x.abs().amax(-1)
        scale = _kept(most / torch.full_like(most, 127.0))
        inv = torch.where(scale > 0, torch.full_like(most, 127.0) / most, torch.zeros_like(most))
        return torch.round(x * inv.unsqueeze(-1)).clamp(-127, 127), scale
    d = s["case"]["dim"]
    x = x.double()  # a code turns at a threshold: values next to one need the bits
    w = (x * s["signs"].double()) @ s["had"]
    scale = _kept(torch.sqrt(x.square().sum(-1) / d).float())
    m = s["mags"].double()
    edge = 0.5 * (m[1:] + m[:-1]) * (scale.double() * math.sqrt(d)).unsqueeze(-1).unsqueeze(-1)
    index = (w.abs().unsqueeze(-1) > edge).sum(-1)
    return torch.where(scale.unsqueeze(-1) > 0, index + 8 * (w < 0), torch.zeros_like(index)), scale


def _levels(s, codes):
    """4-bit codes -> +-magnitudes, f32."""
    return s["mags"][(codes & 7).long()] * (1.0 - 2.0 * (codes >> 3).float())


def _unrotate(s, x):
    """Rotated values f32 [..., d] -> the values they stand for."""
    return (x @ s["had"].float()) * (s["signs"] / math.sqrt(s["case"]["dim"]))


def _store(s):
    """Rows into the pages, in the cache's own format."""
    case, pool = s["case"], s["pool"]
    shape = (s["rows"], case["kvh"], case["dim"])
    page, at, _, _ = _places(s)
    k, v = s["k"].reshape(shape), s["v"].reshape(shape)
    if case["fmt"] in ("f16", "bf16"):
        pool["k"][page, :, at] = k
        pool["v"][page, :, at // 8, :, at % 8] = v
        return
    kc, pool["k_scale"][page, :, at] = _quantize(s, k.float())
    vc, pool["v_scale"][page, :, at] = _quantize(s, v.float())
    if case["fmt"] == "q8":
        pool["k"][page, :, at] = kc.to(torch.int8)
        pool["v"][page, :, at // 8, :, at % 8] = vc.to(torch.int8)
        return
    pool["k"][page, :, at] = _nibbles(kc.reshape(*shape[:2], -1, 8))
    whole = _codes(pool["v"])  # a word holds eight tokens: the others stay
    whole[page, :, at // 8, :, at % 8] = vc.to(torch.int32)
    pool["v"].copy_(_nibbles(whole))


def _values(s, k, v, ks, vs):
    """Cached K [..., d] (tq4: words) and V, both token-major, as f32 values."""
    fmt = s["case"]["fmt"]
    if fmt in ("f16", "bf16"):
        return k.float(), v.float()
    if fmt == "q8":
        return k.float() * ks.unsqueeze(-1), v.float() * vs.unsqueeze(-1)
    k = _levels(s, _codes(k).flatten(-2)) * ks.unsqueeze(-1)
    return _unrotate(s, k), _unrotate(s, _levels(s, v) * vs.unsqueeze(-1))


def _restore(s):
    case, pool = s["case"], s["pool"]
    page, at, _, _ = _places(s)
    v = pool["v"][page, :, at // 8]  # [n, H, d, 8], or words [n, H, d]
    pick = (at % 8).view(-1, 1, 1, 1).expand(*v.shape[:3], 1)
    v = (_codes(v) if case["fmt"] == "tq4" else v).gather(-1, pick).squeeze(-1)
    ks, vs = (pool[n][page, :, at] if n in pool else None for n in ("k_scale", "v_scale"))
    k, v = _values(s, pool["k"][page, :, at], v, ks, vs)
    io = DTYPES[case["io"]]
    return {"k": k.to(io).flatten(1), "v": v.to(io).flatten(1)}


def _attend(s):
    case, pool = s["case"], s["pool"]
    b, kvh, d, h = case["batch"], case["kvh"], case["dim"], case["heads"]
    table = s["table"].long().clamp(min=0)
    t = table.shape[1] * case["page"]

    def tokens(x):  # [B, pages, H, P, ...] -> [B, H, tokens, ...]
        return x.transpose(1, 2).flatten(2, 3)

    v = pool["v"][table]  # [B, pages, H, P / 8, d, 8]
    v = tokens((_codes(v) if case["fmt"] == "tq4" else v).transpose(-1, -2).flatten(3, 4))
    ks, vs = (tokens(pool[n][table]) if n in pool else None for n in ("k_scale", "v_scale"))
    k, v = _values(s, tokens(pool["k"][table]), v, ks, vs)
    _, _, seq, pos = _places(s)
    row = torch.arange(s["rows"], device=DEV) - s["offsets"].long()[seq]
    q = torch.zeros(b, s["most_rows"], h, d, device=DEV)
    q[seq, row] = s["q"].reshape(-1, h, d).float()
    at = torch.full((b, s["most_rows"]), -1, device=DEV)
    at[seq, row] = pos
    # The heads of a group, row by row, against their one key head.
    q = q.view(b, -1, kvh, h // kvh, d).permute(0, 2, 3, 1, 4).flatten(2, 3)
    x = (q @ k.transpose(-1, -2)) / math.sqrt(d)  # [B, H, group * rows, tokens]
    key = torch.arange(t, device=DEV)
    seen = key <= at.unsqueeze(-1)
    if case["window"]:
        seen &= key > at.unsqueeze(-1) - case["window"]
    x = x.view(b, kvh, h // kvh, -1, t).masked_fill_(~seen[:, None, None], -math.inf)
    x = x.sub_(x.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    x = x.div_(x.sum(-1, keepdim=True).clamp(min=1e-30)).flatten(2, 3)
    x = (x @ v).view(b, kvh, h // kvh, -1, d).permute(0, 3, 1, 2, 4).flatten(2)
    return x[seq, row].to(DTYPES[case["io"]])


def run(s):
    if own:
        return _run_own(s)
    kind = s["case"]["kind"]
    if kind == "attend":
        return _attend(s)
    if kind == "store":
        _store(s)
    return _restore(s)


# ------------------------------------------------------------------- 64 bits


def exact(case, seed):
    """The definition in 64 bits, a sequence and a key-value head at a time."""
    rows, lens = _sizes(case)
    if case["batch"] * case["kvh"] > 1600:
        return None
    s = _inputs(case, seed)
    fmt, kvh, d, p = case["fmt"], case["kvh"], case["dim"], case["page"]
    had = s["had"] / math.sqrt(d)
    signs, mags = s["signs"].double(), s["mags"].double()
    edge = (mags[1:] + mags[:-1]) / 2

    def stands(x):  # rows f64 -> what the cache keeps of them
        if fmt in ("f16", "bf16"):
            return x
        if fmt == "q8":
            a = x.abs().amax(-1, keepdim=True) / 127.0
            return torch.where(a > TINY, torch.round(x / a) * a, torch.zeros_like(x))
        rms = x.square().mean(-1, keepdim=True).sqrt()
        u = (x * signs) @ had
        idx = torch.bucketize(u.abs() / rms, edge)
        return ((torch.copysign(mags[idx], u) * rms) @ had) * signs

    if case["kind"] == "store":
        k, v = (stands(s[n].double().view(-1, kvh, d)).flatten(1) for n in ("k", "v"))
        return {"k": k, "v": v}

    def head(name, b, h, upto):  # values f64 [upto, d] of one sequence and head
        ids = s["table"][b, :-(-upto // p)].long()
        x = s["pool"][name][ids, h]
        if fmt == "tq4":
            c = torch.stack([(x >> (4 * j)) & 15 for j in range(8)], -1).long()
            c = c.reshape(-1, d) if name == "k" else c.transpose(-1, -2).reshape(-1, d)
            x = torch.where(c >= 8, -mags[c % 8], mags[c % 8])
        else:
            x = x.double()
            x = x.reshape(-1, d) if name == "k" else x.transpose(-1, -2).reshape(-1, d)
        if fmt in ("q8", "tq4"):
            x = x * s["pool"][name + "_scale"][ids, h].double().reshape(-1, 1)
        x = x[:upto]
        return (x @ had) * signs if fmt == "tq4" else x

    if case["kind"] == "restore":
        got = {n: torch.empty(s["rows"], kvh, d, dtype=torch.float64, device=DEV) for n in ("k", "v")}
        at = 0
        for b, r in enumerate(rows):
            for h in range(kvh):
                for n in ("k", "v"):
                    got[n][at:at + r, h] = head(n, b, h, lens[b])[lens[b] - r:]
            at += r
        return {n: x.flatten(1) for n, x in got.items()}
    group = case["heads"] // kvh
    out = torch.empty(s["rows"], case["heads"], d, dtype=torch.float64, device=DEV)
    q = s["q"].double().view(s["rows"], case["heads"], d)
    at = 0
    for b, r in enumerate(rows):
        pos = torch.arange(lens[b] - r, lens[b], device=DEV).unsqueeze(1)
        key = torch.arange(lens[b], device=DEV)
        hidden = key > pos
        if case["window"]:
            hidden |= key <= pos - case["window"]
        for h in range(kvh):
            k, v = head("k", b, h, lens[b]), head("v", b, h, lens[b])
            for j in range(h * group, (h + 1) * group):
                x = (q[at:at + r, j] @ k.T) * d ** -0.5
                x = torch.softmax(x.masked_fill(hidden, -math.inf), -1)
                out[at:at + r, j] = x @ v
        at += r
    return out.flatten(1)
