"""The operators of a decoding step around the paged cache, measured.

Rows in microscaled 4-bit floating point (MXFP4) and the linear layer over
weights held so, rotary positions of queries and keys, and the page tables and
slot maps of a batch built from the lengths of its requests. `run` computes
them in their plain form with elementary torch operations, or through the
package's entry points where `own` is true.

MXFP4 rows of k values: a block is 32 consecutive ones (the last may be
ragged, zeros behind it). Its scale is 2^e, stored as e + 127 in a byte, with
e = floor(log2(largest magnitude)) - 2 in -127..127; an element is x / 2^e
rounded to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to the even code)
and their negatives, saturating; codes [rows][16 blocks] bytes, element 2 i in
the low half of byte i; scales [rows][blocks] bytes.

The package's calls are enqueued on its runtime's own stream, which torch's
streams do not wait for: whoever reads the outputs of `run`, or drops a state
whose memory torch may then hand out again, synchronises the device first.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def listed():
    return [
        # A decoding batch's rows held in 4 bits and taken back: the smallest call.
        dict(name="quant_step", kind="quant", io="bf16", rows=32, k=4096, packed=False),
        # A prompt's rows, slices of a wider projection's output.
        dict(name="quant_prompt", kind="quant", io="bf16", rows=16384, k=4096, packed=True),
        # One token through the projection to queries, keys and values: latency and weights.
        dict(name="linear_one", kind="linear", io="bf16", out="bf16", rows=1, k=4096, n=6144,
             bias=False),
        # A serving batch through a wide layer: the weights' bytes.
        dict(name="linear_batch", kind="linear", io="bf16", out="bf16", rows=48, k=4096, n=16384,
             bias=False),
        # Odd sizes with a bias, results in 32 bits, as a scoring head takes them.
        dict(name="linear_ragged", kind="linear", io="f16", out="f32", rows=777, k=1000, n=1531,
             bias=True),
        # Rows quantised once for several layers.
        dict(name="linear_codes", kind="linear", io="mxfp4", out="f16", rows=2048, k=4096, n=4096,
             bias=True),
        # Long prompts through a large layer: the largest product.
        dict(name="linear_prompt", kind="linear", io="bf16", out="bf16", rows=8192, k=8192, n=8192,
             bias=False),
        # One new token for each of 32 conversations, heads 32 on 8 of 128.
        dict(name="rotary_step", kind="rotary", io="bf16", heads=32, kvh=8, dim=128, rot=128,
             layout="halves", batch=32, rows=1, shortest=1, cached=4000, packed=True,
             inverse=False),
        # Ragged prompts behind cached prefixes, the first quarter of each head, pairs.
        dict(name="rotary_prompt", kind="rotary", io="f16", heads=32, kvh=8, dim=128, rot=32,
             layout="pairs", batch=16, rows=1021, shortest=77, cached=120000, packed=True,
             inverse=False),
        # The gradients of a long batch's queries and keys.
        dict(name="rotary_back", kind="rotary", io="bf16", heads=32, kvh=32, dim=128, rot=128,
             layout="halves", batch=4, rows=4096, shortest=4096, cached=0, packed=False,
             inverse=True),
        # 64 conversations get a token each, whose draft is then dropped.
        dict(name="pages_step", kind="pages", slots=64, stride=128, page=64, new=1, busy=1.0,
             cached=8000, tight=False),
        # A large server: prompts for some requests, none for others.
        dict(name="pages_prompts", kind="pages", slots=4096, stride=512, page=16, new=2000, busy=0.4,
             cached=4000, tight=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["quant", "linear", "linear", "linear", "rotary", "rotary", "pages"])
    if kind == "quant":
        k = _log_int(rng, 32, 16384)
        return dict(kind=kind, io=rng.choice(["f16", "bf16", "f32"]), k=k,
                    rows=_log_int(rng, 1, min(16384, 2 ** 25 // k)), packed=rng.random() < 0.5)
    if kind == "linear":
        k, n = _log_int(rng, 64, 16384), _log_int(rng, 16, 16384)
        if rng.random() < 0.6:
            k, n = -(-k // 32) * 32, -(-n // 16) * 16
        most = max(1, min(8192, 2 ** 38 // (k * n), 2 ** 26 // n, 2 ** 26 // k))
        rows = rng.choice([1, rng.randint(1, min(64, most)), _log_int(rng, 1, most)])
        return dict(kind=kind, io=rng.choice(["f16", "bf16", "bf16", "f32", "mxfp4"]),
                    out=rng.choice(["f16", "bf16", "bf16", "f32"]), rows=rows, k=k, n=n,
                    bias=rng.random() < 0.5)
    if kind == "rotary":
        dim = rng.choice([32, 64, 80, 96, 128, 128, 256])
        rot = rng.choice([dim, dim, dim // 2, dim // 4, dim - 6])
        kvh = rng.choice([1, 2, 4, 8])
        heads = kvh * rng.choice([1, 2, 4, 7])
        most = 2 ** 26 // ((heads + kvh) * dim)
        batch = _log_int(rng, 1, min(256, most))
        rows = rng.choice([1, _log_int(rng, 1, min(8192, most // batch))])
        return dict(kind=kind, io=rng.choice(["f16", "bf16", "f32"]), heads=heads, kvh=kvh, dim=dim,
                    rot=rot, layout=rng.choice(["halves", "pairs"]), batch=batch, rows=rows,
                    shortest=rng.randint(1, rows), cached=_log_int(rng, 1, 1000000),
                    packed=rng.random() < 0.5, inverse=rng.random() < 0.3)
    slots, page = _log_int(rng, 1, 4096), rng.choice([16, 32, 64, 128])
    stride = _log_int(rng, 2, min(2048, 2 ** 21 // slots))
    room = stride * page
    return dict(kind=kind, slots=slots, stride=stride, page=page,
                new=rng.choice([1, _log_int(rng, 1, max(1, min(room // 3, 2 ** 22 // slots)))]),
                busy=rng.choice([1.0, rng.uniform(0.05, 1.0)]), cached=rng.randint(0, room // 2),
                tight=rng.random() < 0.2)


# ------------------------------------------------------------------- sizes


def _spread(lo, hi, n, phase):
    """n whole numbers over [lo, hi], the last of them hi."""
    got = [lo + int((hi - lo + 1) * (((i + 1) * 0.6180339887498949 + phase) % 1.0)) for i in range(n)]
    return got[:-1] + [hi]


def _rows_of(case):
    """Rows of each sequence of a rotary case, and its length with them."""
    rows = _spread(case["shortest"], case["rows"], case["batch"], 0.0)
    cached = _spread(0, case["cached"], case["batch"], 0.37)
    return rows, [r + c for r, c in zip(rows, cached)]


def _requests(case):
    """Lengths of a pages case's slots, and the new tokens of each."""
    n = case["slots"]
    lens = _spread(0, case["cached"], n, 0.37)
    want = _spread(1, case["new"], n, 0.11)
    idle = _spread(0, 9999, n, 0.73)
    new = [w if i < 10000 * case["busy"] else 0 for w, i in zip(want[:-1], idle[:-1])] + want[-1:]
    return lens, new


def _pages(tokens, page):
    return -(-tokens // page)


def work(case):
    kind = case["kind"]
    if kind == "quant":
        size = {"f16": 2, "bf16": 2, "f32": 4}[case["io"]]
        held = case["rows"] * _pages(case["k"], 32) * 17
        return {"bytes": 2 * (case["rows"] * case["k"] * size + held), "flops": 0}
    if kind == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        block = _pages(k, 32)
        x = m * (17 * block if case["io"] == "mxfp4" else k * (4 if case["io"] == "f32" else 2))
        y = m * n * (4 if case["out"] == "f32" else 2)
        return {"bytes": x + y + 17 * block * n + (4 * n if case["bias"] else 0),
                "flops": 2 * m * k * n}
    if kind == "rotary":
        rows, _ = _rows_of(case)
        size = 4 if case["io"] == "f32" else 2
        n = sum(rows) * (case["heads"] + case["kvh"])
        return {"bytes": 2 * n * case["dim"] * size, "flops": 3 * n * case["rot"]}
    lens, new = _requests(case)
    p, s = case["page"], case["slots"]
    live = [(t, n) for t, n in zip(lens, new) if n > 0]
    held = sum(_pages(t + n, p) for t, n in live)
    fresh = sum(_pages(t + n, p) - _pages(t, p) for t, n in live)
    # extend: requests, lengths twice; the batch; its table rows; rows. trim: back again.
    return {"bytes": 12 * s + 12 * len(live) + 8 * held + 8 * fresh + 12 * sum(new)
            + 12 * s + 12 * fresh, "flops": 0}


# ------------------------------------------------------------------ inputs


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        _bind(s)
    return s


def _wide(rows, k, dtype, pad=0):
    """Zeroed rows of k values whose distance is a multiple of 8."""
    return torch.zeros(rows, -(-(k + pad) // 8) * 8, dtype=dtype, device=DEV)[:, :k]


def _activations(rows, k, g):
    """Rows as a norm leaves them: a few large channels, tokens of unlike size."""
    x = torch.randn(rows, k, generator=g, device=DEV)
    x *= torch.exp(0.7 * torch.randn(k, generator=g, device=DEV))
    return x.mul_(torch.exp(0.3 * torch.randn(rows, 1, generator=g, device=DEV)))


def _inputs(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = {"case": case}
    kind = case["kind"]
    if kind == "quant":
        io, k = DTYPES[case["io"]], case["k"]
        s["x"] = _wide(case["rows"], k, io, 2 * k if case["packed"] else 0)
        s["x"].copy_(_activations(case["rows"], k, g))
        s["out"] = _wide(case["rows"], k, io)
        blocks = _pages(k, 32)
        s["codes"] = torch.zeros(case["rows"], 16 * blocks, dtype=torch.uint8, device=DEV)
        s["scales"] = torch.zeros(case["rows"], blocks, dtype=torch.uint8, device=DEV)
    elif kind == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        w = torch.randn(n, k, generator=g, device=DEV) / math.sqrt(k)
        w *= torch.exp(0.3 * torch.randn(n, 1, generator=g, device=DEV))
        s["w"], s["w_scales"] = _quantize(w)
        s["bias"] = torch.randn(n, generator=g, device=DEV) if case["bias"] else None
        x = _activations(m, k, g)
        if case["io"] == "mxfp4":
            s["x"], s["x_scales"] = _quantize(x)
        else:
            s["x"] = _wide(m, k, DTYPES[case["io"]])
            s["x"].copy_(x)
        s["out"] = _wide(m, n, DTYPES[case["out"]])
    elif kind == "rotary":
        rows, lens = _rows_of(case)
        io, d, h, kvh = DTYPES[case["io"]], case["dim"], case["heads"], case["kvh"]
        n, r = sum(rows), case["rot"]
        s["rows"], s["most_rows"] = n, max(rows)
        offsets = [0]
        for a in rows:
            offsets.append(offsets[-1] + a)
        s["offsets"] = torch.tensor(offsets, dtype=torch.int32, device=DEV)
        s["lengths"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        # Frequencies of a context stretched by four.
        s["freq"] = (10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64) / r) / 4.0).to(DEV)
        s["factor"] = 1.0 + 0.1 * math.log(4.0)
        if case["packed"]:  # slices of one projection's output, values behind them
            x = torch.randn(n, (h + 2 * kvh) * d, generator=g, device=DEV).to(io)
            s["q"], s["k"] = x[:, :h * d], x[:, h * d:(h + kvh) * d]
        else:
            s["q"] = torch.randn(n, h * d, generator=g, device=DEV).to(io)
            s["k"] = torch.randn(n, kvh * d, generator=g, device=DEV).to(io)
        s["q_out"] = torch.zeros(n, h * d, dtype=io, device=DEV)
        s["k_out"] = torch.zeros(n, kvh * d, dtype=io, device=DEV)
    else:
        lens, new = _requests(case)
        p, n, stride = case["page"], case["slots"], case["stride"]
        i32 = dict(dtype=torch.int32, device=DEV)
        held = torch.tensor([_pages(t, p) for t in lens])
        need = [_pages(t + a, p) if t + a <= stride * p else _pages(t, p)
                for t, a in zip(lens, new)]
        fresh = sum(need) - int(held.sum())
        spare = fresh // 2 if case["tight"] else fresh + 7
        pages = int(held.sum()) + spare
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).int()
        table = torch.full((n, stride), -1, dtype=torch.int32)
        table[torch.arange(stride) < held.unsqueeze(1)] = order[:int(held.sum())]
        free = torch.full((pages,), -1, dtype=torch.int32)
        free[:spare] = order[int(held.sum()):]
        batch, rows = sum(a > 0 for a in new), sum(new)
        s.update(pages=pages, batch=batch, rows=rows, want=sum(need) - int(held.sum()),
                 most=max(need), table=table.to(DEV), lengths=torch.tensor(lens, **i32),
                 free=free.to(DEV), free_count=torch.tensor([spare], **i32),
                 new=torch.tensor(new, **i32), keep=torch.tensor(lens, **i32),
                 b_slots=torch.zeros(n, **i32), b_lengths=torch.zeros(n, **i32),
                 b_offsets=torch.zeros(n + 1, **i32), b_table=torch.full((n, stride), -1, **i32),
                 positions=torch.zeros(rows, **i32),
                 slot_map=torch.zeros(rows, dtype=torch.int64, device=DEV))
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
    """The program's runtime, its layer, rotation or pager, and its buffers."""
    global _rt
    from eos_amd.runtime import Runtime
    if _rt is None:
        _rt = Runtime(0)
    case, kind = s["case"], s["case"]["kind"]
    dev = s["dev"] = {n: _Dev(t) for n, t in s.items() if isinstance(t, torch.Tensor)}
    torch.cuda.synchronize()  # the runtime's own stream does not wait for torch's
    if kind == "linear":
        from eos_amd.microscale import MXLinear
        s["layer"] = MXLinear(_rt, dev["w"], dev["w_scales"], case["n"], case["k"],
                              bias=dev.get("bias"))
    elif kind == "rotary":
        from eos_amd.kvcache import KVBatch
        from eos_amd.rotary import Rotary
        s["rotary"] = Rotary(_rt, case["dim"], s["freq"].cpu().numpy(), case["layout"], s["factor"])
        s["plan"] = KVBatch(None, 0, case["batch"], dev["lengths"],
                            None if s["most_rows"] == 1 else dev["offsets"], s["rows"])
    elif kind == "pages":
        from eos_amd.kvcache import KVPager, KVPlan
        s["pager"] = KVPager(_rt, case["slots"], case["stride"], case["page"], s["pages"],
                             page_table=dev["table"], lengths=dev["lengths"], free=dev["free"],
                             free_count=dev["free_count"])
        s["plan"] = KVPlan(dev["b_slots"], dev["b_table"], dev["b_lengths"], dev["b_offsets"],
                           dev["positions"], dev["slot_map"], s["rows"])


def _run_own(s):
    case, kind, dev = s["case"], s["case"]["kind"], s["dev"]
    if kind == "quant":
        from eos_amd import microscale
        microscale.quantize(_rt, dev["x"], case["rows"], case["k"], case["io"], dev["codes"],
                            dev["scales"], x_stride=s["x"].stride(0))
        microscale.dequantize(_rt, dev["codes"], dev["scales"], case["rows"], case["k"], dev["out"],
                              case["io"], out_stride=s["out"].stride(0))
        return s["out"]
    if kind == "linear":
        if case["io"] == "mxfp4":
            s["layer"].apply(dev["x"], case["rows"], "mxfp4", dev["out"], case["out"],
                             x_scales=dev["x_scales"], out_stride=s["out"].stride(0))
        else:
            s["layer"].apply(dev["x"], case["rows"], case["io"], dev["out"], case["out"],
                             x_stride=s["x"].stride(0), out_stride=s["out"].stride(0))
        return s["out"]
    if kind == "rotary":
        s["rotary"].apply(s["plan"], case["io"], dev["q"], case["heads"], dev["k"], case["kvh"],
                          q_out=dev["q_out"], k_out=dev["k_out"], q_stride=s["q"].stride(0),
                          k_stride=s["k"].stride(0), inverse=case["inverse"])
        return {"q": s["q_out"], "k": s["k_out"]}
    s["pager"].extend(dev["new"], s["plan"])
    s["pager"].trim(dev["keep"])
    return _state(s)


def _state(s):
    return {n: s[n] for n in ("b_slots", "b_lengths", "b_offsets", "b_table", "positions",
                              "slot_map", "table", "lengths", "free", "free_count")}


# --------------------------------------------------------------- plain forms


def _quantize(x):
    """Rows -> codes u8 [rows, 16 blocks] and scales u8 [rows, blocks]."""
    rows, k = x.shape
    x = torch.nn.functional.pad(x.float(), (0, -k % 32)).view(rows, -1, 32)
    most = x.abs().amax(-1, keepdim=True)
    e = (torch.frexp(most).exponent - 3).clamp(-127, 127)
    e = torch.where(most > 0, e, torch.full_like(e, -127))
    x = torch.ldexp(x, -e)
    a = x.abs()
    # Thresholds half way between levels; a tie goes to the even code.
    code = ((a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5)
            + (a > 5.0) + 8 * (x < 0))
    code = code.view(rows, -1, 2)
    return ((code[..., 0] | code[..., 1] << 4).to(torch.uint8),
            (e.squeeze(-1) + 127).to(torch.uint8))


def _values(codes, scales, k):
    """Codes and scales -> the f32 values they stand for [rows, k]."""
    rows = codes.shape[0]
    c = torch.stack([codes & 15, codes >> 4], -1).view(rows, -1, 32).long()
    level = torch.tensor(LEVELS + [-a for a in LEVELS], device=DEV)[c]
    return torch.ldexp(level, scales.int().unsqueeze(-1) - 127).flatten(1)[:, :k]


def _linear(s):
    case = s["case"]
    x, xs = (s["x"], s["x_scales"]) if case["io"] == "mxfp4" else _quantize(s["x"])
    y = _values(x, xs, case["k"]) @ _values(s["w"], s["w_scales"], case["k"]).T
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(DTYPES[case["out"]])


def _rotate(s):
    case = s["case"]
    d, r, off = case["dim"], case["rot"], s["offsets"].long()
    seq = torch.repeat_interleave(torch.arange(case["batch"], device=DEV), off[1:] - off[:-1],
                                  output_size=s["rows"])
    pos = torch.arange(s["rows"], device=DEV) - off[seq + 1] + s["lengths"].long()[seq]
    angle = pos.double().view(-1, 1, 1) * s["freq"]
    cos = (angle.cos() * s["factor"]).float()
    sin = (angle.sin() * (-s["factor"] if case["inverse"] else s["factor"])).float()
    got = {}
    for name in ("q", "k"):
        x = s[name].float().view(s["rows"], -1, d)
        if case["layout"] == "pairs":
            a, b = x[..., 0:r:2], x[..., 1:r:2]
        else:
            a, b = x[..., :r // 2], x[..., r // 2:r]
        a, b = a * cos - b * sin, a * sin + b * cos
        turned = torch.stack([a, b], -1).flatten(-2) if case["layout"] == "pairs" else torch.cat([a, b], -1)
        got[name] = torch.cat([turned, x[..., r:]], -1).flatten(1).to(DTYPES[case["io"]])
    return got


def _spans(counts, total):
    """For counts [n] of sum total: of every item its owner and place in it."""
    owner = torch.repeat_interleave(torch.arange(len(counts), device=DEV), counts, output_size=total)
    return owner, torch.arange(total, device=DEV) - (counts.cumsum(0) - counts)[owner]


def _extend(s):
    case = s["case"]
    p, stride, n = case["page"], case["stride"], case["slots"]
    lens, new, count = s["lengths"].long(), s["new"].long(), s["free_count"].long()
    held, want = (lens + p - 1) // p, (lens + new + p - 1) // p
    fits = lens + new <= stride * p
    need = torch.where(fits, want - held, torch.zeros_like(lens))
    upto = need.cumsum(0)
    granted = fits & ((need == 0) | (upto <= count))
    after = torch.where(granted, lens + new, lens)
    # New pages from the top of the stack, slot by slot (column `stride`: thrown away).
    owner, at = _spans(need, s["want"])
    page = s["free"][(count - 1 - torch.arange(s["want"], device=DEV)).clamp(min=0)]
    table = torch.nn.functional.pad(s["table"], (0, 1))
    table[owner, torch.where(granted[owner], held[owner] + at, stride)] = page
    s["table"].copy_(table[:, :stride])
    s["lengths"].copy_(after)
    s["free_count"].sub_(torch.where(granted, need, torch.zeros_like(need)).sum().int())
    # The batch: slots with new rows, in order.
    slots = torch.argsort((new <= 0).int(), stable=True)[:s["batch"]]
    rows = new[slots]
    length = torch.where(granted[slots], after[slots], torch.zeros_like(rows))
    s["b_slots"][:s["batch"]] = slots.int()
    s["b_lengths"][:s["batch"]] = length.int()
    s["b_offsets"][1:s["batch"] + 1] = rows.cumsum(0).int()
    live = torch.arange(stride, device=DEV) < ((length + p - 1) // p).unsqueeze(1)
    s["b_table"][:s["batch"]] = torch.where(live, s["table"][slots], s["b_table"][:s["batch"]])
    owner, at = _spans(rows, s["rows"])
    ok = granted[slots][owner]
    pos = lens[slots][owner] + at
    place = s["table"][slots[owner], (pos // p).clamp(max=stride - 1)].long() * p + pos % p
    s["positions"].copy_(torch.where(ok, pos, -1))
    s["slot_map"].copy_(torch.where(ok, place, -1))


def _trim(s):
    p, stride = s["case"]["page"], s["case"]["stride"]
    lens, keep = s["lengths"].long(), s["keep"].long()
    keep = torch.where((keep < 0) | (keep > lens), lens, keep)
    held, left = (lens + p - 1) // p, (keep + p - 1) // p
    col = torch.arange(stride, device=DEV)
    gone = (col >= left.unsqueeze(1)) & (col < held.unsqueeze(1))
    # Back onto the stack so that they come off again in order: the last goes first.
    rank = gone.flatten().cumsum(0) - 1
    total = rank[-1] + 1
    count = s["free_count"].long()
    to = torch.where(gone.flatten(), count + total - 1 - rank, len(s["free"]))
    free = torch.nn.functional.pad(s["free"], (0, 1))
    free[to] = s["table"].flatten()
    s["free"].copy_(free[:-1])
    s["free_count"].add_(total.int())
    s["table"].masked_fill_(gone, -1)
    s["lengths"].copy_(keep)


def run(s):
    if own:
        return _run_own(s)
    kind = s["case"]["kind"]
    if kind == "quant":
        codes, scales = _quantize(s["x"])
        return _values(codes, scales, s["case"]["k"]).to(DTYPES[s["case"]["io"]])
    if kind == "linear":
        return _linear(s)
    if kind == "rotary":
        return _rotate(s)
    _extend(s)
    _trim(s)
    return _state(s)


# ------------------------------------------------------------------- 64 bits


def _stands(x):
    """Rows f64 -> the f64 values that their MXFP4 form stands for."""
    rows, k = x.shape
    x = torch.cat([x, x.new_zeros(rows, -k % 32)], 1).unflatten(1, (-1, 32))
    top = torch.floor(torch.log2(x.abs().amax(2, keepdim=True).clamp(min=2.0 ** -200)))
    top = torch.where(2.0 ** top > x.abs().amax(2, keepdim=True), top - 1, top)  # (log2 rounds)
    unit = 2.0 ** (top - 2).clamp(-127, 127)
    a = (x / unit).abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    return (torch.sign(x) * (torch.round(a / step) * step).clamp(max=6.0) * unit).flatten(1)[:, :k]


def _held(codes, scales, k):
    """The f64 values of codes and scales, from the bits of their format."""
    c = torch.stack([codes % 16, codes // 16], 2).flatten(1).double()
    sign, c = torch.where(c >= 8, -1.0, 1.0).double(), c % 8
    ex = torch.floor(c / 2)
    mag = torch.where(ex == 0, 0.5 * c, 2.0 ** (ex - 1) * (1 + 0.5 * (c % 2)))
    unit = 2.0 ** (scales.double() - 127)
    return (sign * mag * unit.repeat_interleave(32, 1))[:, :k]


def exact(case, seed):
    """The definitions in 64 bits, from the inputs alone."""
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "quant":
        return _stands(s["x"].double())
    if kind == "linear":
        k = case["k"]
        x = _held(s["x"], s["x_scales"], k) if case["io"] == "mxfp4" else _stands(s["x"].double())
        y = torch.matmul(x, _held(s["w"], s["w_scales"], k).t().contiguous())
        return y if s["bias"] is None else y + s["bias"].double()
    if kind == "rotary":
        rows, lens = _rows_of(case)
        d, r = case["dim"], case["rot"]
        got = {n: torch.empty(s[n].shape, dtype=torch.float64, device=DEV) for n in ("q", "k")}
        at = 0
        for a, t in zip(rows, lens):
            turn = torch.polar(torch.full((a, r // 2), s["factor"], dtype=torch.float64, device=DEV),
                               torch.outer(torch.arange(t - a, t, device=DEV).double(), s["freq"]))
            if case["inverse"]:
                turn = turn.conj()
            for n in ("q", "k"):
                x = s[n][at:at + a].double().unflatten(1, (-1, d))
                y = x.clone()
                if case["layout"] == "pairs":
                    z = torch.complex(x[..., 0:r:2], x[..., 1:r:2]) * turn.unsqueeze(1)
                    y[..., 0:r:2], y[..., 1:r:2] = z.real, z.imag
                else:
                    z = torch.complex(x[..., :r // 2], x[..., r // 2:r]) * turn.unsqueeze(1)
                    y[..., :r // 2], y[..., r // 2:r] = z.real, z.imag
                got[n][at:at + a] = y.flatten(1)
            at += a
        return got
    # Request by request, as a scheduler on the host would go about it.
    p, stride = case["page"], case["stride"]
    lens, new = _requests(case)
    table, free = s["table"].cpu().numpy(), s["free"].cpu().numpy()
    left = used = int(s["free_count"])
    out = {n: s[n].cpu().numpy() for n in ("b_slots", "b_lengths", "b_offsets", "b_table",
                                           "positions", "slot_map")}
    j = row = 0
    asked = 0
    for i, (t, a) in enumerate(zip(lens, new)):
        if a == 0:
            continue
        have, want = _pages(t, p), _pages(t + a, p)
        fits = t + a <= stride * p
        asked += want - have if fits else 0
        ok = fits and (want == have or asked <= used)
        ids = list(table[i, :have])
        if ok:
            ids += [free[left - 1 - m] for m in range(want - have)]
            left -= want - have
            out["b_table"][j, :want] = ids
        out["b_slots"][j], out["b_lengths"][j] = i, t + a if ok else 0
        pos = torch.arange(t, t + a).numpy()
        out["positions"][row:row + a] = pos if ok else -1
        if ok:
            out["slot_map"][row:row + a] = torch.tensor(ids).numpy()[pos // p].astype("int64") * p + pos % p
        else:
            out["slot_map"][row:row + a] = -1
        row, j = row + a, j + 1
        out["b_offsets"][j] = row
    out = {n: torch.from_numpy(x).to(DEV) for n, x in out.items()}
    # Everything new is dropped again: the pages stand as they stood.
    return out | {n: s[n] for n in ("table", "lengths", "free", "free_count")}
