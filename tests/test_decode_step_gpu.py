"""A decoding step as a server runs it, on the device from the lengths of its
requests to its outputs: pages and positions planned, rows projected by layers
of 4-bit weights, turned, appended, attended and projected back; against the
same in 64 bits from what each call stored."""
import numpy as np
import pytest

import mx_reference as mx
from eos_amd.kvcache import KVCache, KVPager
from eos_amd.microscale import MXLinear
from eos_amd.rotary import Rotary, frequencies
from eos_amd.runtime import DeviceBuffer

pytestmark = pytest.mark.gpu

HEADS, KVH, D, HIDDEN, PAGE = 4, 2, 64, 192, 16


class Layer:
    def __init__(self, rt, rng, n, k):
        w = mx.to_bits(rng.normal(size=(n, k)) / np.sqrt(k), "bf16")
        self.w = mx.values(*mx.quantize(mx.from_bits(w, "bf16")), k)
        self.layer = MXLinear.from_rows(rt, DeviceBuffer.from_array(rt, w), n, k, "bf16")


def _softmax_rows(q, k, v, pos):
    """q [n, heads, d] at positions pos over k, v [t, kvh, d]."""
    out = np.zeros_like(q)
    for h in range(HEADS):
        x = q[:, h] @ k[:, h * KVH // HEADS].T / np.sqrt(D)
        x = np.where(np.arange(len(k)) <= pos[:, None], x, -np.inf)
        p = np.exp(x - x.max(1, keepdims=True))
        out[:, h] = (p / p.sum(1, keepdims=True)) @ v[:, h * KVH // HEADS]
    return out


@pytest.mark.parametrize("layout,rotary_dim", [("halves", D), ("pairs", 32)])
def test_steps_from_lengths_to_outputs(rt, layout, rotary_dim):
    print(f"[case] step {layout} {rotary_dim}", flush=True)
    rng = np.random.default_rng(rotary_dim)
    slots, stride, pages, most = 9, 12, 60, 300
    width = (HEADS + 2 * KVH) * D
    proj, back = Layer(rt, rng, width, HIDDEN), Layer(rt, rng, HIDDEN, HEADS * D)
    freq = frequencies(rotary_dim, scaling="linear", stretch=2)[0]
    rotary = Rotary(rt, D, freq, layout)
    pager = KVPager(rt, slots, stride, PAGE, pages)
    cache = KVCache(rt, "bf16", KVH, D, PAGE, pages)
    plan = pager.plan(most)
    buf = lambda n: DeviceBuffer(rt, n)  # noqa: E731
    x, qkv = buf(most * HIDDEN * 2), buf(most * width * 2)
    att, out = buf(most * HEADS * D * 2), buf(most * HIDDEN * 2)
    held = [np.zeros((2, 0, KVH, D)) for _ in range(slots)]  # keys (turned), values

    def step(new, positions):
        new = np.asarray(new, np.int32)
        batch, rows = int((new > 0).sum()), int(new.sum())
        xb = mx.to_bits(rng.normal(size=(rows, HIDDEN)), "bf16")
        x.upload(xb)
        pager.extend(DeviceBuffer.from_array(rt, new), plan)
        b = plan.batch(stride, batch, None if rows == batch else rows)
        proj.layer.apply(x, rows, "bf16", qkv)
        q, k, v = (qkv.view(a * D * 2, qkv.nbytes - a * D * 2) for a in (0, HEADS, HEADS + KVH))
        where = (plan.positions, rows) if positions else b
        rotary.apply(where, "bf16", q, HEADS, k, KVH, q_stride=width, k_stride=width)
        cache.append(b, k, v, "bf16", width, width)
        cache.attend(b, q, HEADS, att, "bf16", q_stride=width)
        back.layer.apply(att, rows, "bf16", out)
        assert pager.status() == 0 and cache.status() == 0
        got = mx.from_bits(qkv.download(np.uint16, (rows, width)), "bf16")
        # the projection, turned: bf16 twice
        want, tol = mx.linear(mx.values(*mx.quantize(mx.from_bits(xb, "bf16")), HIDDEN), proj.w, None,
                              "bf16")
        pos = np.concatenate([held[s].shape[1] + np.arange(n) for s, n in enumerate(new) if n])
        r = rotary_dim
        p = want.reshape(rows, -1, D)
        i, j = (slice(0, r, 2), slice(1, r, 2)) if layout == "pairs" else (slice(0, r // 2), slice(r // 2, r))
        c, s = np.cos(pos[:, None, None] * freq), np.sin(pos[:, None, None] * freq)
        turned = p.copy()
        turned[:, :, i], turned[:, :, j] = p[:, :, i] * c - p[:, :, j] * s, p[:, :, i] * s + p[:, :, j] * c
        turned[:, HEADS + KVH:] = p[:, HEADS + KVH:]
        size, t = np.abs(p), tol.reshape(p.shape)
        for y in (size, t):
            y[:, :HEADS + KVH, i] = y[:, :HEADS + KVH, j] = y[:, :HEADS + KVH, i] + y[:, :HEADS + KVH, j]
        bound = t + mx.U["bf16"] * (np.abs(turned) + t) + 32 * mx.U["f32"] * size
        assert (np.abs(got.reshape(p.shape) - turned) <= bound).all()
        # attention over everything stored so far, from the rows as they were stored
        rows_of = got.reshape(rows, -1, D)
        at, want_att = 0, []
        for sl, n in enumerate(new):
            if not n:
                continue
            kv = np.stack([rows_of[at:at + n, HEADS:HEADS + KVH], rows_of[at:at + n, HEADS + KVH:]])
            held[sl] = np.concatenate([held[sl], kv], 1)
            total = held[sl].shape[1]
            want_att.append(_softmax_rows(rows_of[at:at + n, :HEADS], *held[sl], np.arange(total - n, total)))
            at += n
        a = mx.from_bits(att.download(np.uint16, (rows, HEADS * D)), "bf16")
        # weights rounded to bf16, twice the largest value's half step at most, and the result's
        big = max(np.abs(h[1]).max() for h in held if h.size)
        assert np.abs(a - np.concatenate(want_att).reshape(a.shape)).max() <= 3.5 * mx.U["bf16"] * big
        want, tol = mx.linear(mx.values(*mx.quantize(a), HEADS * D), back.w, None, "bf16")
        got = mx.from_bits(out.download(np.uint16, (rows, HIDDEN)), "bf16")
        assert (np.abs(got - want) <= tol).all()

    def trim(keep):
        pager.trim(DeviceBuffer.from_array(rt, np.asarray(keep, np.int32)))
        for s, k in enumerate(keep):
            if 0 <= k < held[s].shape[1]:
                held[s] = held[s][:, :k]

    step([33, 0, 5, 70, 0, 1, 16, 0, 0], False)    # prompts
    step([1, 0, 1, 1, 0, 1, 1, 0, 0], True)        # a token each
    step([3, 17, 2, 1, 0, 4, 1, 40, 0], True)      # drafts, new requests beside them
    trim([35, -1, 7, -1, -1, 2, -1, -1, -1])       # drafts dropped
    trim([-1, -1, -1, 0, -1, -1, -1, -1, -1])      # a request over
    step([1, 1, 1, 0, 90, 1, 1, 1, 2], False)      # its pages given to others
    step([1, 1, 1, 0, 1, 1, 1, 1, 1], True)


@pytest.mark.parametrize("one_each", [True, False])
def test_a_refused_request_is_padding(rt, one_each):
    """Requests that the pages do not cover: no row of theirs is turned, stored
    or attended, and nothing of the others' changes."""
    rng = np.random.default_rng(1)
    pager = KVPager(rt, 4, 3, PAGE, 3)
    cache = KVCache(rt, "bf16", KVH, D, PAGE, 3)
    plan = pager.plan(64)
    rotary = Rotary(rt, D, frequencies(D)[0])
    i32 = lambda a: DeviceBuffer.from_array(rt, np.asarray(a, np.int32))  # noqa: E731
    width = (HEADS + 2 * KVH) * D
    pager.extend(i32([16, 15, 0, 0]), plan)  # a page each, one left
    x = mx.to_bits(rng.normal(size=(31, width)), "bf16")
    qkv = DeviceBuffer.from_array(rt, x)
    part = lambda b, a: b.view(a * D * 2, b.nbytes - a * D * 2)  # noqa: E731
    b = plan.batch(3, 2, 31)
    cache.append(b, part(qkv, HEADS), part(qkv, HEADS + KVH), "bf16", width, width)
    new = [1, 1, 1, 1] if one_each else [2, 1, 17, 3]
    rows = sum(new)
    pager.extend(i32(new), plan)             # the first takes it, the third and fourth wait
    assert pager.status() == 1
    assert plan.lengths.download(np.int32, (4,)).tolist() == [16 + new[0], 16, 0, 0]
    x = mx.to_bits(rng.normal(size=(rows, width)), "bf16")
    qkv = DeviceBuffer.from_array(rt, x)
    b = plan.batch(3, 4, None if one_each else rows)
    before = [p.download(np.uint16, (p.nbytes // 2,)) for p in (cache.k, cache.v)]
    live = new[0] + new[1]
    for where in (b, (plan.positions, rows)):
        rotary.apply(where, "bf16", qkv, HEADS, part(qkv, HEADS), KVH, q_stride=width, k_stride=width)
        got = qkv.download(np.uint16, x.shape)
        np.testing.assert_array_equal(got[live:], x[live:])
        assert (got[:live, :HEADS * D] != x[:live, :HEADS * D]).any(1).all()
    cache.append(b, part(qkv, HEADS), part(qkv, HEADS + KVH), "bf16", width, width)
    after = [p.download(np.uint16, (p.nbytes // 2,)) for p in (cache.k, cache.v)]
    for p, q in zip(before, after):
        assert (p != q).sum() <= live * KVH * D
    out = DeviceBuffer.from_array(rt, np.full((rows, HEADS * D), 0x4141, np.uint16))
    cache.attend(b, qkv, HEADS, out, "bf16", q_stride=width)
    got = out.download(np.uint16, (rows, HEADS * D))
    assert (got[live:] == 0).all() and (got[:live] != 0).any(1).all()
    assert cache.status() == 0


def test_every_kernel_is_reached(rt):
    """Each variant by a call that takes it."""
    types = ("f16", "bf16", "f32")
    names = [f"eos_mx_{op}_{t}" for op in ("quantize", "dequantize", "lay") for t in types]
    names += ["eos_mx_lay_codes"] + [f"eos_mx_product_{n}_{t}" for n in (64, 128, 256) for t in types]
    names += [f"eos_mx_few_{t}_4_{n}" for t in types for n in (1, 2)]
    names += [f"eos_mx_few_{t}_16_{n}" for t in types for n in (1, 2, 4)]
    names += [f"eos_mx_few_codes_16_{n}" for n in (1, 2)]
    names += [f"eos_mx_few_laid_{m}_{n}" for m in (32, 48, 64) for n in (1, 2)]
    rng = np.random.default_rng(0)
    cus = rt.info()["compute_units"]
    big = DeviceBuffer.from_array(rt, np.zeros(96 << 20, np.uint8))

    def layer(n, k):
        c, s = mx.quantize(rng.normal(size=(n, k)))
        return MXLinear(rt, DeviceBuffer.from_array(rt, c), DeviceBuffer.from_array(rt, s), n, k)

    widths = {1: layer(16 * cus, 32), 2: layer(16 * cus + 1, 32), 4: layer(32 * cus + 1, 32)}

    def calls():
        from eos_amd import microscale
        for t in types:
            microscale.quantize(rt, big, 2, 32, t, big.view(4096, 4096), big.view(8192, 4096))
            microscale.dequantize(rt, big.view(4096, 4096), big.view(8192, 4096), 2, 32, big, t)
            for w in widths.values():
                for rows in (1, 16, 20):
                    w.apply(big, rows, t, big.view(48 << 20, 48 << 20), "f16", out_stride=32 * cus + 8)
        for w in widths.values():
            w.apply(big, 3, "mxfp4", big.view(48 << 20, 48 << 20), "f16", out_stride=32 * cus + 8,
                    x_scales=big)
            for rows in (40, 60):
                w.apply(big, rows, "mxfp4", big.view(48 << 20, 48 << 20), "f16",
                        out_stride=32 * cus + 8, x_scales=big)
        small = layer(64, 32)
        for t in types:
            small.apply(big, 65, "f16", big.view(48 << 20, 48 << 20), t)
            small.apply(big, 64 * 2 * cus + 1, "f16", big.view(48 << 20, 48 << 20), t)
            widths[1].apply(big, 4096, "f16", big.view(16 << 20, 80 << 20), t)

    rt.profile(True)
    rt.profile_reset()
    calls()
    rt.sync()
    seen = {n for n in names if rt.profile_read(n)[0] > 0}  # (none begins with another)
    rt.profile(False)
    rt.profile_reset()
    assert seen == set(names), sorted(set(names) - seen)
