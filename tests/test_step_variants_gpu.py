"""Page tables by many workgroups and of long table rows, and rotary positions of
many heads: the forms that large servers take, against plain loops and 64 bits."""
import numpy as np
import pytest

from eos_amd.kvcache import KVBatch
from eos_amd.rotary import Rotary, frequencies
from eos_amd.runtime import DeviceBuffer
from mx_reference import from_bits, to_bits
from test_kv_pager_gpu import World
from test_rotary_gpu import Rows, _check, _turned

pytestmark = pytest.mark.gpu


# A workgroup has 2,048 table entries or rows; from 64 of them on they are counted in
# eight groups, and a table row of more than 256 pages is moved in pieces.
@pytest.mark.parametrize("slots,stride,rows,blocks", [
    (130, 1024, 40000, 65), (134, 1024, 40000, 67), (100, 2000, 90000, 97), (1500, 99, 100000, 72),
    (70, 300, 300000, 146), (1025, 300, 200000, 150), (4096, 300, 260000, 600)])
def test_many_workgroups(rt, slots, stride, rows, blocks):
    print(f"[case] slots {slots} stride {stride} rows {rows}", flush=True)
    assert max(slots * stride, rows) // 2048 == blocks
    rng = np.random.default_rng(slots + stride)
    page, room = 16, stride * 16
    w = World(rt, slots, stride, page, slots * min(stride, 24) + 9 * stride, rows)
    kernel = "some" if slots <= 1024 else "many"
    rt.profile(True)
    rt.profile_reset()
    for i in range(5):
        # short requests for most, a few that fill a table row's pieces
        new = np.where(rng.random(slots) < 0.8, rng.integers(1, 9, slots), 0)
        some = rng.integers(0, slots, slots // 20 + 1)
        new[some] = rng.integers(1, 1 + min(room, 4 * rows // (10 * len(some))), len(some))
        long = rng.integers(0, slots, 3)
        new[long] = np.minimum(room - w.ref.lengths[long], rows // 8)
        if i == 3:
            new[:] = 1
        w.extend(new)
        keep = np.where(rng.random(slots) < 0.4, rng.integers(0, room, slots), -1)
        keep[long] = np.where(rng.random(3) < 0.5, rng.integers(0, room // 3, 3), -1)
        w.trim(np.where(rng.random(slots) < 0.1, 0, keep))
    taken = [rt.profile_read(f"eos_pager_{op}_{kernel}")[0] for op in ("extend", "trim")]
    rt.profile(False)
    rt.profile_reset()
    assert taken == [5, 5]


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("d,r", [(128, 32), (128, 128), (64, 32)])
@pytest.mark.parametrize("heads,kvh", [(32, 8), (7, 2)])
def test_pairs_of_many_heads(rt, dtype, d, r, heads, kvh):
    """Heads of several rows in flight together, rows of padding among them."""
    print(f"[case] {dtype} {heads}+{kvh} x {d}/{r}", flush=True)
    rng = np.random.default_rng(d + r + heads)
    cus = rt.info()["compute_units"]
    n = rng.integers(0, 90, 130)
    n[3] = 9 * cus - n.sum() + n[3] + 7 if n.sum() < 9 * cus else n[3]
    n[60] += 1
    lens = n + rng.integers(0, 100000, len(n))
    lens[rng.integers(0, len(n), 20)] = 0  # padding
    lens[60] = n[60] - 1 if n[60] > 1 else 1  # and rows in front of a sequence
    off = np.concatenate([[0], n.cumsum()])
    rows = int(off[-1]) + 5
    assert rows > 8 * cus  # two rows a workgroup at least
    pos = np.full(rows, -1, np.int64)
    for b in range(len(n)):
        pos[off[b]:off[b + 1]] = lens[b] - n[b] + np.arange(n[b])
    live = pos >= 0
    assert (~live).sum() > 100
    x = Rows(rt, rng, rows, heads, kvh, d, dtype)
    freq, factor = frequencies(r, scaling="linear", stretch=4)[0], 1.125
    rot = Rotary(rt, d, freq, "pairs", factor)
    i32 = lambda a: DeviceBuffer.from_array(rt, np.asarray(a, np.int32))  # noqa: E731
    batch = KVBatch(None, 0, len(n), i32(lens), i32(off), rows)
    gaps = {w: to_bits(np.full((rows, m * d + 8), 776.0), dtype) for w, m in (("q", heads), ("k", kvh))}
    out = {w: DeviceBuffer.from_array(rt, g) for w, g in gaps.items()}
    rot.apply(batch, dtype, x.part(x.dev, "q"), heads, x.part(x.dev, "k"), kvh, out["q"], out["k"],
              x.width, x.width, heads * d + 8, kvh * d + 8)
    rot.apply(batch, dtype, x.part(x.dev, "q"), heads, x.part(x.dev, "k"), kvh, q_stride=x.width,
              k_stride=x.width)
    here = x.dev.download(x.bits.dtype, x.bits.shape)
    np.testing.assert_array_equal(here[~live], x.bits[~live])
    np.testing.assert_array_equal(here[:, (heads + kvh) * d:], x.bits[:, (heads + kvh) * d:])
    for w, m in (("q", heads), ("k", kvh)):
        got = out[w].download(gaps[w].dtype, gaps[w].shape)
        np.testing.assert_array_equal(got[~live], gaps[w][~live])
        np.testing.assert_array_equal(got[:, m * d:], gaps[w][:, m * d:])
        got = from_bits(got[:, :m * d], dtype)
        want, e = _turned(x.values(x.bits, w)[live], pos[live], freq, "pairs", factor)
        _check(got[live].reshape(want.shape), want, e, dtype)
        np.testing.assert_array_equal(x.values(here, w)[live].reshape(want.shape), got[live].reshape(want.shape))
