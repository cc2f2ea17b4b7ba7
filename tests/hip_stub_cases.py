"""Calls on the host's stand-in for devices (tests/hip_stub.cpp), each in a
process of its own: python hip_stub_cases.py STUB CASE."""
import ctypes as C
import os
import sys

stub = C.CDLL(sys.argv[1], C.RTLD_GLOBAL)  # before the library, whose calls it takes
stub.stub_device_of.argtypes = [C.c_void_p]
stub.stub_launches.argtypes = [C.c_char_p]
stub.stub_launches.restype = C.c_long
sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import numpy as np  # noqa: E402

from eos_amd import _lib, microscale  # noqa: E402
from eos_amd._lib import EosHipError  # noqa: E402
from eos_amd.kvcache import KVBatch, KVCache, KVPager, KVPlan  # noqa: E402
from eos_amd.microscale import MXLinear  # noqa: E402
from eos_amd.rotary import Rotary  # noqa: E402
from eos_amd.runtime import DeviceBuffer, Runtime  # noqa: E402


def refused(what, call, *args, **kw):
    try:
        call(*args, **kw)
    except EosHipError as e:
        assert what in str(e), f"refused with {e}, not {what}"
        return
    raise AssertionError(f"not refused: {what}")


def linear_overlap():
    """Outputs among the rows that a layer reads, or beside them."""
    rt = Runtime(0)
    n, k = 48, 64
    layer = MXLinear(rt, DeviceBuffer(rt, n * 32), DeviceBuffer(rt, n * 2), n, k)
    buf = DeviceBuffer(rt, 1 << 16)
    part = lambda at: buf.view(at, buf.nbytes - at)  # noqa: E731
    for rows in (1, 16, 17, 40, 100):
        refused("out overlaps x", layer.apply, buf, rows, "bf16", buf)
        refused("out overlaps x", layer.apply, buf, rows, "f32", part(rows * k * 4 - 16))
        refused("out overlaps x", layer.apply, part(rows * n * 2 - 16), rows, "f16", buf)
        layer.apply(buf, rows, "bf16", part(rows * k * 2))
        layer.apply(part(rows * n * 2), rows, "bf16", buf)
        # columns of one wider array: beside each other, then one into the other
        layer.apply(buf, rows, "bf16", part(k * 2), x_stride=112, out_stride=112)
        refused("out overlaps x", layer.apply, buf, rows, "bf16", part(k * 2 - 16), x_stride=112,
                out_stride=112)
        refused("out overlaps x", layer.apply, buf, rows, "mxfp4", part(rows * 32 - 16), "bf16",
                x_scales=part(1 << 15))
        refused("out overlaps x's scales", layer.apply, buf, rows, "mxfp4", part(rows * 32), "bf16",
                x_scales=part(rows * 32 + rows * 96 - 1))
        layer.apply(buf, rows, "mxfp4", part(rows * 32), "bf16", x_scales=part(rows * 32 + rows * 96))
    assert rows > 64 and stub.stub_launches(b"eos_mx_product_64_bf16") == 4


def rows_overlap():
    """Codes, scales and values in each other's place."""
    rt = Runtime(0)
    buf = DeviceBuffer(rt, 1 << 16)
    part = lambda at: buf.view(at, buf.nbytes - at)  # noqa: E731
    rows, k = 20, 96  # x 192 bytes a row, codes 48, scales 3
    x, c, s = rows * 192, rows * 48, rows * 3
    q = lambda *a, **kw: microscale.quantize(rt, *a, **kw)  # noqa: E731
    q(buf, rows, k, "bf16", part(x), part(x + c))
    q(part(c + 64), rows, k, "bf16", buf, part(c))
    refused("codes or scales overlap x", q, buf, rows, k, "bf16", part(x - 16), part(1 << 15))
    refused("codes or scales overlap x", q, part(16), rows, k, "bf16", part(1 << 15), part(16 + x - 1))
    refused("scales overlap codes", q, buf, rows, k, "bf16", part(1 << 15), part((1 << 15) + c - 1))
    # behind a row's values
    q(buf, 1, k, "bf16", part(256), part(192), x_stride=96)
    d = lambda *a, **kw: microscale.dequantize(rt, *a, **kw)  # noqa: E731
    d(buf, part(c), rows, k, part(c + 64), "bf16")
    d(part(x), part(x + c), rows, k, buf, "bf16")
    refused("out overlaps codes or scales", d, buf, part(1 << 15), rows, k, part(c - 16), "f32")
    refused("out overlaps codes or scales", d, part(1 << 15), buf, rows, k, part(s - s % 16), "f16")
    refused("out overlaps codes or scales", d, part(16), part(1 << 15), rows, k, buf, "f16", out_stride=104)
    assert stub.stub_launches(b"eos_mx_quantize_bf16") == 3


def rotary_overlap():
    """Turned rows in the place of others, or of their positions."""
    rt = Runtime(0)
    d, rows = 64, 10
    rot = Rotary(rt, d, np.ones(d // 2))
    buf, pos = DeviceBuffer(rt, 1 << 18), DeviceBuffer(rt, 4 * rows)
    part = lambda at: buf.view(at, buf.nbytes - at)  # noqa: E731
    where = (pos, rows)
    far = part(1 << 17)

    def turn(q=None, k=None, q_out=None, k_out=None, stride=6 * d, at=where, **kw):
        rot.apply(at, "bf16", q, 4 if q else 0, k, 2 if k else 0, q_out, k_out, stride, stride, **kw)

    packed = dict(q=buf, k=part(4 * d * 2))  # q | k, two bytes a value
    turn(**packed)
    turn(**packed, q_out=far, k_out=part((1 << 17) + 4 * d * 2), q_out_stride=6 * d, k_out_stride=6 * d)
    turn(**packed, q_out=far)                                # the keys stay where they are
    turn(**packed, k_out=far)
    turn(q=buf, k=far, q_out=part(6 * d * 2 * rows))
    refused("q_out overlaps k", turn, q=buf, k=part(4 * d * 2 - 16))
    refused("q_out overlaps k", turn, q=buf, k=buf)
    refused("q_out overlaps q", turn, q=buf, q_out=part(16), q_out_stride=6 * d)
    refused("q_out overlaps q", turn, q=far, q_out=part((1 << 17) - 4 * d * 2 * rows + 16))
    refused("k_out overlaps k", turn, k=buf, k_out=part(6 * d * 2), k_out_stride=8 * d)
    refused("k_out overlaps q", turn, q=buf, k=far, q_out=part(1 << 16), k_out=part(2 * d * 2), k_out_stride=6 * d)
    refused("q_out overlaps k_out", turn, q=buf, k=part(4 * d * 2), q_out=far, k_out=far)
    refused("an output overlaps positions", turn, q=buf, at=(part(6 * d * 2 * 9 + 4 * d * 2 - 16), rows))
    turn(q=buf, at=(part(6 * d * 2 * 9 + 4 * d * 2), rows))
    i32 = DeviceBuffer(rt, 4096)
    turn(q=buf, at=KVBatch(None, 0, rows, i32))
    refused("an output overlaps positions", turn, q=buf, at=KVBatch(None, 0, rows, buf))
    refused("an output overlaps positions", turn, k=buf, at=KVBatch(None, 0, 3, i32, buf, rows))
    assert stub.stub_launches(b"eos_rot_halves_bf16") == 7


def pager_overlap():
    """A pager's arrays, a plan's and a call's in each other's place, by a byte of
    their last element or whole."""
    rt = Runtime(0)
    slots, stride, pages, rows = 6, 5, 40, 32
    size = dict(page_table=4 * slots * stride, lengths=4 * slots, free=4 * pages, free_count=4)
    plan_size = dict(slots=4 * slots, page_table=4 * slots * stride, lengths=4 * slots,
                     offsets=4 * slots + 4, positions=4 * rows, slot_map=8 * rows)
    buf = DeviceBuffer(rt, 1 << 16)
    at = {}  # every array's place, one behind the other

    def place(names, sizes, first):
        for n in names:
            first = -(-first // 8) * 8
            at[n] = buf.view(first, sizes[n.split(".")[-1]])
            first += sizes[n.split(".")[-1]]
        return first

    end = place([f"own.{n}" for n in size], size, 0)
    end = place([f"plan.{n}" for n in plan_size], plan_size, end)
    new = buf.view(-(-end // 8) * 8, 4 * slots)
    own = {n: at[f"own.{n}"] for n in size}
    pager = KVPager(rt, slots, stride, 16, pages, **own)

    def plan(**kw):
        return KVPlan(**({n: at[f"plan.{n}"] for n in plan_size} | dict(rows=rows) | kw))

    pager.extend(new, plan())
    pager.extend(new, plan(page_table=None, positions=None, slot_map=None))
    pager.extend(own["lengths"], plan())  # read before they are written
    pager.trim(own["lengths"])
    pager.trim(new)
    n = 0
    for name in plan_size:
        first = at[f"plan.{name}"].ptr.value
        others = [(w, a) for w, a in at.items() if w != f"plan.{name}"]
        for where, other in others:
            for put in (other.ptr.value, other.ptr.value + other.nbytes - 8, other.ptr.value - plan_size[name] + 8):
                put -= buf.ptr.value + (put - buf.ptr.value) % 8
                if put < 0 or put + buf.ptr.value == first:
                    continue
                # (a place may also meet a third array; that is refused as well)
                moved = buf.view(put, plan_size[name])
                refused("a plan's arrays overlap", pager.extend, new, plan(**{name: moved}))
                n += 1
        refused("new overlaps", pager.extend, buf.view(first - buf.ptr.value, 4 * slots), plan())
    assert n > 100
    for name, what in (("page_table", "new overlaps"),):
        refused(what, pager.extend, buf.view(own[name].ptr.value - buf.ptr.value + 8, 4 * slots), plan())
    for name in ("page_table", "free"):
        refused("keep overlaps", pager.trim, buf.view(own[name].ptr.value - buf.ptr.value + 8, 4 * slots))
    for a in size:
        for b in size:
            if a != b and size[a] <= size[b]:
                refused("arrays overlap", KVPager, rt, slots, stride, 16, pages,
                        **(own | {a: buf.view(own[b].ptr.value - buf.ptr.value + size[b] - size[a], size[a])}))
    # without lists their sizes do not count
    pager.extend(new, plan(positions=None, slot_map=None, rows=1 << 30))


def rotary_alignment():
    """Positions, lengths and offsets are read as words: wherever else they stand,
    a scalar load takes others."""
    rt = Runtime(0)
    rot = Rotary(rt, 64, np.ones(32))
    buf, i32 = DeviceBuffer(rt, 1 << 16), DeviceBuffer(rt, 4096)
    for at in (1, 2, 3):
        odd = i32.view(at, 2048)
        refused("4-byte aligned", rot.apply, (odd, 3), "f16", buf, 1)
        refused("4-byte aligned", rot.apply, KVBatch(None, 0, 3, odd), "f16", buf, 1)
        refused("4-byte aligned", rot.apply, KVBatch(None, 0, 3, i32, odd, 3), "f16", buf, 1)
    rot.apply((i32.view(4, 2048), 3), "f16", buf, 1)


def another_current_device():
    """A runtime's memory is its own device's, whichever the program made current,
    and that one stays current."""
    near, far = Runtime(0), Runtime(1)
    for rt, device in ((near, 0), (far, 1)):
        for current in (0, 1):
            stub.stub_set_device(current)
            own = lambda b: stub.stub_device_of(b.ptr) == device  # noqa: E731
            buf = DeviceBuffer(rt, 4096)
            assert own(buf) and stub.stub_device() == current
            layer = MXLinear.from_rows(rt, buf, 16, 32, "f32")
            layer.apply(buf, 20, "f16", DeviceBuffer(rt, 4096), "f16")
            pager = KVPager(rt, 3, 2, 16, 9)
            plan = pager.plan(8)
            assert all(map(own, (pager.page_table, pager.free, plan.slots, plan.slot_map)))
            pager.extend(DeviceBuffer(rt, 12), plan)
            pager.trim(DeviceBuffer(rt, 12))
            assert pager.status() == 0
            cache = KVCache(rt, "q8", 1, 32, 16, 2)
            assert own(cache.k) and own(cache.v_scale)
            Rotary(rt, 32, np.ones(16)).apply((buf, 3), "f16", DeviceBuffer(rt, 256), 1)
            for x in (layer, pager, cache):
                x.release()
            assert stub.stub_device() == current


def largest_calls():
    """The most that a call takes is what its documentation says, and more is
    refused by that name before anything is enqueued."""
    rt = Runtime(0)
    near, far = C.c_void_p(1 << 20), C.c_void_p(1 << 60)
    quant = lambda rows, k: _lib.call(  # noqa: E731
        "eoship_mx_quantize_device", rt.handle, near, -(-k // 8) * 8, 1, rows, k, far, 1 << 61)
    back = lambda rows, k: _lib.call(  # noqa: E731
        "eoship_mx_dequantize_device", rt.handle, far, 1 << 61, rows, k, near, -(-k // 8) * 8, 1)
    for rows, k in ((2 ** 30 - 64, 32), (2 ** 30 - 64, 1), (2 ** 29 - 32, 64), (2 ** 11 - 1, 2 ** 24)):
        quant(rows, k)
        back(rows, k)
    for rows, k in ((2 ** 30 - 63, 32), (2 ** 29 - 31, 33), (2 ** 11, 2 ** 24), (2 ** 31 - 1, 1)):
        refused("more than 2^30 - 64 blocks", quant, rows, k)
        refused("more than 2^30 - 64 blocks", back, rows, k)
    handle = C.c_void_p()
    bind = lambda n, k: _lib.call(  # noqa: E731
        "eoship_mx_bind", rt.handle, near, far, n, k, None, C.byref(handle))
    refused("more than 2^24 - 1 tiles of 32 rows by 256", bind, 2 ** 13, 2 ** 24)
    refused("more than 2^24 - 1 tiles of 32 rows by 256", bind, 2 ** 24, 2 ** 13)
    layer = MXLinear(rt, DeviceBuffer(rt, 16 * 16), DeviceBuffer(rt, 16), 16, 32)
    apply = lambda rows: _lib.call(  # noqa: E731
        "eoship_mx_linear_device", rt.handle, layer.handle, near, 32, 1, None, rows, far, 16, 1)
    refused("more than 2^24 - 1 tiles of 32 rows by 256", apply, 2 ** 29)
    d = 1024
    turn = lambda rot, rows: _lib.call(  # noqa: E731
        "eoship_rotary_device", rt.handle, rot.handle, None, far, rows, 0, 1, near, d, 1, near, d,
        None, 0, 0, None, 0)
    for half, each in ((512, 1), (256, 1), (64, 4), (48, 5), (4, 16)):
        rot = Rotary(rt, d, np.ones(half))
        most = min((2 ** 24 - 1) * each, 2 ** 31 - 1)
        turn(rot, most)
        refused(f"more than {most} rows", turn, rot, most + 1)


if __name__ == "__main__":
    globals()[sys.argv[2]]()
    print("OK")
