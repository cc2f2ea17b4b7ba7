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

from eos_amd import microscale  # noqa: E402
from eos_amd._lib import EosHipError  # noqa: E402
from eos_amd.microscale import MXLinear  # noqa: E402
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


if __name__ == "__main__":
    globals()[sys.argv[2]]()
    print("OK")
