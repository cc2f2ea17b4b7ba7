"""The paged key-value cache on the host: the kernels' index arithmetic walked
over random sound and damaged batches, sizes, and refusals (no GPU call)."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from eos_amd import _lib
from eos_amd._lib import EosHipError
from eos_amd.kvcache import KVBatch, check_batch, gaussian_codebook, kv_bytes

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_work_units_cover_every_row_and_stay_inside(tmp_path):
    exe = str(tmp_path / "kv_index_check")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror",
                    "-fsanitize=address,undefined", "-fno-sanitize-recover=undefined",
                    "-I", os.path.join(ROOT, "eos_amd", "csrc", "kernels"), "-o", exe,
                    os.path.join(ROOT, "tests", "kv_index_check.cpp")], check=True)
    r = subprocess.run([exe, "1500"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "OK", r.stdout + r.stderr


@pytest.mark.parametrize("fmt,bits", [("f16", 16), ("bf16", 16), ("q8", 8), ("tq4", 4)])
def test_pool_sizes(fmt, bits):
    pool, scale = kv_bytes(fmt, 8, 128, 64, 1000)
    assert pool == 1000 * 8 * 64 * 128 * bits // 8
    assert scale == (1000 * 8 * 64 * 4 if bits < 16 else 0)


@pytest.mark.parametrize("kw,what", [
    (dict(kv_heads=0), "kv_heads"), (dict(kv_heads=1025), "kv_heads"),
    (dict(head_dim=96), "head_dim"), (dict(head_dim=0), "head_dim"),
    (dict(page_tokens=8), "page_tokens"), (dict(page_tokens=48), "page_tokens"),
    (dict(page_tokens=512), "page_tokens"), (dict(pages=0), "pages"),
    (dict(pages=2 ** 31), "pages"),
])
def test_descriptor_refusals(kw, what):
    base = dict(fmt="q8", kv_heads=2, head_dim=64, page_tokens=16, pages=4) | kw
    with pytest.raises(EosHipError, match=what):
        kv_bytes(**base)


def test_unknown_format_refused():
    with pytest.raises(ValueError, match="format"):
        kv_bytes("q5", 1, 64, 16, 1)
    d = _lib.EosHipKVDesc(format=7, kv_heads=1, head_dim=64, page_tokens=16, pages=1)
    with pytest.raises(EosHipError, match="format"):
        _lib.call("eoship_kv_bytes", C.byref(d), None, None)


def _bind(**kw):
    """eoship_kv_bind without a runtime: what it refuses before it needs one."""
    d = _lib.EosHipKVDesc(format=3, kv_heads=1, head_dim=32, page_tokens=16, pages=1, d_k=4096,
                          d_v=4096, d_k_scale=4096, d_v_scale=4096)
    cb, sg = kw.pop("codebook", gaussian_codebook()), kw.pop("signs", np.ones(32, np.float32))
    d.codebook = cb.ctypes.data if cb is not None else None
    d.signs = sg.ctypes.data if sg is not None else None
    for k, v in kw.items():
        setattr(d, k, v)
    out = C.c_void_p()
    _lib.call("eoship_kv_bind", None, C.byref(d), C.byref(out))


def test_bind_refusals():
    cb = gaussian_codebook()
    with pytest.raises(EosHipError, match="codebook and signs"):
        _bind(codebook=None)
    with pytest.raises(EosHipError, match="codebook and signs"):
        _bind(signs=None)
    with pytest.raises(EosHipError, match="ascending"):
        _bind(codebook=cb[::-1].copy())
    with pytest.raises(EosHipError, match="positive f16"):
        _bind(codebook=np.concatenate([[0.0], cb[1:]]).astype(np.float32))
    with pytest.raises(EosHipError, match="positive f16"):
        _bind(codebook=(cb * np.float32(1.0001)).astype(np.float32))
    with pytest.raises(EosHipError, match="signs must be 1 or -1"):
        _bind(signs=np.full(32, 0.5, np.float32))
    with pytest.raises(EosHipError, match="NULL pool"):
        _bind(d_k=None)
    with pytest.raises(EosHipError, match="aligned"):
        _bind(d_v=4100)
    with pytest.raises(EosHipError, match="scale pools"):
        _bind(d_v_scale=None)
    with pytest.raises(EosHipError, match="NULL argument"):
        _bind()


def test_calls_without_a_cache_are_refused():
    for name, args in (("eoship_kv_append_device", (None, None, None, None, 0, None, 0, 0)),
                       ("eoship_kv_read_device", (None, None, None, None, 0, None, 0, 0)),
                       ("eoship_kv_attention_device",
                        (None, None, None, None, 0, 1, 0, 1.0, 0, None, 0, None)),
                       ("eoship_kv_status", (None, None, None))):
        with pytest.raises(EosHipError, match="NULL argument"):
            _lib.call(name, *args)
    assert _lib.load().eoship_kv_release(None, None, None) == 0


CACHE = ("q8", 2, 64, 16, 10)


def test_check_batch_accepts_sound_batches():
    check_batch(*CACHE, [[1, 2, -1], [3, -1, -1]], [20, 16], writes=True)
    check_batch(*CACHE, [[1, 2, 0], [3, 4, 5]], [48, 48], [0, 40, 48], writes=True)
    # a shared prefix: read by both, written by neither
    check_batch(*CACHE, [[1, 2, -1], [1, 3, -1]], [20, 20], writes=True)
    check_batch(*CACHE, [[7, 7, 7]], [48])
    # nothing cached, padding rows, an empty batch
    check_batch(*CACHE, [[-1], [-1]], [0, 0], writes=True)
    check_batch(*CACHE, np.zeros((0, 1)), [])


@pytest.mark.parametrize("table,lens,off,rows,what", [
    ([[1, 10]], [32], None, None, "page 1 of its table row is 10"),
    ([[1, -1]], [17], None, None, "page 1 of its table row is -1"),
    ([[1, 2]], [33], None, None, "length 33"),
    ([[1, 2]], [-1], None, None, "length -1"),
    ([[1], [2]], [4, 4], [0, 3, 2], 3, "offsets must ascend"),
    ([[1], [2]], [4, 4], [0, 1, 4], 3, "offsets must ascend"),
    ([[1], [2]], [4, 4], [1, 2, 3], 3, r"offsets\[0\]"),
    ([[1], [2]], [4, 4], None, 3, "one row"),
    ([[1], [1]], [4, 4], None, None, "page 1 is written twice"),
    ([[4, 4]], [32], [0, 32], None, "page 4 is written twice"),
])
def test_check_batch_refusals(table, lens, off, rows, what):
    with pytest.raises(EosHipError, match=what):
        check_batch(*CACHE, table, lens, off, rows, writes=True)


def test_python_arguments():
    class Buf:
        ptr, nbytes = C.c_void_p(4096), 64
    with pytest.raises(ValueError, match="rows is needed"):
        KVBatch(Buf, 1, 4, Buf, Buf)
    with pytest.raises(ValueError, match="smaller"):
        KVBatch(Buf, 5, 4, Buf)
    with pytest.raises(ValueError, match="lengths must"):
        check_batch(*CACHE, [[1]], [1, 2])
