"""Page tables on the host: refusals, and the plain pager's own invariants."""
import ctypes as C

import numpy as np
import pytest

import pager_reference as ref
from eos_amd import _lib
from eos_amd._lib import EosHipError
from eos_amd.kvcache import KVPager, KVPlan


@pytest.mark.parametrize("kw,what", [
    (dict(slots=0), "slots"), (dict(slots=4097), "slots"), (dict(table_stride=0), "table_stride"),
    (dict(table_stride=2 ** 26 + 1), "table_stride"), (dict(page_tokens=8), "page_tokens"),
    (dict(page_tokens=48), "page_tokens"), (dict(page_tokens=512), "page_tokens"),
    (dict(pages=0), "pages"), (dict(pages=2 ** 31), "pages"), (dict(d_page_table=None), "NULL page"),
    (dict(d_free_count=None), "NULL page"), (dict(d_lengths=4098), "4-byte"), (dict(), "NULL argument")])
def test_bind_refused(kw, what):
    a = dict(slots=4, table_stride=8, page_tokens=16, pages=9, d_page_table=4096, d_lengths=4096,
             d_free=4096, d_free_count=4096) | kw
    out = C.c_void_p(1)
    with pytest.raises(EosHipError, match=what):
        _lib.call("eoship_kv_pager_bind", None, C.byref(_lib.EosHipKVPagerDesc(**a)), C.byref(out))
    assert not out


def test_null_refused():
    for name, args in (("reset_device", ()), ("extend_device", (4096, C.byref(_lib.EosHipKVPlan()))),
                       ("trim_device", (4096,)), ("status", (C.byref(C.c_int32()),))):
        with pytest.raises(EosHipError, match="NULL"):
            _lib.call("eoship_kv_pager_" + name, None, None, *args)
    _lib.call("eoship_kv_pager_release", None, None)


class _Buf:
    def __init__(self, nbytes):
        self.nbytes, self.ptr = nbytes, C.c_void_p(4096)


def test_wrapper_checks_sizes():
    with pytest.raises(ValueError, match="together"):
        KVPager(None, 4, 8, 16, 9, lengths=_Buf(16))
    with pytest.raises(ValueError, match="smaller"):
        KVPager(None, 4, 8, 16, 9, _Buf(127), _Buf(16), _Buf(36), _Buf(4))
    with pytest.raises(ValueError, match="row array"):
        KVPlan(_Buf(16), None, _Buf(16), _Buf(20), _Buf(12), None, 4)
    with pytest.raises(ValueError, match="plan's array"):
        KVPlan(_Buf(16), None, _Buf(16), _Buf(16))._check(4, 8)


def test_plain_pager_keeps_every_page_once():
    rng = np.random.default_rng(0)
    p = ref.Pager(7, 6, 16, 25)
    for _ in range(300):
        new = np.where(rng.random(7) < 0.5, rng.integers(0, 60, 7), 0)
        rows = int(new.sum())
        plan = dict(slots=np.zeros(7, np.int32), lengths=np.zeros(7, np.int32),
                    offsets=np.zeros(8, np.int32), table=np.full((7, 6), -1, np.int32),
                    positions=np.zeros(rows, np.int32), slot_map=np.zeros(rows, np.int64))
        before = (p.table.copy(), p.lengths.copy(), p.free[:p.count].copy())
        p.extend(new, plan, rows)
        live = plan["slot_map"][plan["slot_map"] >= 0]
        assert len(np.unique(live)) == len(live)
        held = p.table[p.table >= 0]
        assert sorted(np.concatenate([held, p.free[:p.count]])) == list(range(25))
        if rng.random() < 0.5:  # undone: as it was, the stack's order included
            p.trim(before[1])
            np.testing.assert_array_equal(p.table, before[0])
            np.testing.assert_array_equal(p.free[:p.count], before[2])
        p.trim(np.where(rng.random(7) < 0.3, rng.integers(0, 90, 7), -1))
        held = p.table[p.table >= 0]
        assert sorted(np.concatenate([held, p.free[:p.count]])) == list(range(25))
