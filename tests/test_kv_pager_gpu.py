"""Page tables built on the GPU against plain loops: every array, every entry."""
import numpy as np
import pytest

import pager_reference as ref
from eos_amd._lib import EosHipError
from eos_amd.kvcache import KVPager, KVPlan
from eos_amd.runtime import DeviceBuffer, Runtime

pytestmark = pytest.mark.gpu


def _case(name):
    print(f"[case] {name}", flush=True)


class World:
    def __init__(self, rt, slots, stride, page, pages, rows, table=True, lists=True):
        self.rt, self.rows = rt, rows
        self.ref = ref.Pager(slots, stride, page, pages)
        self.dev = {n: DeviceBuffer.from_array(rt, np.full(max(k, 1), 77, np.int32))
                    for n, k in (("page_table", slots * stride), ("lengths", slots), ("free", pages),
                                 ("free_count", 1))}
        self.pager = KVPager(rt, slots, stride, page, pages, **self.dev)
        self.pager.reset()
        self.plan_np = dict(slots=np.full(slots, 77, np.int32), lengths=np.full(slots, 77, np.int32),
                            offsets=np.full(slots + 1, 77, np.int32),
                            table=np.full((slots, stride), 77, np.int32),
                            positions=np.full(rows, 77, np.int32), slot_map=np.full(rows, 77, np.int64))
        self.plan_dev = {n: DeviceBuffer.from_array(rt, np.concatenate([a.reshape(-1), a.reshape(-1)[:0]])
                                                    if a.size else np.zeros(2, a.dtype))
                         for n, a in self.plan_np.items()}
        d = self.plan_dev
        self.plan = KVPlan(d["slots"], d["table"] if table else None, d["lengths"], d["offsets"],
                           d["positions"] if lists else None, d["slot_map"] if lists else None, rows)
        self.skip = set() if table else {"table"}
        self.skip |= set() if lists else {"positions", "slot_map"}

    def put(self, lengths=None, table=None, free=None, count=None):
        """Both sides' state from outside."""
        for name, attr, a in (("lengths", "lengths", lengths), ("page_table", "table", table),
                              ("free", "free", free)):
            if a is not None:
                a = np.ascontiguousarray(a, np.int32)
                setattr(self.ref, attr, a.copy())
                self.dev[name].upload(a)
        if count is not None:
            self.ref.count = count
            self.dev["free_count"].upload(np.array([count], np.int32))

    def extend(self, new):
        new = np.asarray(new, np.int32)
        self.pager.extend(DeviceBuffer.from_array(self.rt, new), self.plan)
        got = self.ref.extend(new, self.plan_np, self.rows)
        assert self.pager.status() == got[2]
        self.check()
        return got

    def trim(self, keep):
        keep = np.asarray(keep, np.int32)
        self.pager.trim(DeviceBuffer.from_array(self.rt, keep))
        bad = self.ref.trim(keep)
        assert self.pager.status() == bad
        self.check()

    def check(self):
        r = self.ref
        for name, want in (("page_table", r.table), ("lengths", r.lengths), ("free", r.free),
                           ("free_count", np.array([r.count], np.int32))):
            np.testing.assert_array_equal(self.dev[name].download(np.int32, want.shape), want, name)
        for name, want in self.plan_np.items():
            if name not in self.skip and want.size:
                np.testing.assert_array_equal(self.plan_dev[name].download(want.dtype, want.shape), want, name)


@pytest.mark.parametrize("slots,stride,page,pages,rows", [
    (1, 1, 16, 1, 16), (1, 9, 16, 30, 100), (5, 4, 32, 12, 300), (33, 7, 16, 200, 900),
    (64, 128, 64, 5000, 3000), (257, 3, 256, 400, 5000), (1025, 6, 16, 3000, 9000),
    (4096, 5, 16, 9000, 30000)])
def test_steps_of_a_server(rt, slots, stride, page, pages, rows):
    """Random extends and trims, with requests that are refused for each reason."""
    _case(f"slots {slots} stride {stride} page {page} pages {pages}")
    rng = np.random.default_rng(slots)
    w = World(rt, slots, stride, page, pages, rows)
    w.check()
    room, seen = stride * page, 0
    for i in range(14):
        new = rng.integers(1, max(2, min(room, 2 * rows // slots)), slots)
        if i % 3 == 1:
            new = np.ones(slots, int)
        new = np.where(rng.random(slots) < (1.0, 0.5, 0.1)[i % 3], new, 0)
        if i % 4 == 3:  # within the plan's rows
            new = np.where(new.cumsum() <= rows, new, 0)
        new[rng.integers(0, slots)] = rng.choice([0, -3, room, 1])
        seen |= w.extend(new)[2]
        keep = np.where(rng.random(slots) < 0.5, rng.integers(-1, room, slots), -1)
        w.trim(np.where(rng.random(slots) < 0.2, 0, keep))
    assert slots < 5 or seen


def test_an_extend_undone_leaves_the_stack_as_it_was(rt):
    w = World(rt, 40, 20, 16, 500, 4000)
    rng = np.random.default_rng(4)
    w.extend(rng.integers(0, 90, 40))
    for _ in range(3):
        lens, free, count = w.ref.lengths.copy(), w.ref.free[:w.ref.count].copy(), w.ref.count
        w.extend(rng.integers(0, 40, 40))
        w.trim(lens)
        assert w.ref.count == count
        np.testing.assert_array_equal(w.ref.free[:count], free)


def test_empty_calls_and_one_long_request(rt):
    w = World(rt, 3, 5000, 16, 5100, 70000)
    assert w.extend([0, 0, 0])[0] == 0
    w.trim([-1, 0, 5])
    w.extend([0, 70000, 0])
    w.extend([1, 0, 0])
    w.trim([0, 3, 0])
    w.trim([0, 0, 0])


@pytest.mark.parametrize("table,lists", [(False, True), (True, False), (False, False)])
def test_parts_of_a_plan(rt, table, lists):
    w = World(rt, 50, 8, 32, 300, 2000, table, lists)
    rng = np.random.default_rng(1)
    for _ in range(4):
        w.extend(rng.integers(0, 40, 50))
    w.trim(rng.integers(-1, 100, 50))


def test_pages_run_out(rt):
    """From the first request that the stack does not cover on, those that need
    a page wait; those that need none go on."""
    w = World(rt, 6, 10, 16, 10, 200)
    w.extend([10, 10, 10, 0, 0, 0])           # a page each
    b, _, bad = w.extend([3, 100, 5, 40, 1, 0])  # slot 1 needs 6 of 7, slot 2 none, slot 3 three
    assert b == 5 and bad == 1
    assert list(w.ref.lengths) == [13, 110, 15, 0, 0, 0]
    assert w.ref.count == 1
    w.trim([0, -1, -1, -1, -1, -1])
    w.extend([0, 0, 0, 17, 1, 16])
    w.extend([0, 0, 0, 1, 0, 0])


def test_damaged_state_is_reported_and_touches_nothing_else(rt):
    w = World(rt, 5, 4, 16, 20, 100)
    w.extend([5, 20, 0, 7, 0])
    w.put(lengths=[-5, 20, 1000, 7, 0])
    assert w.extend([1, 1, 1, 1, 1])[2] == 4
    w.trim([0, 0, 0, -1, -1])
    w.put(lengths=[0, 0, 0, 8, 1])
    assert w.extend([2 ** 31 - 1, 2 ** 31 - 1, 1, 2 ** 31 - 1, 1])[2] & 4
    # a free count out of range counts as the nearest that is not
    for count, counts_as in ((-3, 0), (21, 20)):
        w.put(count=counts_as)
        w.dev["free_count"].upload(np.array([count], np.int32))
        w.pager.extend(DeviceBuffer.from_array(rt, np.zeros(5, np.int32)), w.plan)
        assert w.pager.status() == 4
        w.ref.extend(np.zeros(5, np.int32), w.plan_np, w.rows)
        w.check()


def test_own_arrays_two_runtimes_and_refusals(rt):
    pager = KVPager(rt, 4, 4, 16, 10)
    plan = pager.plan(64)
    new = DeviceBuffer.from_array(rt, np.array([3, 0, 20, 1], np.int32))
    pager.extend(new, plan)
    assert plan.lengths.download(np.int32, (3,)).tolist() == [3, 20, 1]
    assert plan.offsets.download(np.int32, (4,)).tolist() == [0, 3, 23, 24]
    assert pager.lengths.download(np.int32, (4,)).tolist() == [3, 0, 20, 1]
    b = plan.batch(4, 3, 24)
    assert b.batch == 3 and b.rows == 24
    with pytest.raises(ValueError, match="new is smaller"):
        pager.extend(new.view(0, 12), plan)
    with pytest.raises(ValueError, match="keep is smaller"):
        pager.trim(new.view(0, 12))
    with pytest.raises(EosHipError, match="aligned"):
        pager.extend(DeviceBuffer(rt, 64).view(2, 32), plan)
    plan.c.rows = -1
    with pytest.raises(EosHipError, match="rows"):
        pager.extend(new, plan)
    with Runtime(0) as other:
        mine = KVPager(other, 4, 4, 16, 10)
        mine.rt = rt
        with pytest.raises(EosHipError, match="another runtime"):
            mine.trim(new)
        mine.rt = other
        mine.release()
    pager.release()
    pager.release()
