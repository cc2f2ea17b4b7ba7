"""A pager's arrays kept by plain loops."""
import numpy as np

ROOM = 1 << 30


class Pager:
    def __init__(self, slots, stride, page, pages):
        self.slots, self.stride, self.p, self.pages = slots, stride, page, pages
        self.table = np.full((slots, stride), -1, np.int32)
        self.lengths = np.zeros(slots, np.int32)
        self.free = np.arange(pages - 1, -1, -1, dtype=np.int32)
        self.count = pages

    def _held(self, tokens):
        return -(-tokens // self.p)

    def extend(self, new, plan, rows):
        """Fills plan's arrays in place; returns (batch, rows, status)."""
        room = min(self.stride * self.p, ROOM)
        bad, j, row, asked, left = 0, 0, 0, 0, self.count
        top = self.count
        for s in range(self.slots):
            n, t = int(new[s]), int(self.lengths[s])
            if n < 0:
                bad |= 4
            if n <= 0:
                continue
            ok = True
            if t < 0 or t > room or row + n > rows:
                ok, bad = False, bad | 4
            elif t + n > room:
                ok, bad = False, bad | 2
            need = self._held(t + n) - self._held(t) if ok else 0
            asked += need
            if ok and need and asked > top:
                ok, bad = False, bad | 1
            lo, hi = min(row, rows), min(row + n, rows)
            plan["slots"][j], plan["offsets"][j] = s, lo
            plan["lengths"][j] = t + n if ok else 0
            if ok:
                for i in range(self._held(t), self._held(t + n)):
                    left -= 1
                    self.table[s, i] = self.free[left]
                end = self._held(t + n)
                plan["table"][j, :end] = self.table[s, :end]
                self.lengths[s] = t + n
                pos = np.arange(t, t + n)
                plan["positions"][lo:hi] = pos
                plan["slot_map"][lo:hi] = self.table[s, pos // self.p].astype(np.int64) * self.p + pos % self.p
            else:
                plan["positions"][lo:hi] = -1
                plan["slot_map"][lo:hi] = -1
            row += n
            j += 1
        plan["offsets"][j] = min(row, rows)
        self.count = left
        return j, row, bad

    def trim(self, keep):
        bad, out = 0, []
        room = min(self.stride * self.p, ROOM)
        for s in range(self.slots):
            t, k = int(self.lengths[s]), int(keep[s])
            if t < 0 or t > room:
                bad |= 4
                continue
            if k < 0 or k >= t:
                continue
            a, b = self._held(k), self._held(t)
            out += list(self.table[s, a:b])
            self.table[s, a:b] = -1
            self.lengths[s] = k
        for page in out[::-1]:
            self.free[self.count] = page
            self.count += 1
        return bad
