// Walks the work units of the key-value cache kernels on the host, with the
// kernels' own index arithmetic (kv_index.h), over random batches: every row
// is covered exactly once, every access stays inside pools, rows and
// workspace, with sound batches and with damaged ones. Prints OK.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "kv_index.h"

namespace {

std::mt19937_64 rng;
int between(int a, int b) { return a + (int)(rng() % (uint64_t)(b - a + 1)); }

#define CHECK(cond)                                                      \
  do {                                                                   \
    if (!(cond)) {                                                       \
      std::printf("%s:%d: %s (case %d)\n", __FILE__, __LINE__, #cond, at); \
      std::exit(1);                                                      \
    }                                                                    \
  } while (0)

// find_seq of the kernels: how many sequences start at or before unit u.
bool find(const KvCacheArgs& c, long long u, int mul, int per, int extra, KvSeq& s,
          long long& within) {
  int count = 0;
  for (int b = 0; b < c.batch; ++b) count += kv_unit_base(c, b, mul, per, extra) <= u;
  if (count == 0) return false;
  s = kv_seq(c, count - 1);
  within = u - kv_unit_base(c, count - 1, mul, per, extra);
  return true;
}

void one(int at, bool sound) {
  KvCacheArgs c{};
  c.batch = between(1, 9);
  c.page_shift = between(4, 8);
  c.table_stride = between(1, 6);
  c.pages = between(1, 40);
  c.kv_heads = 1;
  const int P = 1 << c.page_shift, cap = c.table_stride * P;
  const bool one_each = between(0, 3) == 0;
  std::vector<int32_t> table(c.batch * c.table_stride), lengths(c.batch), offsets(c.batch + 1);
  for (auto& p : table) p = between(0, c.pages - 1);
  for (int b = 0; b < c.batch; ++b) {
    lengths[b] = between(0, cap);
    offsets[b + 1] = offsets[b] + (one_each ? 1 : between(0, 2) == 0 ? between(0, 3) : between(0, cap + 5));
  }
  c.rows = offsets[c.batch] + (one_each ? 0 : between(0, 9));
  if (!sound) {
    const int many = between(1, 4);
    for (int i = 0; i < many; ++i) {
      const int32_t odd[] = {-1, INT32_MIN, INT32_MAX, between(-1000, 100000)};
      const int32_t v = odd[between(0, 3)];
      switch (between(0, 2)) {
        case 0: table[between(0, (int)table.size() - 1)] = v; break;
        case 1: lengths[between(0, c.batch - 1)] = v; break;
        default: offsets[between(0, c.batch)] = v;
      }
    }
  }
  c.table = table.data();
  c.lengths = lengths.data();
  c.offsets = one_each ? nullptr : offsets.data();

  // workgroups dealt to the XCDs: every item of every head once
  {
    const int heads = between(1, 20);
    const long long items = between(1, 40), blocks = kv_place_blocks(heads, items);
    std::vector<int> got(heads * items, 0);
    for (long long i = 0; i < blocks; ++i) {
      const KvPlace p = kv_place((unsigned)i, heads, items);
      CHECK(p.head >= 0 && p.head < heads && p.item >= 0);
      if (p.item < items) ++got[p.head * items + p.item];
    }
    for (int n : got) CHECK(n == 1);
  }

  // append / read
  const int run = one_each ? kKvGroup : kKvRun;
  std::vector<int> seen(c.rows, 0);
  const long long runs = one_each ? c.batch : kv_units(c.rows, c.batch, 1, run, 2);
  for (long long u = 0; u < runs; ++u) {
    KvSeq s;
    long long within = 0;
    if (one_each) s = kv_seq(c, (int)u);
    else if (!find(c, u, 1, run, 2, s, within)) continue;
    KvRun g;
    if (!kv_run(s, within, run, g)) continue;
    CHECK(g.pos0 % 8 == 0 && g.from >= 0 && g.upto <= run && g.from < g.upto);
    for (int r = g.from; r < g.upto; ++r) {
      CHECK(g.row + r >= 0 && g.row + r < c.rows);
      const int page = kv_page(c, s.b, g.pos0 + r / 8 * 8);
      CHECK(page < c.pages && page == kv_page(c, s.b, g.pos0 + r));
      ++seen[g.row + r];
      if (sound) CHECK(g.pos0 + r == s.len - s.n + (g.row + r - s.row0));
    }
  }
  if (sound)
    for (int b = 0; b < c.batch; ++b) {
      const int lo = one_each ? b : offsets[b], n = one_each ? 1 : offsets[b + 1] - lo;
      for (int i = 0; i < n; ++i) CHECK(seen[lo + i] == (lengths[b] - n + i >= 0 ? 1 : 0));
    }

  // the stream's shares: every step of every tile of every head once, and the
  // parts that a join looks for are those that were written
  if (one_each) {
    const int group = between(1, 40), window = between(0, 1) ? 0 : between(1, cap + 3);
    const int heads = between(1, 5), workgroups = between(1, 30);
    const int tiles = (group + kKvTileRows - 1) / kKvTileRows;
    std::vector<long long> pre(c.batch + 1, 0);
    for (int b = 0; b < c.batch; ++b) pre[b + 1] = pre[b] + (long long)kv_steps(c, b, group, window) * tiles;
    const long long total = pre[c.batch], all = total * heads, share = kv_share(all, workgroups);
    std::vector<int> done(all, 0);
    std::vector<long long> left(workgroups * 2 * kKvTileRows, -1);  // the tile whose part lies there
    for (int w = 0; w < workgroups; ++w) {
      const long long start = w * share, end = start + share < all ? start + share : all;
      for (long long pos = start; pos < end;) {
        const int h = (int)(pos / total);
        const long long rel = pos - h * total;
        int b = 0;
        for (int o = kKvStreamBatch; o > 0; o /= 2)
          if (b + o < c.batch && pre[b + o] <= rel) b += o;
        const int steps = (int)((pre[b + 1] - pre[b]) / tiles);
        CHECK(steps > 0 && rel >= pre[b] && rel < pre[b + 1]);
        const KvSegment g = kv_segment(rel, rel + (end - pos), pre[b], steps);
        KvTile t;
        t.s = kv_seq(c, b);
        CHECK(kv_tile(t, g.tile, kKvTileRows, group, window, 1));
        CHECK(g.from < g.upto && g.upto <= steps && t.base + 128 * g.from < t.hi);
        CHECK(t.base + 128 * steps >= t.hi);
        for (int i = g.from; i < g.upto; ++i) ++done[pos - g.from + i];
        if (!(g.from == 0 && g.upto == steps)) {
          const long long at_part = kv_part(w, start, pos - g.from);
          CHECK(at_part >= 0 && at_part + kKvTileRows <= (long long)left.size() && left[at_part] == -1);
          left[at_part] = pos - g.from;
        }
        pos += g.upto - g.from;
      }
    }
    CHECK(all <= share * workgroups);
    for (int n : done) CHECK(n == 1);
    for (int h = 0; h < heads; ++h)
      for (int b = 0; b < c.batch; ++b)
        for (int tile = 0; tile < tiles; ++tile) {
          const int steps = (int)((pre[b + 1] - pre[b]) / tiles);
          const long long first = h * total + pre[b] + (long long)tile * steps;
          const long long w0 = first / share, w1 = steps > 0 ? (first + steps - 1) / share : w0 - 1;
          if (w0 < w1)
            for (long long w = w0; w <= w1; ++w) {
              CHECK(w < workgroups && left[kv_part(w, w * share, first)] == first);
            }
        }
  }

  // attention
  for (int tile_rows : {16, 64, 128}) {
    const int group = between(1, 20), window = between(0, 1) ? 0 : between(1, cap + 3);
    const int splits = between(1, 7);
    const int per = (group + tile_rows - 1) / tile_rows;
    const long long tiles = one_each ? (long long)c.batch * per
                                     : kv_units(c.rows, c.batch, group, tile_rows, 1);
    std::vector<int> rows(c.rows * group, 0);
    for (long long u = 0; u < tiles; ++u) {
      KvTile t;
      long long within = u % per;
      if (one_each) t.s = kv_seq(c, (int)(u / per));
      else if (!find(c, u, group, tile_rows, 1, t.s, within)) continue;
      if (!kv_tile(t, within, tile_rows, group, window, splits)) continue;
      CHECK(t.splits <= splits && t.lo >= 0 && t.hi <= cap && t.base % 32 == 0);
      CHECK(t.base <= t.lo && (t.splits > 0 || t.hi == 0));
      CHECK((long long)t.base + (long long)t.splits * t.chunk >= t.hi);
      CHECK(t.splits == 0 || t.base + (t.splits - 1) * t.chunk < t.hi);
      for (int r = t.r0; r < t.r0 + tile_rows && r < t.s.n * group; ++r) {
        const long long row = t.s.row0 + r / group;
        CHECK(row >= 0 && row < c.rows);
        ++rows[row * group + r % group];
        if (!sound) continue;
        // The row's own keys lie in [lo, hi), and [all_lo, all_hi) in them.
        const int pos = kv_row_pos(t.s, r / group);
        const int hi = kv_min(pos + 1, t.s.keys), lo = window > 0 ? kv_max(0, pos - window + 1) : 0;
        if (hi > lo) CHECK(lo >= t.lo && hi <= t.hi);
        CHECK(t.all_hi <= kv_max(hi, 0) && t.all_lo >= (window > 0 ? pos - window + 1 : 0));
        // The unit that the join computes for this row.
        const long long unit = (one_each ? (long long)t.s.b * per
                                         : kv_unit_base(c, t.s.b, group, tile_rows, 1)) +
                               r / tile_rows;
        CHECK(unit == u && unit < tiles);
      }
    }
    if (sound) {
      const long long used = one_each ? c.batch : offsets[c.batch];
      for (long long i = 0; i < c.rows * group; ++i) CHECK(rows[i] == (i < used * group ? 1 : 0));
    }
  }
}

}  // namespace

int main(int argc, char** argv) {
  const int cases = argc > 1 ? std::atoi(argv[1]) : 2000;
  for (int i = 0; i < cases; ++i) {
    rng.seed(1000 + i);
    one(i, i % 2 == 0);
  }
  std::printf("OK\n");
  return 0;
}
