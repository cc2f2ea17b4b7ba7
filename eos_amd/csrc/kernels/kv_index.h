// Which rows, positions, pages and keys a workgroup of the key-value cache
// kernels has: integer arithmetic only, compiled into the kernels and, for
// tests, into host programs.
#ifndef EOSHIP_KV_INDEX_H
#define EOSHIP_KV_INDEX_H

#include "kv_args.h"

#ifdef __HIP_DEVICE_COMPILE__
#define KV_HD __device__ __forceinline__
#elif defined(__HIP__)
#define KV_HD __device__ __host__ inline
#else
#define KV_HD inline
#endif

KV_HD int kv_min(int a, int b) { return a < b ? a : b; }
KV_HD int kv_max(int a, int b) { return a > b ? a : b; }

// The rows of sequence b in a call: rows row0 .. row0 + n - 1 stand at
// positions len - n .. len - 1, of which the page table can hold the first
// `keys`. What is out of range counts as empty and is reported in `bad`.
struct KvSeq {
  int b = 0;
  long long row0 = 0;
  int n = 0, len = 0, keys = 0, bad = 0;
};

// From its row range [lo, hi) and length as they stand in memory.
KV_HD KvSeq kv_seq_of(const KvCacheArgs& c, int b, long long lo, long long hi, int len) {
  KvSeq s;
  s.b = b;
  if (lo < 0 || hi < lo || hi > c.rows) {
    s.bad |= kKvBadOffset;
    lo = hi = 0;
  }
  s.row0 = lo;
  s.n = (int)(hi - lo);
  s.len = len;
  const long long room = (long long)c.table_stride << c.page_shift;
  const long long cap = room < kKvMostKeys ? room : kKvMostKeys;
  if (s.len < 0 || s.len > cap) s.bad |= kKvBadLength;
  if (s.len < 0) s.len = 0;
  s.keys = s.len > cap ? (int)cap : s.len;
  return s;
}
KV_HD KvSeq kv_seq(const KvCacheArgs& c, int b) {
  return c.offsets != nullptr ? kv_seq_of(c, b, c.offsets[b], c.offsets[b + 1], c.lengths[b])
                              : kv_seq_of(c, b, b, (long long)b + 1, c.lengths[b]);
}

// Work units are numbered through a batch without knowing its row counts on
// the host: sequence b's first unit is floor(offset * mul / per) + extra * b,
// which leaves it floor(n * mul / per) + extra of them at least.
KV_HD long long kv_unit_base_of(long long offset, int b, int mul, int per, int extra) {
  return offset * mul / per + (long long)extra * b;
}
KV_HD long long kv_unit_base(const KvCacheArgs& c, int b, int mul, int per, int extra) {
  return kv_unit_base_of(c.offsets[b], b, mul, per, extra);
}
// Units of the whole batch.
KV_HD long long kv_units(long long rows, int batch, int mul, int per, int extra) {
  return rows * mul / per + (long long)extra * batch;
}

// The page of a token, or -1 where it has none in range.
KV_HD int kv_page(const KvCacheArgs& c, int b, int token) {
  const int i = token >> c.page_shift;
  if (token < 0 || i >= c.table_stride) return -1;
  const int p = c.table[(long long)b * c.table_stride + i];
  return p >= 0 && p < c.pages ? p : -1;
}

// Unit `within` of a sequence in append and read: `run` positions (whole
// groups) from pos0 on, of which [from, upto) are rows of the call. False
// where it has none.
struct KvRun {
  int pos0 = 0, from = 0, upto = 0;
  long long row = 0;  // the call's row of position pos0 (before `from`: not one)
};

KV_HD bool kv_run(const KvSeq& s, long long within, int run, KvRun& g) {
  const long long first = (long long)s.len - s.n;  // negative: padding rows before position 0
  const long long pos0 = ((first > 0 ? first : 0) / run + within) * run;
  if (s.n == 0 || within < 0 || pos0 >= s.keys) return false;
  g.pos0 = (int)pos0;
  g.from = first > pos0 ? (int)(first - pos0) : 0;
  g.upto = s.keys - pos0 < run ? (int)(s.keys - pos0) : run;
  g.row = s.row0 + (pos0 - first);
  return true;
}

// Where workgroup `block` works when consecutive ones go to the 8 XCDs in
// turn and each of `heads` heads has `items` pieces: heads are dealt to as
// many groups of XCDs as divide both, a group's XCDs take its heads' items in
// turn. The item may lie past the last one.
struct KvPlace {
  int head = 0;
  long long item = 0;
};
KV_HD int kv_xcd_groups(int heads) { return heads % 8 == 0 ? 8 : heads % 4 == 0 ? 4 : heads % 2 == 0 ? 2 : 1; }
KV_HD KvPlace kv_place(unsigned block, int heads, long long items) {
  const int groups = kv_xcd_groups(heads), share = 8 / groups;
  const unsigned xcd = block % 8, turn = block / 8;
  const unsigned per = (unsigned)((items + share - 1) / share);  // of a head, an XCD
  KvPlace p;
  p.head = (int)(xcd % groups + groups * (turn / per));
  p.item = (long long)(turn % per) * share + xcd / groups;
  return p;
}
// Workgroups of such a launch.
KV_HD long long kv_place_blocks(int heads, long long items) {
  const int share = 8 / kv_xcd_groups(heads);
  return heads * ((items + share - 1) / share * share);
}

// 16 query rows of a sequence and a head group (row r: row r / group of the
// sequence, head r % group), and the keys they attend.
struct KvTile {
  KvSeq s;
  int r0 = 0;
  int lo = 0, hi = 0;          // keys [lo, hi) that any row attends
  int all_lo = 0, all_hi = 0;  // keys [all_lo, all_hi) that every row attends
  int base = 0;                // lo, down to a whole 32
  int chunk = 0, splits = 0;   // keys of a split (whole 128s), splits with any
};

KV_HD int kv_row_pos(const KvSeq& s, int row) { return s.len - s.n + row; }

// Tile `within` of rows of sequence t.s; false where it has no rows.
KV_HD bool kv_tile(KvTile& t, long long within, int tile_rows, int group, int window, int splits) {
  if (within < 0 || within * tile_rows >= (long long)t.s.n * group) return false;
  t.r0 = (int)within * tile_rows;
  const int last = kv_min(t.r0 + tile_rows, t.s.n * group) - 1;
  const int p0 = kv_row_pos(t.s, t.r0 / group), p1 = kv_row_pos(t.s, last / group);
  t.hi = kv_min(t.s.keys, p1 + 1);
  t.lo = window > 0 ? kv_max(0, p0 - window + 1) : 0;
  if (t.hi <= t.lo) t.hi = t.lo = 0;
  t.all_hi = kv_min(t.s.keys, p0 + 1);
  t.all_lo = window > 0 ? p1 - window + 1 : 0;
  t.base = t.lo & ~31;
  const int steps = (t.hi - t.base + 127) / 128;
  const int per = kv_max((steps + splits - 1) / splits, 1);
  t.chunk = per * 128;
  t.splits = (steps + per - 1) / per;
  return true;
}

// The stream kernels' order of work, one row a sequence: head by head, in it
// sequence by sequence, in it 16-row tile by tile, in it 128-key step by step.
// Every workgroup takes `share` consecutive steps, so that long and short
// sequences keep all of them busy alike.
KV_HD int kv_steps(const KvCacheArgs& c, int b, int group, int window) {
  KvTile t;
  t.s = kv_seq(c, b);
  if (!kv_tile(t, 0, kKvTileRows, group, window, 1)) return 0;
  return (t.hi - t.base + 127) / 128;
}
// ... of all its tiles (64 bits: 2^23 steps of a thousand tiles pass 32).
KV_HD int kv_tiles_of(int group) { return (group + kKvTileRows - 1) / kKvTileRows; }
KV_HD long long kv_seq_steps(const KvCacheArgs& c, int b, int group, int window) {
  return (long long)kv_steps(c, b, group, window) * kv_tiles_of(group);
}
KV_HD long long kv_share(long long steps, int workgroups) {
  const long long q = (steps + workgroups - 1) / workgroups;
  return q < 2 ? 2 : q;
}
// The step at `pos` of a head whose sequence b has `steps` of them a tile from
// `first` on: the tile, and the steps [from, upto) of it that end at `end`.
struct KvSegment {
  int tile = 0, from = 0, upto = 0;
};
KV_HD KvSegment kv_segment(long long pos, long long end, long long first, int steps) {
  KvSegment g;
  const long long in = pos - first;
  g.tile = (int)(in / steps);
  g.from = (int)(in % steps);
  const long long left = end - pos;
  g.upto = left < steps - g.from ? g.from + (int)left : steps;
  return g;
}
// Where a workgroup that starts at step `start` leaves the part of a tile that
// begins at step `tile`: its first segment's place or its last one's.
KV_HD long long kv_part(long long workgroup, long long start, long long tile) {
  return (workgroup * 2 + (tile > start ? 1 : 0)) * kKvTileRows;
}

#endif
