// The key-value cache kernels' index arithmetic (kv_index.h) at its largest:
// sequences of 2^30 tokens and thousands of heads to a key-value head, whose
// steps pass 32 bits. Prints OK.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "kv_index.h"

#define CHECK(cond)                                              \
  do {                                                           \
    if (!(cond)) {                                               \
      std::printf("%s:%d: %s\n", __FILE__, __LINE__, #cond);     \
      std::exit(1);                                              \
    }                                                            \
  } while (0)

int main() {
  for (int group : {1, 16, 4096, 16368, 65535}) {
    KvCacheArgs c{};
    c.batch = 3;
    c.page_shift = 8;
    c.table_stride = 1 << 22;
    c.pages = 1;
    const int32_t lengths[] = {1 << 30, 5, (1 << 30) - 77};
    c.lengths = lengths;
    c.rows = 3;
    const int tiles = kv_tiles_of(group), heads = 1, workgroups = 512;
    CHECK((long long)tiles * 16 >= group && (tiles - 1) * 16 < group);
    std::vector<long long> pre(c.batch + 1, 0);
    for (int b = 0; b < c.batch; ++b) {
      const long long n = kv_seq_steps(c, b, group, 0);
      CHECK(n == (long long)((lengths[b] + 127LL) / 128) * tiles);
      pre[b + 1] = pre[b] + n;
    }
    const long long total = pre[c.batch], all = total * heads, share = kv_share(all, workgroups);
    long long covered = 0;
    for (int w = 0; w < workgroups; ++w) {
      const long long start = w * share, end = start + share < all ? start + share : all;
      for (long long pos = start; pos < end;) {
        int b = 0;
        for (int o = kKvStreamBatch; o > 0; o /= 2)
          if (b + o < c.batch && pre[b + o] <= pos) b += o;
        const int steps = (int)((pre[b + 1] - pre[b]) / tiles);
        CHECK(steps > 0 && pos >= pre[b] && pos < pre[b + 1]);
        const KvSegment g = kv_segment(pos, end, pre[b], steps);
        CHECK(g.tile >= 0 && g.tile < tiles && g.from >= 0 && g.from < g.upto && g.upto <= steps);
        KvTile t;
        t.s = kv_seq(c, b);
        CHECK(kv_tile(t, g.tile, kKvTileRows, group, 0, 1));
        CHECK(t.r0 >= 0 && t.r0 < group && t.hi == lengths[b]);
        CHECK((long long)t.base + 128LL * g.from < t.hi && (long long)t.base + 128LL * steps <= INT32_MAX);
        CHECK(kv_part(w, start, pos - g.from) < (long long)workgroups * 2 * kKvTileRows);
        covered += g.upto - g.from;
        pos += g.upto - g.from;
      }
    }
    CHECK(covered == all);
  }
  std::printf("OK\n");
  return 0;
}
