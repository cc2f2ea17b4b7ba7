// Rows that meet: random pairs of strided rows against every byte of them, and
// pairs of sizes that no loop could go through.
#include "row_ranges.h"

#include <cstdio>
#include <random>
#include <vector>

using eoship::Rows;
using eoship::rows_meet;

int main() {
  std::mt19937_64 g(1);
  const auto pick = [&](int lo, int hi) { return (int64_t)(lo + g() % (uint64_t)(hi - lo + 1)); };
  std::vector<char> mem(4096);
  int met = 0;
  for (int t = 0; t < 400000; ++t) {
    Rows r[2];
    for (Rows& x : r) {
      x.width = pick(0, 9) == 0 ? 0 : pick(1, 12);
      x.count = pick(0, 9) == 0 ? 0 : pick(1, 12);
      x.stride = x.width + (pick(0, 2) == 0 ? 0 : pick(0, 40));
      x.at = (uintptr_t)mem.data() + pick(0, 300);
    }
    if (pick(0, 3) == 0) r[1].stride = r[0].stride < r[1].width ? r[1].width : r[0].stride;
    std::fill(mem.begin(), mem.end(), 0);
    bool meet = false;
    for (int64_t i = 0; i < r[0].count; ++i)
      for (int64_t b = 0; b < r[0].width; ++b) mem[r[0].at - (uintptr_t)mem.data() + i * r[0].stride + b] = 1;
    for (int64_t i = 0; i < r[1].count; ++i)
      for (int64_t b = 0; b < r[1].width; ++b)
        meet |= mem[r[1].at - (uintptr_t)mem.data() + i * r[1].stride + b] != 0;
    if (rows_meet(r[0], r[1]) != meet || rows_meet(r[1], r[0]) != meet) {
      printf("case %d: %d\n", t, meet);
      return 1;
    }
    met += meet;
  }
  if (met < 50000 || met > 350000) return 2;
  // 2^31 rows: those of even places beside those of odd ones; strides that meet only
  // far out (row 3 * 2^29 of one and 2^30 of the other, a byte deep); 2^41 apart.
  const int64_t n = (int64_t)1 << 31, far = (int64_t)1 << 41;
  if (rows_meet({4096, n, 64, 32}, {4128, n, 64, 32}) || !rows_meet({4096, n, 64, 33}, {4128, n, 64, 32}))
    return 3;
  const uintptr_t b = 4096 + 3 * ((uintptr_t)1 << 29) * 1000 - ((uintptr_t)1 << 30) * 1500 + 7;
  if (!rows_meet({4096, n, 1000, 8}, {b, n, 1500, 8}) || rows_meet({4096, n, 1000, 7}, {b, n, 1500, 8}))
    return 4;
  if (rows_meet({4096, 1000, far, 16}, {4112, 1000, far, 16}) || !rows_meet({4096, 1000, far, 17}, {4112, 1000, far, 16}))
    return 5;
  // sizes that no memory has
  if (!rows_meet({4096, n, far * 2, 16}, {4096, n, far * 2 - 16, 16})) return 6;
  printf("OK\n");
  return 0;
}
