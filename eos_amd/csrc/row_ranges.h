// Whether rows that lie a stride apart share a byte with others: outputs may
// stand between the rows of an input (columns of one array), not in them.
#ifndef EOSHIP_ROW_RANGES_H
#define EOSHIP_ROW_RANGES_H

#include <stdint.h>

namespace eoship {

struct Rows {
  uintptr_t at;
  int64_t count, stride, width;  // bytes; a row is no wider than the stride
  __int128 end() const { return (__int128)at + (__int128)(count - 1) * stride + width; }
};

inline Rows rows_of(const void* p, int64_t count, int64_t stride, int64_t width) {
  return Rows{(uintptr_t)p, count, stride, width};
}
inline Rows bytes_of(const void* p, int64_t bytes) { return Rows{(uintptr_t)p, 1, bytes, bytes}; }

// The first x >= 0 for which a x mod m lies in l..r, -1 if there is none
// (0 <= a < m, 0 < l <= r < m): a multiple of a in l..r itself, or, as in
// Euclid's division, the same question for m modulo a.
inline __int128 first_within(__int128 a, __int128 m, __int128 l, __int128 r) {
  if (a == 0) return -1;
  const __int128 x = (l + a - 1) / a;
  if (x * a <= r) return x;
  // a x - m y in l..r: m y mod a in -r..-l, which holds no multiple of a
  const __int128 y = first_within(m % a, a, (a - r % a) % a, (a - l % a) % a);
  return y < 0 ? -1 : (l + m * y + a - 1) / a;
}

inline bool rows_meet(const Rows& a, const Rows& b) {
  if (a.count < 1 || b.count < 1 || a.width < 1 || b.width < 1) return false;
  if (a.end() <= (__int128)b.at || b.end() <= (__int128)a.at) return false;
  if (a.stride == b.stride && a.count > 1 && b.count > 1) {
    // columns of one array: all rows stand alike
    const int64_t c = ((int64_t)(a.at - b.at) + a.width - 1) % a.stride;
    return (c < 0 ? c + a.stride : c) <= a.width + b.width - 2;
  }
  // a's rows from i0 to i1 reach into the bytes that b's first row to its last
  // span. There one shares a byte with a row of b if, counted from b's first, its
  // last byte stands less than both widths behind a multiple of b's stride.
  const int64_t s = a.stride, t = b.count > 1 ? b.stride : (int64_t)(b.end() - b.at);
  const __int128 from = (__int128)b.at - a.at - a.width, to = b.end() - a.at;
  const __int128 i0 = from < 0 ? 0 : from / s + 1;
  const __int128 i1 = (to - 1) / s < a.count - 1 ? (to - 1) / s : a.count - 1;
  if (i0 > i1) return false;
  const int64_t most = a.width + b.width - 2;
  if (most >= t - 1) return true;
  const int64_t c = (int64_t)((a.at + i0 * s - b.at + a.width - 1) % t);
  if (c <= most) return true;
  const __int128 x = first_within(s % t, t, t - c, t - c + most);
  return x >= 0 && x <= i1 - i0;
}

}  // namespace eoship

#endif
