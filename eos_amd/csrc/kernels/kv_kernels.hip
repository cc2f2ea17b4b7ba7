// Paged key-value cache on gfx950: rows written in a storage format, read
// back, and attended.
//
// Pools, for pages of P tokens, H key-value heads of width D:
//   K       [pages][H][P][D]        f16 / bf16 / int8 codes
//           [pages][H][P][D / 8]    tq4: words, dimension 8 w + j at bits 4 j
//   V       [pages][H][P / 8][D][8]  f16 / bf16 / int8 codes
//           [pages][H][P / 8][D]    tq4: words, token 8 g + j at bits 4 j
//   scales  [pages][H][P] f32 for K and for V (q8, tq4)
// V keeps 8 tokens of a dimension side by side because the product with the
// probabilities sums over tokens: an MFMA operand register holds consecutive
// summands of one output, so a lane's load is its operand as it lies.
//
// q8:  s = max|x| / 127, code = rint(x * (127 / max|x|)), stands for code * s.
// tq4: w = Hd (signs * x) (Walsh-Hadamard, unnormalised), s = sqrt(sum x^2 / D),
//      index = number of edges below |w| / (s sqrt(D)), code = 8 [w < 0] + index,
//      stands for signs * Hd (+-magnitude) * s / sqrt(D). Attention stays in
//      the rotated space: q is rotated once, the output once.
// A scale below 2^-60 is stored as zero, one above 2^40 or not finite as NaN.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv_index.h"

#define EOS_DEV __device__ __forceinline__
#define KV_INLINE __attribute__((always_inline))

namespace {

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v2b __attribute__((ext_vector_type(2)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

constexpr float kTiny = 0x1p-60f, kHuge = 0x1p40f;
constexpr float kLowest = -0x1.fffffep127f;  // softmax reference before any key: below every score

constexpr int bits_of(int fmt) { return fmt == kKvQ8 ? 8 : fmt == kKvTq4 ? 4 : 16; }
constexpr int log2i(int x) { return x <= 1 ? 0 : 1 + log2i(x / 2); }

EOS_DEV uint32_t perm(uint32_t hi, uint32_t lo, uint32_t sel) {
  return __builtin_amdgcn_perm(hi, lo, sel);
}

EOS_DEV float bf16_to_f32(uint32_t u) { return __builtin_bit_cast(float, u << 16); }
// Nearest, ties to even; NaN stays NaN.
EOS_DEV uint32_t f32_to_bf16(float f) {
  return __builtin_bit_cast(uint16_t, (__bf16)f);
}
EOS_DEV uint32_t f32_to_f16(float f) { return __builtin_bit_cast(uint16_t, (_Float16)f); }
EOS_DEV float f16_to_f32(uint32_t u) {
  return (float)__builtin_bit_cast(_Float16, (uint16_t)u);
}

// 8 consecutive elements of a caller's row, and back.
EOS_DEV void unpack8(v4u u, int dtype, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t a = u[i] & 0xffffu, b = u[i] >> 16;
    x[2 * i] = dtype == kKvRowF16 ? f16_to_f32(a) : bf16_to_f32(a);
    x[2 * i + 1] = dtype == kKvRowF16 ? f16_to_f32(b) : bf16_to_f32(b);
  }
}
EOS_DEV void load8(const uint8_t* p, int dtype, float (&x)[8]) {
  unpack8(*reinterpret_cast<const v4u*>(p), dtype, x);
}
EOS_DEV void store8(uint8_t* p, int dtype, const float (&x)[8]) {
  if (dtype == kKvRowF32) {
    reinterpret_cast<v4f*>(p)[0] = v4f{x[0], x[1], x[2], x[3]};
    reinterpret_cast<v4f*>(p)[1] = v4f{x[4], x[5], x[6], x[7]};
    return;
  }
  v4u u;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    u[i] = dtype == kKvRowF16 ? f32_to_f16(x[2 * i]) | f32_to_f16(x[2 * i + 1]) << 16
                              : f32_to_bf16(x[2 * i]) | f32_to_bf16(x[2 * i + 1]) << 16;
  *reinterpret_cast<v4u*>(p) = u;
}

// The value of lane ^ S, by the vector unit's own lane moves where it has them
// (a shuffle goes through LDS).
template <int CTRL>
EOS_DEV uint32_t dpp(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true);
}
template <int S>
EOS_DEV uint32_t lane_xor(uint32_t x) {
  if constexpr (S == 1) return dpp<0xb1>(x);                // quad_perm 1 0 3 2
  else if constexpr (S == 2) return dpp<0x4e>(x);           // quad_perm 2 3 0 1
  else if constexpr (S == 4) return dpp<0x1b>(dpp<0x141>(x));  // half mirror, quad reversed
  else if constexpr (S == 8) return dpp<0x128>(x);          // row rotated by 8
  else return (uint32_t)__shfl_xor((int)x, S);
}
template <int S>
EOS_DEV float lane_xor(float x) {
  return __builtin_bit_cast(float, lane_xor<S>(__builtin_bit_cast(uint32_t, x)));
}
template <int S>
EOS_DEV double lane_xor(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  return __builtin_bit_cast(double, (uint64_t)lane_xor<S>((uint32_t)(u >> 32)) << 32 |
                                        lane_xor<S>((uint32_t)u));
}
template <int LANES, int S = 1>
EOS_DEV double row_sum(double x) {
  if constexpr (S < LANES) return row_sum<LANES, 2 * S>(x + lane_xor<S>(x));
  else return x;
}
template <int LANES, int S = 1>
EOS_DEV float row_max(float x) {
  if constexpr (S < LANES) return row_max<LANES, 2 * S>(fmaxf(x, lane_xor<S>(x)));
  else return x;
}
template <int LANES, int S = 1>
EOS_DEV uint32_t row_or(uint32_t x) {
  if constexpr (S < LANES) return row_or<LANES, 2 * S>(x | lane_xor<S>(x));
  else return x;
}

// Walsh-Hadamard transform of a row spread over LANES neighbouring lanes, 8
// consecutive elements each.
template <int LANES, int S = 1>
EOS_DEV void hadamard_lanes(float (&x)[8]) {
  if constexpr (S < LANES) {
    const uint32_t flip = (threadIdx.x & S) != 0 ? 0x80000000u : 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float o = lane_xor<S>(x[i]);
      x[i] = o + __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x[i]) ^ flip);
    }
    hadamard_lanes<LANES, 2 * S>(x);
  }
}
template <int LANES>
EOS_DEV void hadamard8(float (&x)[8]) {
#pragma unroll
  for (int s = 1; s < 8; s *= 2)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if ((i & s) == 0) {
        const float a = x[i], b = x[i + s];
        x[i] = a + b;
        x[i + s] = a - b;
      }
  hadamard_lanes<LANES>(x);
}

// ------------------------------------------------------------- sequences

EOS_DEV void flag(const KvCacheArgs& c, int bits) {
  if (bits != 0 && threadIdx.x == 0) atomicOr(c.status, bits);
}

// The sequence that unit u belongs to and u's index within it; false where
// no sequence has it. All threads of the workgroup call it; each looks at one
// sequence of 256 (of 64, 128, 512), so that its numbers come with one load's
// latency.
EOS_DEV bool find_seq(const KvCacheArgs& c, long long u, int mul, int per, int extra, KvSeq& s,
                      long long& within) {
  __shared__ int found[4];
  int count = 0;
  for (int b0 = 0; b0 < c.batch; b0 += blockDim.x) {
    const int b = b0 + threadIdx.x;
    const bool in = b < c.batch;
    const int lo = in ? c.offsets[b] : 0, hi = in ? c.offsets[b + 1] : 0, len = in ? c.lengths[b] : 0;
    const int n = __syncthreads_count(in && kv_unit_base_of(lo, b, mul, per, extra) <= u);
    if ((int)threadIdx.x == n - 1) {
      found[0] = b;
      found[1] = lo;
      found[2] = hi;
      found[3] = len;
    }
    count += n;
  }
  if (count == 0) return false;
  __syncthreads();
  s = kv_seq_of(c, found[0], found[1], found[2], found[3]);
  flag(c, s.bad);
  within = u - kv_unit_base_of(found[1], s.b, mul, per, extra);
  return true;
}

// --------------------------------------------------------- append and read

template <int FMT>
EOS_DEV v4f mfma16(v4u a, v4u b, v4f c) {
  if constexpr (FMT == kKvBf16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, a),
                                                   __builtin_bit_cast(v8b, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a),
                                                  __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

// The rotation of tq4 on the matrix cores. A wavefront has 16 rows; lane (row r
// = lane % 16, part g = lane / 16) holds elements 32 s + 8 g + j of its row as
// 16-bit operands x[s][j] and receives elements 32 (t / 2) + 8 g + 4 (t % 2) + i
// of the transform as y[t][i]. The other operand is the Walsh-Hadamard matrix,
// whose entries are signs: the parity of i & j % 4, t % 2 & j / 4, g' & g and
// t / 2 & s for output (t, g', i) and input (s, g, j). So there are two fragments,
// for even and odd t, and the rest is a sign of x. Products by +-1 are exact,
// sums f32. (32,768 tokens x 8 heads x 128 appended, the same ones again: 88 us,
// by butterflies between lanes 106; 24,576 read, other pages each time: 56 and 62.)
// One row a sequence stays with the butterflies: 16 rows of 8 heads of 128 take
// 5.3 us, on the matrix cores 6.8, of 256 5.2 and 11.8. Either adds in f32, in an
// order of its own: a value next to a threshold may take another code.
template <int FMT, int D>
EOS_DEV void rotate16(const v4u (&x)[D / 32], v4f (&y)[D / 16]) {
  constexpr uint32_t kOne = FMT == kKvBf16 ? 0x3f80u : 0x3c00u;
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  v4u f[2];
#pragma unroll
  for (int odd = 0; odd < 2; ++odd)
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      uint32_t u = kOne | kOne << 16;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int j = 2 * w + b;
        const int par = __builtin_popcount(r & 3 & j & 3) ^ __builtin_popcount((r >> 2) & g) ^ (odd & j >> 2);
        u |= (uint32_t)(par & 1) << (15 + 16 * b);
      }
      f[odd][w] = u;
    }
#pragma unroll
  for (int t = 0; t < D / 16; ++t) {
    y[t] = v4f{0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < D / 32; ++s) {
      const uint32_t flip = (__builtin_popcount((t >> 1) & s) & 1) != 0 ? 0x80008000u : 0u;
      y[t] = mfma16<FMT>(f[t & 1], x[s] ^ v4u{flip, flip, flip, flip}, y[t]);
    }
  }
}

// Codes (a byte each) -> f16 magnitudes with their signs, four of them.
EOS_DEV void bytes_to_f16(const KvTables& t, uint32_t k, uint32_t& p0, uint32_t& p1) {
  const uint32_t idx = k & 0x07070707u;
  const uint32_t fh = perm(t.hi[1], t.hi[0], idx) | (k << 4 & 0x80808080u);
  const uint32_t fl = perm(t.lo[1], t.lo[0], idx);
  p0 = perm(fh, fl, 0x05010400u);
  p1 = perm(fh, fl, 0x07030602u);
}

// The 4-bit code of a rotated value: the edges ascend, so three comparisons
// place it among the seven.
EOS_DEV uint32_t code_of(float x, const float (&e)[7]) {
  const float w = fabsf(x);
  const bool b2 = w > e[3];
  const bool b1 = w > (b2 ? e[5] : e[1]);
  const bool b0 = w > (b2 ? (b1 ? e[6] : e[4]) : (b1 ? e[2] : e[0]));
  return (x < 0.0f ? 8u : 0u) | (b2 ? 4u : 0u) | (b1 ? 2u : 0u) | (b0 ? 1u : 0u);
}

// The positions of a workgroup of append or read and their sequence.
template <int RUN>
EOS_DEV bool find_run(const KvCacheArgs& c, KvRun& g, int& b) {
  KvSeq s;
  long long within = 0;
  if (RUN == kKvGroup) {
    s = kv_seq(c, blockIdx.x);
    flag(c, s.bad);
  } else if (!find_seq(c, blockIdx.x, 1, RUN, 2, s, within)) {
    return false;
  }
  b = __builtin_amdgcn_readfirstlane(s.b);
  if (!kv_run(s, within, RUN, g)) return false;
  g.pos0 = __builtin_amdgcn_readfirstlane(g.pos0);
  return true;
}

// Tokens of the pools in front of the run's groups, or -1 where the group has
// no row of the call or no page. The page ids are loaded together.
template <int NG>
EOS_DEV void find_blocks(const KvCacheArgs& c, const KvRun& g, int b, int h, long long (&at)[NG]) {
  const int32_t* row = c.table + (size_t)b * c.table_stride;
  int page[NG];
#pragma unroll
  for (int j = 0; j < NG; ++j)
    page[j] = row[kv_min((g.pos0 + 8 * j) >> c.page_shift, c.table_stride - 1)];
  bool bad = false;
#pragma unroll
  for (int j = 0; j < NG; ++j) {
    const bool need = 8 * j < g.upto && 8 * j + 8 > g.from;
    const bool in = (unsigned)page[j] < (unsigned)c.pages;
    bad |= need && !in;
    at[j] = need && in ? ((((long long)page[j] * c.kv_heads + h) << c.page_shift) +
                          ((g.pos0 + 8 * j) & ((1 << c.page_shift) - 1)))
                       : -1;
  }
  if (bad) flag(c, kKvBadPage);
}

// One workgroup of 2 D threads: RUN positions of one head, in groups of 8 (the
// tokens that V stores side by side); the first half of the threads has K, the
// second V, D / 8 lanes a row of 8 elements. A group's words are one
// workgroup's, so a partly filled 4-bit word is read and merged without
// another writer. Bound by the rows' bytes and the latency of three dependent
// loads (numbers, page ids, rows), which runs of 32 positions share among four
// groups: 8 x 1,021 ragged rows of 12 heads of 64 in q8 appended and read back,
// 20 us, by single groups 23. 32,768 rows of 8 heads of 128 appended and read: f16
// 65 and 59 us, 4.1 and 4.5 TB/s, q8 69 and 59.
template <int FMT, int D, int RUN>
EOS_DEV void append_run(const KvRowsArgs& a) {
  constexpr int LANES = D / 8, NG = RUN / 8;
  constexpr bool kPlain = FMT == kKvF16 || FMT == kKvBf16;
  __shared__ __align__(16) uint16_t vt[FMT == kKvTq4 ? 8 : NG * D * 8];
  static_assert(__alignof__(vt) >= 16, "read by 16 bytes");
  __shared__ uint32_t vw[FMT == kKvTq4 ? NG * 8 * LANES : 1];
  const KvCacheArgs& c = a.c;
  const int tid = threadIdx.x, h = blockIdx.y;
  KvRun g;
  int b;
  if (!find_run<RUN>(c, g, b)) return;
  long long at[NG];
  find_blocks<NG>(c, g, b, h, at);
  const bool is_v = tid >= D;
  const int r = (tid / LANES) & 7, l8 = tid % LANES;
  const uint8_t* src = (is_v ? a.v : a.k) + ((size_t)h * D + l8 * 8) * 2;
  const size_t stride = (size_t)(is_v ? a.v_stride : a.k_stride) * 2;
  v4u raw[NG];
  bool live[NG];
#pragma unroll
  for (int j = 0; j < NG; ++j) {
    const int p = 8 * j + r;
    live[j] = at[j] >= 0 && p >= g.from && p < g.upto;
    raw[j] = v4u{0, 0, 0, 0};
    if (live[j]) raw[j] = *reinterpret_cast<const v4u*>(src + (size_t)(g.row + p) * stride);
  }
  float sgn[8];
  if constexpr (FMT == kKvTq4) {
    const v4f s0 = reinterpret_cast<const v4f*>(c.t.signs + l8 * 8)[0];
    const v4f s1 = reinterpret_cast<const v4f*>(c.t.signs + l8 * 8)[1];
#pragma unroll
    for (int i = 0; i < 8; ++i) sgn[i] = i < 4 ? s0[i & 3] : s1[i & 3];
  }
#pragma unroll
  for (int j = 0; j < NG; ++j) {
    if (at[j] < 0) continue;
    if constexpr (kPlain) {
      if (!is_v) {
        if (live[j]) *reinterpret_cast<v4u*>(c.k + ((size_t)(at[j] + r) * D + l8 * 8) * 2) = raw[j];
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          vt[(j * D + l8 * 8 + 2 * i) * 8 + r] = (uint16_t)raw[j][i];
          vt[(j * D + l8 * 8 + 2 * i + 1) * 8 + r] = (uint16_t)(raw[j][i] >> 16);
        }
      }
      continue;
    }
    float x[8];
    unpack8(raw[j], a.dtype, x);
    if constexpr (FMT == kKvQ8) {
      float m = 0.0f;
      uint32_t bad = 0;  // NaN or infinity
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        m = fmaxf(m, fabsf(x[i]));
        bad |= !(fabsf(x[i]) <= 3.4028234e38f);
      }
      m = row_max<LANES>(m);
      bad = row_or<LANES>(bad);
      float scale = __fdiv_rn(m, 127.0f);
      const bool none = scale < kTiny;
      const bool nan = bad != 0 || scale > kHuge;
      const float inv = none || nan ? 0.0f : __fdiv_rn(127.0f, m);
      scale = nan ? __builtin_nanf("") : none ? 0.0f : scale;
      uint32_t code[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float q = nan ? 0.0f : fminf(fmaxf(rintf(x[i] * inv), -127.0f), 127.0f);
        code[i] = (uint32_t)(int)q & 0xffu;
      }
      if (live[j] && l8 == 0) (is_v ? c.v_scale : c.k_scale)[at[j] + r] = scale;
      if (!is_v) {
        if (live[j])
          *reinterpret_cast<v2u*>(c.k + (size_t)(at[j] + r) * D + l8 * 8) =
              v2u{code[0] | code[1] << 8 | code[2] << 16 | code[3] << 24,
                  code[4] | code[5] << 8 | code[6] << 16 | code[7] << 24};
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) vt[(j * D + l8 * 8 + i) * 8 + r] = (uint16_t)code[i];
      }
    }
    if constexpr (FMT == kKvTq4) {
      double ss = 0.0;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += (double)x[i] * (double)x[i];
      ss = row_sum<LANES>(ss);
      float scale = (float)__builtin_sqrt(ss * (1.0 / D));
      const bool none = scale < kTiny;
      const bool nan = !(scale <= kHuge);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = none || nan ? 0.0f : x[i] * sgn[i];
      hadamard8<LANES>(x);
      // |w| / (s sqrt(D)) against the edges, the division moved to their side.
      const float norm = none || nan ? 0.0f : scale * (float)__builtin_sqrt((double)D);
      scale = nan ? __builtin_nanf("") : none ? 0.0f : scale;
      float e[7];
#pragma unroll
      for (int i = 0; i < 7; ++i) e[i] = c.t.edges[i] * norm;
      uint32_t word = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) word |= code_of(x[i], e) << (4 * i);
      if (live[j] && l8 == 0) (is_v ? c.v_scale : c.k_scale)[at[j] + r] = scale;
      if (!is_v) {
        if (live[j]) reinterpret_cast<uint32_t*>(c.k)[(size_t)(at[j] + r) * LANES + l8] = word;
      } else {
        vw[(j * 8 + r) * LANES + l8] = word;
      }
    }
  }
  __syncthreads();
  // V: a group's 8 tokens of one dimension by one thread.
#pragma unroll
  for (int it = 0; it < (NG + 1) / 2; ++it) {
    const int j = 2 * it + (NG > 1 ? tid / D : 0), dim = tid % D;
    if (NG == 1 && tid >= D) break;
    long long base = at[2 * it];
    if (NG > 1 && j != 2 * it) base = at[(2 * it + 1) % NG];
    if (base < 0) continue;
    const int from = g.from > 8 * j ? g.from - 8 * j : 0;
    const int upto = g.upto - 8 * j < 8 ? g.upto - 8 * j : 8;
    const bool whole = from == 0 && upto == 8;
    const size_t vrow = (size_t)(base / kKvGroup) * D + dim;  // group-dimensions before
    if constexpr (kPlain) {
      uint16_t* dst = reinterpret_cast<uint16_t*>(c.v) + vrow * 8;
      if (whole) {
        *reinterpret_cast<v4u*>(dst) = *reinterpret_cast<const v4u*>(&vt[(j * D + dim) * 8]);
      } else {
        for (int t = from; t < upto; ++t) dst[t] = vt[(j * D + dim) * 8 + t];
      }
    } else if constexpr (FMT == kKvQ8) {
      uint8_t* dst = c.v + vrow * 8;
      if (whole) {
        const v4u u = *reinterpret_cast<const v4u*>(&vt[(j * D + dim) * 8]);
        *reinterpret_cast<v2u*>(dst) = v2u{perm(u[1], u[0], 0x06040200), perm(u[3], u[2], 0x06040200)};
      } else {
        for (int t = from; t < upto; ++t) dst[t] = (uint8_t)vt[(j * D + dim) * 8 + t];
      }
    } else {
      uint32_t* dst = reinterpret_cast<uint32_t*>(c.v) + vrow;
      uint32_t word = 0, mask = 0;
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const bool in = t >= from && t < upto;
        word |= in ? (vw[(j * 8 + t) * LANES + dim / 8] >> (4 * (dim & 7)) & 15u) << (4 * t) : 0u;
        mask |= in ? 15u << (4 * t) : 0u;
      }
      *dst = whole ? word : (*dst & ~mask) | word;
    }
  }
}

// The values of RUN positions of one head, same shape of workgroup; V passes
// through LDS from its groups of 8 tokens into rows.
template <int FMT, int D, int RUN>
EOS_DEV void read_run(const KvRowsArgs& a) {
  constexpr int LANES = D / 8, NG = RUN / 8;
  constexpr bool kPlain = FMT == kKvF16 || FMT == kKvBf16;
  constexpr int kType = FMT == kKvF16 ? kKvRowF16 : kKvRowBf16;
  __shared__ __align__(16) uint16_t vh[kPlain ? NG * 8 * D : 8];
  __shared__ __align__(16) uint8_t vb[kPlain ? 16 : NG * 8 * D];
  static_assert(__alignof__(vh) >= 16 && __alignof__(vb) >= 8, "read by 16 and 8 bytes");
  const KvCacheArgs& c = a.c;
  const int tid = threadIdx.x, h = blockIdx.y;
  KvRun g;
  int b;
  if (!find_run<RUN>(c, g, b)) return;
  long long at[NG];
  find_blocks<NG>(c, g, b, h, at);
  const bool is_v = tid >= D;
  const int r = (tid / LANES) & 7, l8 = tid % LANES;
  // V's groups, one dimension a thread.
#pragma unroll
  for (int it = 0; it < (NG + 1) / 2; ++it) {
    const int j = 2 * it + (NG > 1 ? tid / D : 0), dim = tid % D;
    if (NG == 1 && tid >= D) break;
    long long base = at[2 * it];
    if (NG > 1 && j != 2 * it) base = at[(2 * it + 1) % NG];
    if (base < 0) continue;
    const size_t vrow = (size_t)(base / kKvGroup) * D + dim;
    if constexpr (kPlain) {
      const v4u u = *reinterpret_cast<const v4u*>(c.v + vrow * 16);
#pragma unroll
      for (int t = 0; t < 8; ++t) vh[(j * 8 + t) * D + dim] = (uint16_t)(u[t / 2] >> (16 * (t & 1)));
    } else if constexpr (FMT == kKvQ8) {
      const v2u u = *reinterpret_cast<const v2u*>(c.v + vrow * 8);
#pragma unroll
      for (int t = 0; t < 8; ++t) vb[(j * 8 + t) * D + dim] = (uint8_t)(u[t / 4] >> (8 * (t & 3)));
    } else {
      const uint32_t u = reinterpret_cast<const uint32_t*>(c.v)[vrow];
#pragma unroll
      for (int t = 0; t < 8; ++t) vb[(j * 8 + t) * D + dim] = (uint8_t)(u >> (4 * t) & 15u);
    }
  }
  // K rows and scales; the values a thread has no row for are not stored.
  v4u raw[NG];
  float scale[NG];
  bool live[NG];
#pragma unroll
  for (int j = 0; j < NG; ++j) {
    const int p = 8 * j + r;
    live[j] = at[j] >= 0 && p >= g.from && p < g.upto;
    raw[j] = v4u{0, 0, 0, 0};
    scale[j] = 0.0f;
    if (!live[j]) continue;
    const size_t token = (size_t)(at[j] + r);
    if constexpr (!kPlain) scale[j] = (is_v ? c.v_scale : c.k_scale)[token];
    if (is_v) continue;
    if constexpr (kPlain) {
      raw[j] = *reinterpret_cast<const v4u*>(c.k + (token * D + l8 * 8) * 2);
    } else if constexpr (FMT == kKvQ8) {
      const v2u u = *reinterpret_cast<const v2u*>(c.k + token * D + l8 * 8);
      raw[j][0] = u[0], raw[j][1] = u[1];
    } else {
      raw[j][0] = reinterpret_cast<const uint32_t*>(c.k)[token * LANES + l8];
    }
  }
  float sgn[8];
  if constexpr (FMT == kKvTq4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) sgn[i] = c.t.signs[l8 * 8 + i] * (float)(1.0 / __builtin_sqrt((double)D));
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < NG; ++j) {
    if (at[j] < 0) continue;
    float x[8];
    if (is_v) {
      if constexpr (kPlain) {
        raw[j] = *reinterpret_cast<const v4u*>(&vh[(j * 8 + r) * D + l8 * 8]);
      } else {
        const v2u u = *reinterpret_cast<const v2u*>(&vb[(j * 8 + r) * D + l8 * 8]);
        raw[j][0] = u[0], raw[j][1] = u[1];
      }
    }
    if constexpr (kPlain) {
      unpack8(raw[j], kType, x);
    } else if constexpr (FMT == kKvQ8) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = (float)(int8_t)(raw[j][i / 4] >> (8 * (i & 3))) * scale[j];
    } else {
      // Codes as bytes: K's nibbles spread, V's already are.
      uint32_t lo = raw[j][0], hi = raw[j][1];
      if (!is_v) {
        const uint32_t ev = lo & 0x0f0f0f0fu, od = lo >> 4 & 0x0f0f0f0fu;
        lo = perm(od, ev, 0x05010400u);
        hi = perm(od, ev, 0x07030602u);
      }
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        uint32_t p0, p1;
        bytes_to_f16(c.t, w == 0 ? lo : hi, p0, p1);
        x[4 * w] = f16_to_f32(p0 & 0xffffu);
        x[4 * w + 1] = f16_to_f32(p0 >> 16);
        x[4 * w + 2] = f16_to_f32(p1 & 0xffffu);
        x[4 * w + 3] = f16_to_f32(p1 >> 16);
      }
      hadamard8<LANES>(x);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= scale[j] * sgn[i];
    }
    if (!live[j]) continue;
    const size_t row = (size_t)(g.row + 8 * j + r);
    const size_t to = row * (is_v ? a.v_stride : a.k_stride) + (size_t)h * D + l8 * 8;
    store8((is_v ? a.v : a.k) + to * (a.dtype == kKvRowF32 ? 4 : 2), a.dtype, x);
  }
}

// tq4 rows by the run, on the matrix cores: 4 wavefronts, 16 rows each, two of
// K and two of V.
template <int IO, int D>
EOS_DEV void append_tq4(const KvRowsArgs& a, const KvRun& g, long long at0, long long at1, long long at2,
                        long long at3, uint32_t* vw) {
  constexpr int KS = D / 32, NT = D / 16, LANES = D / 8;
  const KvCacheArgs& c = a.c;
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, part = lane >> 4, h = blockIdx.y;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool is_v = wave >= 2;
  const int half = wave & 1, p = 16 * half + r16;
  const long long base = r16 < 8 ? (half != 0 ? at2 : at0) : (half != 0 ? at3 : at1);
  const bool live = base >= 0 && p >= g.from && p < g.upto;
  v4u x[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) x[s] = v4u{0, 0, 0, 0};
  if (live) {
    const uint8_t* src = (is_v ? a.v : a.k) +
                         ((size_t)(g.row + p) * (is_v ? a.v_stride : a.k_stride) + (size_t)h * D + part * 8) * 2;
#pragma unroll
    for (int s = 0; s < KS; ++s) x[s] = *reinterpret_cast<const v4u*>(src + 64 * s);
  }
  double ss = 0.0;
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    float f[8];
    unpack8(x[s], IO, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += (double)f[i] * (double)f[i];
  }
  ss += __shfl_xor(ss, 16);
  ss += __shfl_xor(ss, 32);
  float scale = (float)__builtin_sqrt(ss * (1.0 / D));
  const bool none = scale < kTiny;
  const bool nan = !(scale <= kHuge);
  const float norm = none || nan ? 0.0f : scale * (float)__builtin_sqrt((double)D);
  scale = nan ? __builtin_nanf("") : none ? 0.0f : scale;
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const uint32_t* sg = reinterpret_cast<const uint32_t*>(c.t.signs) + 32 * s + 8 * part;
#pragma unroll
    for (int w = 0; w < 4; ++w)
      x[s][w] = none || nan ? 0u : x[s][w] ^ ((sg[2 * w] >> 16 & 0x8000u) | (sg[2 * w + 1] & 0x80000000u));
  }
  v4f y[NT];
  rotate16<IO == kKvRowBf16 ? kKvBf16 : kKvF16, D>(x, y);
  float e[7];
#pragma unroll
  for (int i = 0; i < 7; ++i) e[i] = c.t.edges[i] * norm;
  uint32_t word[KS];
#pragma unroll
  for (int w = 0; w < KS; ++w) {
    word[w] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) word[w] |= code_of(y[2 * w + i / 4][i & 3], e) << (4 * i);
  }
  if (live && part == 0) (is_v ? c.v_scale : c.k_scale)[base + r16 % 8] = scale;
  if (!is_v) {
    if (live) {
      uint32_t* dst = reinterpret_cast<uint32_t*>(c.k) + (size_t)(base + r16 % 8) * LANES + part;
#pragma unroll
      for (int w = 0; w < KS; ++w) dst[4 * w] = word[w];
    }
  } else {
#pragma unroll
    for (int w = 0; w < KS; ++w) vw[p * LANES + 4 * w + part] = word[w];
  }
}

template <int D>
EOS_DEV void append_tq4_run(const KvRowsArgs& a) {
  constexpr int LANES = D / 8, NG = kKvRun / 8;
  __shared__ __align__(16) uint32_t vw[kKvRun * LANES];
  const KvCacheArgs& c = a.c;
  KvRun g;
  int b;
  if (!find_run<kKvRun>(c, g, b)) return;
  long long at[NG];
  find_blocks<NG>(c, g, b, blockIdx.y, at);
  if (a.dtype == kKvRowF16)
    append_tq4<kKvRowF16, D>(a, g, at[0], at[1], at[2], at[3], vw);
  else
    append_tq4<kKvRowBf16, D>(a, g, at[0], at[1], at[2], at[3], vw);
  __syncthreads();
  // V: a group's 8 tokens of one dimension by one thread.
#pragma unroll
  for (int j = 0; j < NG; ++j) {
    if (at[j] < 0) continue;
    const int from = g.from > 8 * j ? g.from - 8 * j : 0;
    const int upto = g.upto - 8 * j < 8 ? g.upto - 8 * j : 8;
    // (D of the 256 threads, for the next group others)
    for (int dim = (threadIdx.x + 256 - j * D % 256) % 256; dim < D; dim += 256) {
      uint32_t* dst = reinterpret_cast<uint32_t*>(c.v) + (size_t)(at[j] / kKvGroup) * D + dim;
      uint32_t word = 0, mask = 0;
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const bool in = t >= from && t < upto;
        word |= in ? (vw[(j * 8 + t) * LANES + dim / 8] >> (4 * (dim & 7)) & 15u) << (4 * t) : 0u;
        mask |= in ? 15u << (4 * t) : 0u;
      }
      *dst = mask == ~0u ? word : (*dst & ~mask) | word;
    }
  }
}

template <int D>
EOS_DEV void read_tq4_run(const KvRowsArgs& a) {
  constexpr int KS = D / 32, NT = D / 16, LANES = D / 8, NG = kKvRun / 8;
  constexpr int VS = D + 16;  // bytes between V's rows in LDS: 8 rows on different banks
  __shared__ __align__(16) uint8_t vb[kKvRun * VS];
  static_assert(__alignof__(vb) >= 8 && VS % 8 == 0, "read by 8 bytes");
  const KvCacheArgs& c = a.c;
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, part = lane >> 4, h = blockIdx.y;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  KvRun g;
  int b;
  if (!find_run<kKvRun>(c, g, b)) return;
  long long at[NG];
  find_blocks<NG>(c, g, b, h, at);
#pragma unroll
  for (int j = 0; j < NG; ++j) {
    if (at[j] < 0) continue;
    for (int dim = (tid + 256 - j * D % 256) % 256; dim < D; dim += 256) {
      const uint32_t u = reinterpret_cast<const uint32_t*>(c.v)[(size_t)(at[j] / kKvGroup) * D + dim];
#pragma unroll
      for (int t = 0; t < 8; ++t) vb[(j * 8 + t) * VS + dim] = (uint8_t)(u >> (4 * t) & 15u);
    }
  }
  const bool is_v = wave >= 2;
  const int half = wave & 1, p = 16 * half + r16;
  const long long base = r16 < 8 ? (half != 0 ? at[2] : at[0]) : (half != 0 ? at[3] : at[1]);
  const bool live = base >= 0 && p >= g.from && p < g.upto;
  uint32_t word[KS] = {};
  float scale = 0.0f;
  if (live) {
    scale = (is_v ? c.v_scale : c.k_scale)[base + r16 % 8];
    if (!is_v) {
      const uint32_t* src = reinterpret_cast<const uint32_t*>(c.k) + (size_t)(base + r16 % 8) * LANES + part;
#pragma unroll
      for (int w = 0; w < KS; ++w) word[w] = src[4 * w];
    }
  }
  __syncthreads();
  v4u x[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    uint32_t lo, hi;
    if (is_v) {
      const v2u u = *reinterpret_cast<const v2u*>(&vb[p * VS + 32 * s + 8 * part]);
      lo = live ? u[0] : 0u;
      hi = live ? u[1] : 0u;
    } else {
      const uint32_t ev = word[s] & 0x0f0f0f0fu, od = word[s] >> 4 & 0x0f0f0f0fu;
      lo = perm(od, ev, 0x05010400u);
      hi = perm(od, ev, 0x07030602u);
    }
    uint32_t f[4];
    bytes_to_f16(c.t, lo, f[0], f[1]);
    bytes_to_f16(c.t, hi, f[2], f[3]);
    x[s] = v4u{f[0], f[1], f[2], f[3]};
  }
  v4f y[NT];
  rotate16<kKvF16, D>(x, y);
  if (!live) return;
  scale *= (float)(1.0 / __builtin_sqrt((double)D));
  const float* sg = c.t.signs + 8 * part;
  const size_t to = (size_t)(g.row + p) * (is_v ? a.v_stride : a.k_stride) + (size_t)h * D + 8 * part;
  uint8_t* dst = (is_v ? a.v : a.k) + to * (a.dtype == kKvRowF32 ? 4 : 2);
#pragma unroll
  for (int w = 0; w < KS; ++w) {
    float o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = y[2 * w + i / 4][i & 3] * (scale * sg[32 * w + i]);
    store8(dst + 32 * w * (a.dtype == kKvRowF32 ? 4 : 2), a.dtype, o);
  }
}

// ---------------------------------------------------------------- attention

template <int ROWS>
EOS_DEV bool find_tile(const KvAttnArgs& a, long long u, KvTile& t) {
  long long within = 0;
  if (a.c.offsets == nullptr) {
    const int per = (a.group + ROWS - 1) / ROWS;
    t.s = kv_seq(a.c, (int)(u / per));
    flag(a.c, t.s.bad);
    within = u % per;
  } else if (!find_seq(a.c, u, a.group, ROWS, 1, t.s, within)) {
    return false;
  }
  return kv_tile(t, within, ROWS, a.group, a.window, a.splits);
}

// int8 codes -> f16, exact: 0x6400 | b is 1024 + b.
EOS_DEV void codes_to_f16(uint32_t x, uint32_t (&out)[2]) {
  const uint32_t b = x ^ 0x80808080u;
  const v2h off = v2h{(_Float16)1152.0f, (_Float16)1152.0f};
  out[0] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, perm(0x64646464u, b, 0x04010400u)) - off);
  out[1] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, perm(0x64646464u, b, 0x04030402u)) - off);
}

// Eight 4-bit codes -> f16 magnitudes with their signs, in the order 0 2 4 6
// 1 3 5 7: the magnitudes' bytes by two table lookups each over four codes.
EOS_DEV void nibbles_to_f16(const KvTables& t, uint32_t x, uint32_t (&out)[4]) {
  const uint32_t e = x & 0x07070707u, o = (x >> 4) & 0x07070707u;
  const uint32_t eh = perm(t.hi[1], t.hi[0], e) | ((x << 4) & 0x80808080u);
  const uint32_t el = perm(t.lo[1], t.lo[0], e);
  const uint32_t oh = perm(t.hi[1], t.hi[0], o) | (x & 0x80808080u);
  const uint32_t ol = perm(t.lo[1], t.lo[0], o);
  out[0] = perm(eh, el, 0x05010400u);
  out[1] = perm(eh, el, 0x07030602u);
  out[2] = perm(oh, ol, 0x05010400u);
  out[3] = perm(oh, ol, 0x07030602u);
}

template <int FMT>
EOS_DEV uint32_t pack2(float a, float b) {
  if constexpr (FMT == kKvBf16)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f{a, b}), v2b));
  else
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f{a, b}), v2h));
}

// f16 / bf16 values with NaN and infinity apart: `x` keeps the finite ones, `pos`
// is 1 where +infinity or NaN stood, `neg` where -infinity or NaN did. Returns
// whether there was any.
template <int FMT>
EOS_DEV bool has_odd(v4u x) {
  constexpr uint32_t kExp = FMT == kKvF16 ? 0x7c00u : 0x7f80u;
  bool odd = false;
#pragma unroll
  for (int w = 0; w < 4; ++w) odd |= (x[w] & kExp) == kExp || (x[w] >> 16 & kExp) == kExp;
  return odd;
}
template <int FMT>
EOS_DEV void split_odd(v4u& x, v4u& pos, v4u& neg) {
  constexpr uint32_t kExp = FMT == kKvF16 ? 0x7c00u : 0x7f80u;
  constexpr uint32_t kOne = FMT == kKvF16 ? 0x3c00u : 0x3f80u;
  uint32_t keep[4], up[4], down[4];
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    keep[w] = up[w] = down[w] = 0;
#pragma unroll
    for (int s = 0; s < 32; s += 16) {
      const uint32_t u = x[w] >> s & 0xffffu;
      const bool odd = (u & kExp) == kExp, nan = odd && (u & 0x7fffu) != kExp;
      keep[w] |= (odd ? 0u : u) << s;
      up[w] |= (odd && (nan || u < 0x8000u) ? kOne : 0u) << s;
      down[w] |= (odd && (nan || u >= 0x8000u) ? kOne : 0u) << s;
    }
  }
  x = v4u{keep[0], keep[1], keep[2], keep[3]};
  pos = v4u{up[0], up[1], up[2], up[3]};
  neg = v4u{down[0], down[1], down[2], down[3]};
}
// Where a row's largest weight is put when its reference moves, as a power of
// two: f16 holds weights from 2^-24 to 2^16, so the more of them lie above its
// steps the higher the largest does; bf16 has f32's range. A weight (with its V
// scale) may grow by 2^8 before the reference moves again.
template <int FMT>
constexpr float kTop = FMT == kKvBf16 ? 0.0f : 7.0f;
template <int FMT>
constexpr float kMost = kTop<FMT> + 8.0f;

// Quantized formats: a row's weights are 2^(score - m) for its weights' sum and
// times the V scale for the products. One reference m follows the score plus
// the scale's exponent, over the keys that the row attends and no others, so that
// what it does not see or hardly weighs takes no bits from what it does. An
// exponent counts as -64 at least (a scale of zero): a weight stays below 2^(64
// + 15), and their sum above 2^(6 - 41) as scales end at 2^40.
constexpr float kMostProduct = 0x1p15f, kMostWeight = 0x1p79f;
EOS_DEV float scale_exp(float vs) {
  return vs > 0.0f ? fmaxf((float)__builtin_amdgcn_frexp_expf(vs), -64.0f) : -64.0f;
}
// x 2^d for d <= 0, by halves: a sum of weights may be far above 1 where 2^d
// alone is below f32's range.
EOS_DEV float decay(float x, float d) {
  const float h = __builtin_amdgcn_exp2f(0.5f * d);
  return x * h * h;
}

// What the odd values that a row sees add to its sum.
EOS_DEV float odd_sum(float up, float down) {
  const float inf = __builtin_inff();
  return (up > 0.0f ? inf : 0.0f) + (down > 0.0f ? -inf : 0.0f);
}

// Two elements of a query whose largest is below 2^kQUp: f16, and what f16
// leaves of them (not below 2^-14 before 2^-26 of the largest).
constexpr int kQUp = 12;
template <int FMT>
EOS_DEV v2u query2(float a, float b) {
  const uint32_t hi = pack2<FMT>(a, b);
  return v2u{hi, FMT == kKvTq4 ? pack2<FMT>(a - f16_to_f32(hi & 0xffffu), b - f16_to_f32(hi >> 16)) : 0u};
}

// Place in a word of 8 codes of operand slot i.
template <int FMT>
constexpr int slot_of(int i) {
  return FMT == kKvTq4 ? (i < 4 ? 2 * i : 2 * (i - 4) + 1) : i;
}

EOS_DEV float group_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
EOS_DEV float group_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// Eight outputs of one row: rotated back (tq4), divided, rounded and stored.
template <int FMT, int D>
EOS_DEV void finish_row(const KvAttnArgs& a, const KvSeq& s, int r, int h, int l8, bool live,
                        float (&x)[8], float m, float l) {
  if constexpr (FMT == kKvTq4) {
    hadamard8<D / 8>(x);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      x[i] *= a.c.t.signs[l8 * 8 + i] * (float)(1.0 / __builtin_sqrt((double)D));
  }
  if (!live) return;
  const float inv = l != 0.0f ? __fdiv_rn(1.0f, l) : 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] *= inv;
  const long long row = s.row0 + r / a.group;
  const int head = h * a.group + r % a.group;
  store8(a.out + ((size_t)row * a.out_stride + (size_t)head * D + l8 * 8) * 2, a.dtype, x);
  if (a.lse != nullptr && l8 == 0)
    a.lse[(size_t)row * a.heads + head] =
        l != 0.0f ? (m + __log2f(l)) * 0.69314718056f : -__builtin_inff();
}

// One workgroup: 16 query rows of a head group against keys [begin, end) of
// theirs, 32 keys a wavefront and step. Scores are computed as K q^T and the
// outputs as V^T p^T, so a lane's 8 scores (keys 8 g .. 8 g + 7 of the step, g
// = lane / 16, query lane % 16) are the 8 consecutive summands that its
// operand of the second product holds: nothing crosses lanes between the two.
// K's rows are taken in the order 8 (r / 4) + 4 j + r % 4 for that. Weights are
// rounded to 16 bits, the type that V has or is expanded to, since a matrix
// instruction takes both operands in one; sums and statistics are f32. Bound by
// the cache's bytes in 16 and 8 bits (one sequence of 131,072 tokens of q8, 32
// heads on 8 of 128: 61 us with the join, 4.5 TB/s, read again from the
// memory-side cache 52; 32 ragged ones in bf16: 67 us, 4.3 TB/s); in 4 bits by
// the vector unit, with 440 instructions for 32 keys of 128, half of them the
// codes' expansion (64 sequences, 0.6 GB: 166 us, 3.7 TB/s).
// The whole of the rows' keys goes to the output, else the sums go to place
// `at` of the parts.
template <int FMT, int D>
EOS_DEV void attn_segment(const KvAttnArgs& a, KvTile t, int h, int begin, int end, bool whole, size_t at) {
  constexpr bool kQuant = FMT == kKvQ8 || FMT == kKvTq4, kTwo = FMT == kKvTq4;
  constexpr int BITS = bits_of(FMT), KS = D / 32, NT = D / 16, LANES = D / 8;
  // Dimensions of V in one load of a lane, loads a step, words of a load.
  constexpr int VW = FMT == kKvTq4 ? (D >= 64 ? 4 : 2) : FMT == kKvQ8 ? 2 : 1;
  constexpr int VL = NT / VW, VWORDS = VW * BITS * 8 / 32;
  // Words of K a lane loads of each of its two keys.
  constexpr int KWORDS = D * BITS / 4 / 32;
  __shared__ float so[4][16 * D];
  __shared__ float sm[4][16], sl[4][16];
  const KvCacheArgs& c = a.c;
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // The same in every lane, as the compiler cannot see. Results depend on it: with
  // the loop's bounds in vector registers its body stood under a divergent
  // condition, and a build gave the weights and a fragment of V overlapping
  // registers, both live (f16, width 128). A host test looks for such operands in
  // the built kernels.
  h = __builtin_amdgcn_readfirstlane(h);
  begin = __builtin_amdgcn_readfirstlane(begin);
  end = __builtin_amdgcn_readfirstlane(end);
  t.s.b = __builtin_amdgcn_readfirstlane(t.s.b);
  t.s.n = __builtin_amdgcn_readfirstlane(t.s.n);
  t.s.len = __builtin_amdgcn_readfirstlane(t.s.len);
  t.s.keys = __builtin_amdgcn_readfirstlane(t.s.keys);
  t.r0 = __builtin_amdgcn_readfirstlane(t.r0);
  t.lo = __builtin_amdgcn_readfirstlane(t.lo);
  t.hi = __builtin_amdgcn_readfirstlane(t.hi);
  t.all_lo = __builtin_amdgcn_readfirstlane(t.all_lo);
  t.all_hi = __builtin_amdgcn_readfirstlane(t.all_hi);
  const int P = 1 << c.page_shift;
  const int rr = t.r0 + r16;
  const bool real = rr < t.s.n * a.group;
  const int qrow = real ? rr / a.group : 0;
  const int qpos = kv_row_pos(t.s, qrow);
  const int hi_c = real ? kv_min(qpos + 1, t.s.keys) : t.hi;
  const int lo_c = real && a.window > 0 ? qpos - a.window + 1 : 0;

  // The query as the second operand. Quantized formats take it in f16, its
  // largest element brought to [2^11, 2^12) by a power of two, tq4 rotated and,
  // since that has more bits than f16, in two terms (one would move the weights
  // by 2^-12 of a score).
  v4u q[KS], q2[kTwo ? KS : 1];
  float qs = a.scale;
  {
    const uint8_t* src = a.q + ((size_t)(t.s.row0 + qrow) * a.q_stride +
                                (size_t)(h * a.group + (real ? rr % a.group : 0)) * D) * 2;
    if constexpr (!kQuant) {
#pragma unroll
      for (int s = 0; s < KS; ++s)
        q[s] = real ? *reinterpret_cast<const v4u*>(src + (s * 32 + g * 8) * 2) : v4u{0, 0, 0, 0};
    } else {
      float x[KS][8];
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        if (real) load8(src + (g * (D / 4) + s * 8) * 2, a.dtype, x[s]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (!real) x[s][i] = 0.0f;
          if (FMT == kKvTq4) x[s][i] *= c.t.signs[g * (D / 4) + s * 8 + i];
        }
      }
      if constexpr (FMT == kKvTq4) {
#pragma unroll
        for (int st = 1; st < D / 4; st *= 2)
#pragma unroll
          for (int i = 0; i < D / 4; ++i)
            if ((i & st) == 0) {
              const float p = x[i / 8][i % 8], m = x[(i + st) / 8][(i + st) % 8];
              x[i / 8][i % 8] = p + m;
              x[(i + st) / 8][(i + st) % 8] = p - m;
            }
#pragma unroll
        for (int st = 16; st < 64; st *= 2)
#pragma unroll
          for (int i = 0; i < D / 4; ++i) {
            const float o = __shfl_xor(x[i / 8][i % 8], st);
            x[i / 8][i % 8] = (lane & st) != 0 ? o - x[i / 8][i % 8] : x[i / 8][i % 8] + o;
          }
        qs *= (float)(1.0 / __builtin_sqrt((double)D));
      }
      float most = 0.0f;
#pragma unroll
      for (int i = 0; i < D / 4; ++i) most = fmaxf(most, fabsf(x[i / 8][i % 8]));
      most = group_max(most);
      int ex = most > 0.0f && most < __builtin_inff() ? __builtin_amdgcn_frexp_expf(most) : 0;
      ex = kv_max(ex, -100) - kQUp;
      const float down = __builtin_amdgcn_ldexpf(1.0f, -ex);
      qs = __builtin_amdgcn_ldexpf(qs, ex);
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const v2u w = query2<FMT>(x[s][slot_of<FMT>(2 * i)] * down, x[s][slot_of<FMT>(2 * i + 1)] * down);
          q[s][i] = w[0];
          if (kTwo) q2[kTwo ? s : 0][i] = w[1];
        }
    }
  }

  v4f acc[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) acc[i] = v4f{0, 0, 0, 0};
  // Weights are 2^(score - m): m moves only when one (in quantized formats one
  // times its scale) passes its limit.
  float m = kLowest, l = 0.0f;
  const size_t head_bytes = ((size_t)D * BITS / 8) << c.page_shift;
  bool odd_seen = false;  // a value of V that is NaN or infinite in a masked step
  // A step's codes and scales as loaded: the next step's are on their way
  // while one is computed, and the page ids of the step after it.
  struct Raw {
    uint32_t k[2][KWORDS] = {}, v[VL][VWORDS] = {};
    float ks[kQuant ? 8 : 1] = {}, vs[kQuant ? 8 : 1] = {};
    bool vok = false;
  };
  // The page ids of this lane's keys of K and of V (-1: none there).
  int kid = -1, vid = -1;
  auto ids = [&](int tb) KV_INLINE {
    const int kt = tb + 16 * (r16 >> 3), vt = tb + 16 * (g >> 1);
    const int32_t* row = c.table + (size_t)t.s.b * c.table_stride;
    kid = kt < t.hi && kt + 16 > t.lo ? row[kt >> c.page_shift] : -1;
    vid = vt < t.hi && vt + 16 > t.lo ? row[vt >> c.page_shift] : -1;
  };
  auto fetch = [&](int tb, Raw& x) KV_INLINE {
    const int vt = tb + 16 * (g >> 1);
    const int kp = (unsigned)kid < (unsigned)c.pages ? kid : 0;
    x.vok = (unsigned)vid < (unsigned)c.pages;
    const int vp = x.vok ? vid : 0;
    if (!x.vok && vt < t.hi && vt + 16 > t.lo) atomicOr(c.status, kKvBadPage);
    const uint8_t* kb = c.k + ((size_t)kp * c.kv_heads + h) * head_bytes;
    const uint8_t* vb = c.v + ((size_t)vp * c.kv_heads + h) * head_bytes;
    const int vslot = (tb + 8 * g) & (P - 1);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int slot = (tb + 8 * (r16 >> 2) + 4 * j + (r16 & 3)) & (P - 1);
      const uint8_t* row = kb + (size_t)slot * (D * BITS / 8);
      if constexpr (!kQuant) {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const v4u w = *reinterpret_cast<const v4u*>(row + (s * 32 + g * 8) * 2);
#pragma unroll
          for (int i = 0; i < 4; ++i) x.k[j][4 * s + i] = w[i];
        }
      } else {
        __builtin_memcpy(x.k[j], __builtin_assume_aligned(row + g * (KWORDS * 4), KWORDS >= 4 ? 16 : KWORDS * 4),
                         KWORDS * 4);
      }
    }
    const uint8_t* vrow = vb + (size_t)(vslot / kKvGroup) * (D * BITS);
#pragma unroll
    for (int i = 0; i < VL; ++i)
      __builtin_memcpy(x.v[i], __builtin_assume_aligned(vrow + (i * 16 + r16) * (VWORDS * 4), VWORDS * 4),
                       VWORDS * 4);
    if constexpr (kQuant) {
      const size_t at = (((size_t)vp * c.kv_heads + h) << c.page_shift) + vslot;
      __builtin_memcpy(x.ks, __builtin_assume_aligned(c.k_scale + at, 16), 32);
      __builtin_memcpy(x.vs, __builtin_assume_aligned(c.v_scale + at, 16), 32);
    }
  };
  auto step = [&](int tb, Raw& raw) KV_INLINE {
    auto& kr = raw.k;
    auto& vr = raw.v;
    auto& ks = raw.ks;
    auto& vs = raw.vs;
    const bool vok = raw.vok;
    const bool masked = tb + 32 > t.all_hi || tb < t.all_lo || __any(!vok);

    v4f sc[2] = {v4f{0, 0, 0, 0}, v4f{0, 0, 0, 0}};
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t f[4];
        if constexpr (FMT == kKvTq4) {
          nibbles_to_f16(c.t, kr[j][s], f);
        } else if constexpr (FMT == kKvQ8) {
          uint32_t lo2[2], hi2[2];
          codes_to_f16(kr[j][2 * s], lo2);
          codes_to_f16(kr[j][2 * s + 1], hi2);
          f[0] = lo2[0], f[1] = lo2[1], f[2] = hi2[0], f[3] = hi2[1];
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) f[i] = kr[j][4 * s + i];
        }
        sc[j] = mfma16<FMT>(v4u{f[0], f[1], f[2], f[3]}, q[s], sc[j]);
        if constexpr (kTwo) sc[j] = mfma16<FMT>(v4u{f[0], f[1], f[2], f[3]}, q2[s], sc[j]);
      }
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = sc[i >> 2][i & 3] * qs;
      if (kQuant) x[i] *= ks[i];
    }
    uint32_t vmask[4] = {~0u, ~0u, ~0u, ~0u};
    if (masked) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int key = tb + 8 * g + i;
        const bool there = vok && key >= t.lo && key < t.hi;
        if (!(there && key >= lo_c && key < hi_c)) x[i] = -__builtin_inff();
        if (kQuant && !there) vs[i] = 0.0f;
        if (!there) vmask[i >> 1] &= (i & 1) != 0 ? 0x0000ffffu : 0xffff0000u;
      }
    }
    float p[8];
    if constexpr (!kQuant) {
      float mx = x[0];
#pragma unroll
      for (int i = 1; i < 8; ++i) mx = fmaxf(mx, x[i]);
      if (__any(mx > m + kMost<FMT>)) {
        const float nm = fmaxf(m, group_max(mx) - kTop<FMT>);
        const float f = __builtin_amdgcn_exp2f(m - nm);
        m = nm;
        l *= f;
#pragma unroll
        for (int i = 0; i < NT; ++i) acc[i] *= f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[i] = __builtin_amdgcn_exp2f(x[i] - m);
        l += p[i];
      }
    } else {
      float w[8];
      // (a masked key's scale may be NaN: it must not reach the row)
      auto weigh = [&](bool limit) KV_INLINE {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float d = x[i] - m;
          // (a score beyond 2^24 absorbs an exponent: nothing passes its limit)
          if (limit) {
            const float most = kMost<FMT> - scale_exp(vs[i]);
            d = d > most ? most : d;
          }
          p[i] = __builtin_amdgcn_exp2f(d);
          w[i] = masked && x[i] == -__builtin_inff() ? 0.0f : p[i] * vs[i];
        }
      };
      weigh(false);
      float mw = w[0], mp = p[0];
#pragma unroll
      for (int i = 1; i < 8; ++i) {
        mw = fmaxf(mw, w[i]);
        mp = fmaxf(mp, p[i]);
      }
      if (__any(mw > kMostProduct || mp > kMostWeight)) {
        float y = x[0] + scale_exp(vs[0]);
#pragma unroll
        for (int i = 1; i < 8; ++i) y = fmaxf(y, x[i] + scale_exp(vs[i]));
        const float nm = fmaxf(m, group_max(y) - kTop<FMT>);
        const float f = __builtin_amdgcn_exp2f(m - nm);
        l = decay(l, m - nm);
        m = nm;
#pragma unroll
        for (int i = 0; i < NT; ++i) acc[i] *= f;
        weigh(true);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        l += p[i];
        p[i] = w[i];
      }
    }
    v4u pf;
#pragma unroll
    for (int i = 0; i < 4; ++i) pf[i] = pack2<FMT>(p[slot_of<FMT>(2 * i)], p[slot_of<FMT>(2 * i + 1)]);
    if constexpr (!kQuant) {
      if (masked) {
        // Weight 0 does not stop a NaN or infinity: slots that hold no token
        // count as zero, and so do odd values until the loop is over.
        bool odd = false;
#pragma unroll
        for (int i = 0; i < VL; ++i) {
          v4u v = v4u{vr[i][0] & vmask[0], vr[i][1] & vmask[1], vr[i][2] & vmask[2], vr[i][3] & vmask[3]};
          if (__any(has_odd<FMT>(v))) {
            v4u pos, neg;
            split_odd<FMT>(v, pos, neg);
            odd = true;
          }
#pragma unroll
          for (int w = 0; w < 4; ++w) vr[i][w] = v[w];
        }
        odd_seen |= odd;
      }
    }
#pragma unroll
    for (int i = 0; i < VL; ++i)
#pragma unroll
      for (int w = 0; w < VW; ++w) {
        uint32_t f[4];
        if constexpr (FMT == kKvTq4) {
          nibbles_to_f16(c.t, vr[i][w], f);
        } else if constexpr (FMT == kKvQ8) {
          uint32_t lo2[2], hi2[2];
          codes_to_f16(vr[i][2 * w], lo2);
          codes_to_f16(vr[i][2 * w + 1], hi2);
          f[0] = lo2[0], f[1] = lo2[1], f[2] = hi2[0], f[3] = hi2[1];
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) f[k] = vr[i][k];
        }
        acc[i * VW + w] = mfma16<FMT>(v4u{f[0], f[1], f[2], f[3]}, pf, acc[i * VW + w]);
      }
  };
  // (where registers hold a second step: 32 sequences of 4,000 tokens, width 256
  // in tq4, 46 us without it, 111 with what it spills)
  constexpr bool kAhead = D * BITS <= 1024 && D < 256;
  const int first = begin + 32 * wave;
  Raw ra, rb;
  if (first < end) {
    ids(first);
    fetch(first, ra);
    ids(first + 128);
  }
  for (int tb = first; tb < end;) {
    if constexpr (kAhead) {
      if (tb + 128 < end) fetch(tb + 128, rb);
      ids(tb + 256);
      step(tb, ra);
      if ((tb += 128) >= end) break;
      if (tb + 128 < end) fetch(tb + 128, ra);
      ids(tb + 256);
      step(tb, rb);
      tb += 128;
    } else {
      step(tb, ra);
      if ((tb += 128) >= end) break;
      fetch(tb, ra);
      ids(tb + 128);
    }
  }

  if (!kQuant && odd_seen) {
    // The values left out, for the rows that see them.
    constexpr uint32_t kOne = FMT == kKvF16 ? 0x3c00u : 0x3f80u;
    for (int tb = first; tb < end; tb += 128) {
      const int key = tb + 8 * g, vp = kv_page(c, t.s.b, tb + 16 * (g >> 1));
      if (!(tb + 32 > t.all_hi || tb < t.all_lo || __any(vp < 0))) continue;
      uint32_t see[4] = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (vp >= 0 && key + i >= t.lo && key + i < t.hi && key + i >= lo_c && key + i < hi_c)
          see[i / 2] |= kOne << (16 * (i & 1));
      const v4u sees = v4u{see[0], see[1], see[2], see[3]};
      const uint8_t* vb = c.v + ((size_t)kv_max(vp, 0) * c.kv_heads + h) * head_bytes +
                          (size_t)((key & (P - 1)) / kKvGroup) * (D * BITS);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        v4u v = *reinterpret_cast<const v4u*>(vb + (n * 16 + r16) * 16), pos, neg;
        split_odd<FMT>(v, pos, neg);
        const v4f up = mfma16<FMT>(pos, sees, v4f{0, 0, 0, 0});
        const v4f down = mfma16<FMT>(neg, sees, v4f{0, 0, 0, 0});
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[n][k] += odd_sum(up[k], down[k]);
      }
    }
  }

  // The four wavefronts' parts, brought to one reference.
  l = group_sum(l);
  if (g == 0) {
    sm[wave][r16] = m;
    sl[wave][r16] = l;
  }
  __syncthreads();
  float top = sm[0][r16];
#pragma unroll
  for (int w = 1; w < 4; ++w) top = fmaxf(top, sm[w][r16]);
  const float f = __builtin_amdgcn_exp2f(m - top);
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k)
      so[wave][r16 * D + (i / VW) * 16 * VW + VW * (4 * g + k) + i % VW] = acc[i][k] * f;
  __syncthreads();
  for (int it = tid; it < 16 * LANES; it += 256) {
    const int r = it / LANES, l8 = it % LANES;
    float o[8], mt = sm[0][r], lt = 0.0f;
#pragma unroll
    for (int w = 1; w < 4; ++w) mt = fmaxf(mt, sm[w][r]);
#pragma unroll
    for (int w = 0; w < 4; ++w) lt += decay(sl[w][r], sm[w][r] - mt);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int at = r * D + l8 * 8 + i;
      o[i] = so[0][at] + so[1][at] + so[2][at] + so[3][at];
    }
    const bool live = t.r0 + r < t.s.n * a.group;
    if (whole) {
      finish_row<FMT, D>(a, t.s, t.r0 + r, h, l8, live, o, mt, lt);
    } else if (live) {
      reinterpret_cast<v4f*>(a.part + (at + r) * D + l8 * 8)[0] = v4f{o[0], o[1], o[2], o[3]};
      reinterpret_cast<v4f*>(a.part + (at + r) * D + l8 * 8)[1] = v4f{o[4], o[5], o[6], o[7]};
      if (l8 == 0) {
        a.part_ml[(at + r) * 2] = mt;
        a.part_ml[(at + r) * 2 + 1] = lt;
      }
    }
  }
}

// One split of one tile.
template <int FMT, int D>
EOS_DEV void attn_split(const KvAttnArgs& a) {
  const int split = blockIdx.x % a.splits, h = blockIdx.y;
  const long long u = blockIdx.x / a.splits;
  KvTile t;
  if (!find_tile<kKvTileRows>(a, u, t)) return;
  if (split >= t.splits && (split > 0 || a.splits > 1)) return;
  attn_segment<FMT, D>(a, t, h, t.base + split * t.chunk, kv_min(t.hi, t.base + (split + 1) * t.chunk),
                       a.splits == 1, (((size_t)u * a.c.kv_heads + h) * a.splits + split) * kKvTileRows);
}

// Steps of the sequences before each one, of a head: pre[b], and of all:
// pre[batch]. 256 threads, each with neighbouring sequences.
EOS_DEV void stream_steps(const KvAttnArgs& a, long long* pre) {
  __shared__ long long part[4];
  const KvCacheArgs& c = a.c;
  const int tid = threadIdx.x, lane = tid & 63, per = (c.batch + 255) / 256;
  long long sum = 0;
  for (int i = 0; i < per; ++i) {
    const int b = tid * per + i;
    if (b < c.batch) {
      const long long n = kv_seq_steps(c, b, a.group, a.window);
      pre[b] = n;
      sum += n;
    }
  }
  long long upto = sum;
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const long long x = __shfl_up(upto, o);
    if (lane >= o) upto += x;
  }
  if (lane == 63) part[tid >> 6] = upto;
  __syncthreads();
  long long at = upto - sum;
  for (int w = 0; w < tid >> 6; ++w) at += part[w];
  for (int i = 0; i < per; ++i) {
    const int b = tid * per + i;
    if (b < c.batch) {
      const long long n = pre[b];
      pre[b] = at;
      at += n;
    }
  }
  if (tid == 0) pre[c.batch] = part[0] + part[1] + part[2] + part[3];
  __syncthreads();
}

// One row a sequence, any lengths: equal shares of all steps (see kv_index.h).
template <int FMT, int D>
EOS_DEV void attn_stream(const KvAttnArgs& a) {
  __shared__ long long pre[kKvStreamBatch + 1];
  const KvCacheArgs& c = a.c;
  stream_steps(a, pre);
  const int tiles = kv_tiles_of(a.group);
  const long long total = pre[c.batch], all = total * c.kv_heads;
  const long long share = kv_share(all, a.workgroups), start = share * blockIdx.x;
  const long long end = start + share < all ? start + share : all;
  for (long long pos = start; pos < end;) {
    const int h = (int)(pos / total);
    const long long rel = pos - h * total;
    int b = 0;  // the last sequence that starts at or before rel
    for (int o = kKvStreamBatch; o > 0; o /= 2)
      if (b + o < c.batch && pre[b + o] <= rel) b += o;
    const int steps = (int)((pre[b + 1] - pre[b]) / tiles);
    const KvSegment g = kv_segment(rel, rel + (end - pos), pre[b], steps);
    KvTile t;
    t.s = kv_seq(c, b);
    flag(c, t.s.bad);
    kv_tile(t, g.tile, kKvTileRows, a.group, a.window, 1);
    attn_segment<FMT, D>(a, t, h, t.base + 128 * g.from, kv_min(t.hi, t.base + 128 * g.upto),
                         g.from == 0 && g.upto == steps,
                         kv_part(blockIdx.x, start, pos - g.from));
    pos += g.upto - g.from;
    __syncthreads();
  }
}

typedef float v16f __attribute__((ext_vector_type(16)));

template <int FMT>
EOS_DEV v16f mfma32(v4u a, v4u b, v16f c) {
  if constexpr (FMT == kKvBf16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8b, a),
                                                   __builtin_bit_cast(v8b, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a),
                                                  __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

// 16 bytes a lane from base + off straight into LDS: lane i's at lds + 16 i. A
// wait for the vector loads (lds_wait) and a barrier stand before their first
// use. Written out because the compiler, which cannot tell the two stages of a
// buffer apart, would wait for the builtin's before every read of the other.
EOS_DEV void load_lds16(uint32_t lds, const void* base, uint32_t off) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, %2"
      :
      : "s"(lds), "v"(off), "s"(base)
      : "memory", "m0");
}
EOS_DEV void lds_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
EOS_DEV uint32_t lds_offset(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}

// One 16-byte load of codes as 16-bit operands: BITS / 16 of 8 each.
template <int FMT>
EOS_DEV void expand(const KvTables& t, v4u x, v4u (&out)[16 / bits_of(FMT)]) {
  if constexpr (FMT == kKvTq4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t f[4];
      nibbles_to_f16(t, x[i], f);
      out[i] = v4u{f[0], f[1], f[2], f[3]};
    }
  } else if constexpr (FMT == kKvQ8) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t lo[2], hi[2];
      codes_to_f16(x[2 * i], lo);
      codes_to_f16(x[2 * i + 1], hi);
      out[i] = v4u{lo[0], lo[1], hi[0], hi[1]};
    }
  } else {
    out[0] = x;
  }
}

// One workgroup: 128 query rows of a head group, 32 a wavefront, against a
// split of their keys, 64 (where registers allow, else 32) at a time through
// two LDS stages that hold K and V as 16-bit operands; 16-bit formats are
// loaded straight into them. Products as in attn_segment, on 32 x 32 tiles:
// scores K q^T, outputs V^T p^T, so a lane (query lane % 32, half lane / 32) holds
// the scores of keys 16 k + 8 half .. + 7, its operand of the second product; K's
// rows are read with bits 2 and 3 exchanged for that.
// Two prompts of 8,192 rows in bf16, 32 heads on 8 of 128: 1.34 ms, 0.82
// PFLOP/s. Bound by issue and latency at two wavefronts a SIMD: the matrix
// unit is busy for a third of the time, without the loads it took 1.01 ms,
// without the exponentials 1.30. 256 rows a workgroup: 1.29 to 1.43 ms.
template <int FMT, int D>
EOS_DEV void attn_prompt(const KvAttnArgs& a) {
  constexpr bool kQuant = FMT == kKvQ8 || FMT == kKvTq4, kTwo = FMT == kKvTq4;
  constexpr int BITS = bits_of(FMT), KS = D / 16, NT = D / 32;
  constexpr int NK = D == 256 || (D == 128 && kTwo) ? 32 : 64, TT = NK / 32, BLK = NK / 16;
  // 16-byte pieces of 16 tokens and of a stage (of K, and as many of V), a
  // thread's loads, and the operand pieces of one.
  constexpr int C16 = D * BITS / 8, CH = BLK * C16, PER = (CH + 255) / 256, EX = 16 / BITS;
  constexpr int ROWC = D / 8;  // operand pieces of a K row
  constexpr int RS = ROWC >= 16 ? 1 : 16 / ROWC;  // K rows that share 256 bytes
  __shared__ v4u lk[2][NK * ROWC], lv[2][NK * ROWC];
  __shared__ float lsc[2][3][kQuant ? NK : 1];  // scales of K and of V, exponents of V's
  // Whether a stage that some row masks, or that lacks a page, held a NaN or
  // infinity in V: such values are staged as zero (weight 0 would not stop them)
  // and added at the end to the rows that see them.
  __shared__ int lodd;
  const KvCacheArgs& c = a.c;
  const int tid = threadIdx.x, lane = tid & 63, r32 = lane & 31, hh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // Workgroups go to the 8 XCDs in turn. An XCD takes whole heads, or shares
  // them with as few others as it can, so that the keys and values of few
  // heads pass through its L2; the last tiles of a sequence, which attend the
  // most keys, go first.
  const KvPlace at0 = kv_place(blockIdx.x, c.kv_heads, a.tiles * a.splits);
  if (at0.item >= a.tiles * a.splits) return;
  const int split = (int)(at0.item % a.splits), h = at0.head;
  const long long u = a.tiles - 1 - at0.item / a.splits;
  KvTile t;
  if (!find_tile<kKvPromptRows>(a, u, t)) return;
  if (split >= t.splits && (split > 0 || a.splits > 1)) return;
  const int P = 1 << c.page_shift;
  const int seq = __builtin_amdgcn_readfirstlane(t.s.b);
  const int lo = __builtin_amdgcn_readfirstlane(t.lo), hi = __builtin_amdgcn_readfirstlane(t.hi);
  const int begin = __builtin_amdgcn_readfirstlane(t.base + split * t.chunk);
  const int end = __builtin_amdgcn_readfirstlane(kv_min(t.hi, t.base + (split + 1) * t.chunk));
  const int all_lo = __builtin_amdgcn_readfirstlane(t.all_lo);
  const int all_hi = __builtin_amdgcn_readfirstlane(t.all_hi);
  const size_t head_bytes = ((size_t)D * BITS / 8) << c.page_shift;

  const int nrows = t.s.n * a.group, w0 = t.r0 + 32 * wave, rr = w0 + r32;
  const bool real = rr < nrows;
  const int qrow = real ? rr / a.group : 0;
  const int qpos = kv_row_pos(t.s, qrow);
  const int hi_c = real ? kv_min(qpos + 1, t.s.keys) : 0;
  const int lo_c = real && a.window > 0 ? qpos - a.window + 1 : 0;
  // Keys that some row and that every row of the wavefront attends.
  const bool busy = w0 < nrows;
  const int wp0 = kv_row_pos(t.s, w0 / a.group);
  const int wp1 = kv_row_pos(t.s, (kv_min(w0 + 32, nrows) - 1) / a.group);
  const int w_hi = __builtin_amdgcn_readfirstlane(busy ? kv_min(t.s.keys, wp1 + 1) : 0);
  const int w_lo = __builtin_amdgcn_readfirstlane(a.window > 0 ? wp0 - a.window + 1 : 0);
  const int w_all_hi = __builtin_amdgcn_readfirstlane(kv_min(t.s.keys, wp0 + 1));
  const int w_all_lo = __builtin_amdgcn_readfirstlane(a.window > 0 ? wp1 - a.window + 1 : 0);

  // Staging. K goes one stage ahead of V, so that a stage's scores can be
  // computed beside the exponentials of the one before. This thread's pieces
  // on their way, the page ids of the two stages ahead and, as bits, which of
  // the stages' 16-token blocks have one.
  v4u kr[PER], vr[PER];
  float scr = 0.0f;
  int pid1 = 0, pid2 = 0, ok0 = 0, ok1 = 0, ok2 = 0;
  // Page ids of a stage's blocks, one a lane, loaded a stage before their rows.
  int ids = 0;
  auto pages = [&](int tb) KV_INLINE {
    const int t16 = tb + 16 * (lane & (BLK - 1));
    ids = t16 < hi && t16 + 16 > lo
              ? c.table[(size_t)seq * c.table_stride + (t16 >> c.page_shift)]
              : -1;
  };
  // Those ids made safe (lane j: block j's), and which of them were pages.
  auto resolve = [&](int tb, int& pid) KV_INLINE {
    const bool in = (unsigned)ids < (unsigned)c.pages;
    const int t16 = tb + 16 * lane;
    if (!in && tid < BLK && t16 < hi && t16 + 16 > lo) atomicOr(c.status, kKvBadPage);
    pid = in ? ids : 0;
    pages(tb + NK);
    return (int)__ballot(in) & ((1 << BLK) - 1);
  };
  auto load = [&](const uint8_t* pool, int tb, int pid, v4u (&x)[PER]) KV_INLINE {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int id = tid + 256 * i;
      if (CH % 256 != 0 && id >= CH) break;
      // (a wavefront's pieces lie in one block of 16 tokens, or in several)
      const int blk = C16 >= 64 ? __builtin_amdgcn_readfirstlane(id / C16) : id / C16;
      const int rest = id - blk * C16;
      const int p = C16 >= 64 ? __builtin_amdgcn_readlane(pid, blk) : __shfl(pid, blk);
      x[i] = *reinterpret_cast<const v4u*>(
          pool + ((size_t)p * c.kv_heads + h) * head_bytes +
          (size_t)((tb + 16 * blk) & (P - 1)) * (D * BITS / 8) + rest * 16);
    }
  };
  // 16-bit formats go to LDS without registers: the thread's piece of K is the
  // one that its place in the swizzled stage holds.
  auto direct = [&](const uint8_t* pool, const v4u* lds, int tb, int pid, bool is_k) KV_INLINE {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int id = tid + 256 * i;
      const int blk = __builtin_amdgcn_readfirstlane(id / C16);
      const int row = id / ROWC;
      const uint32_t off = is_k ? (uint32_t)((row % 16) * ROWC + ((id % ROWC) ^ ((row / RS) & (ROWC - 1)))) * 16
                                : (uint32_t)(id % C16) * 16;
      const int p = __builtin_amdgcn_readlane(pid, blk);
      load_lds16(lds_offset(lds) + (uint32_t)(wave * 64 + 256 * i) * 16,
                 pool + ((size_t)p * c.kv_heads + h) * head_bytes +
                     (size_t)((tb + 16 * blk) & (P - 1)) * (D * 2),
                 off);
    }
  };
  // Whether a stage's V may hold what must not be staged as it is.
  auto odd_stage = [&](int tb, int ok) KV_INLINE {
    return ok != (1 << BLK) - 1 || tb + NK > all_hi || tb < all_lo;
  };
  auto load_v = [&](int st, int tb, int pid, int ok) KV_INLINE {
    if constexpr (!kQuant) {
      if (!odd_stage(tb, ok)) direct(c.v, lv[st], tb, pid, false);
      return;
    }
    load(c.v, tb, pid, vr);
    if constexpr (kQuant) {
      if (tid < 2 * NK) {
        const int tok = tb + tid % NK, blk = tid % NK / 16;
        const int p = __shfl(pid, blk);
        const float* sc = tid < NK ? c.k_scale : c.v_scale;
        const bool there = tok < hi && tok >= lo && (ok >> blk & 1) != 0;
        scr = there ? sc[(((size_t)p * c.kv_heads + h) << c.page_shift) + (tok & (P - 1))] : 0.0f;
      }
    }
  };
  auto load_k = [&](int st, int tb, int pid) KV_INLINE {
    if constexpr (kQuant)
      load(c.k, tb, pid, kr);
    else
      direct(c.k, lk[st], tb, pid, true);
  };
  auto store_k = [&](int st) KV_INLINE {
    if constexpr (!kQuant) return;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int id = tid + 256 * i;
      if (CH % 256 != 0 && id >= CH) break;
      const int blk = id / C16, rest = id % C16;
      v4u x[EX];
      expand<FMT>(c.t, kr[i], x);
      const int row = blk * 16 + rest / (ROWC / EX), c0 = rest % (ROWC / EX) * EX;
      const int sw = (row / RS) & (ROWC - 1);
#pragma unroll
      for (int e = 0; e < EX; ++e) lk[st][row * ROWC + ((c0 + e) ^ sw)] = x[e];
    }
  };
  auto store_v = [&](int st, int tb, int pid, int ok) KV_INLINE {
    if constexpr (!kQuant) {
      if (!odd_stage(tb, ok)) return;
      load(c.v, tb, pid, vr);
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int id = tid + 256 * i;
      if (CH % 256 != 0 && id >= CH) break;
      const int blk = id / C16, rest = id % C16;
      v4u x[EX];
      expand<FMT>(c.t, vr[i], x);
      const int grp = rest / (D / EX);
      if constexpr (!kQuant) {
        // Slots that hold no token may hold anything: zeros instead.
        const int t0 = tb + 16 * blk + 8 * grp;
        const bool there = (ok >> blk & 1) != 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int t2 = t0 + 2 * w;
          x[0][w] &= (there && t2 >= lo && t2 < hi ? 0xffffu : 0u) |
                     (there && t2 + 1 >= lo && t2 + 1 < hi ? 0xffff0000u : 0u);
        }
        if (has_odd<FMT>(x[0])) {
          v4u pos, neg;
          split_odd<FMT>(x[0], pos, neg);
          lodd = 1;
        }
      }
#pragma unroll
      for (int e = 0; e < EX; ++e) lv[st][(blk * 2 + grp) * D + rest % (D / EX) * EX + e] = x[e];
    }
    if constexpr (kQuant)
      if (tid < 2 * NK) {
        lsc[st][tid / NK][tid % NK] = scr;
        if (tid >= NK) lsc[st][2][tid % NK] = scale_exp(scr);
      }
  };

  if (tid == 0) lodd = 0;
  __syncthreads();
  if (begin < end) {
    pages(begin);
    ok0 = resolve(begin, pid2);
    load_k(0, begin, pid2);
    load_v(0, begin, pid2, ok0);
  }

  // The query as the second operand (see attn_segment).
  v4u q[KS], q2[kTwo ? KS : 1];
  float qs = fabsf(a.scale);
  {
    const uint8_t* src = a.q + ((size_t)(t.s.row0 + qrow) * a.q_stride +
                                (size_t)(h * a.group + (real ? rr % a.group : 0)) * D) * 2;
    const uint32_t neg = a.scale < 0.0f ? 0x80008000u : 0u;
    // (a factor of zero takes the query itself: the scores' own is never zero)
    const uint32_t keep = a.scale != 0.0f ? ~0u : 0u;
    if constexpr (!kQuant) {
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        q[s] = real ? *reinterpret_cast<const v4u*>(src + (s * 16 + hh * 8) * 2) : v4u{0, 0, 0, 0};
        q[s] = (q[s] ^ v4u{neg, neg, neg, neg}) & v4u{keep, keep, keep, keep};
      }
    } else {
      float x[KS][8];
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        if (real) load8(src + (s * 16 + hh * 8) * 2, a.dtype, x[s]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (!real) x[s][i] = 0.0f;
          if (FMT == kKvTq4) x[s][i] *= c.t.signs[s * 16 + hh * 8 + i];
        }
      }
      if constexpr (FMT == kKvTq4) {
#pragma unroll
        for (int st = 1; st < D / 2; st *= 2)
#pragma unroll
          for (int i = 0; i < D / 2; ++i)
            if ((i & st) == 0) {
              const float p = x[i / 8][i % 8], m = x[(i + st) / 8][(i + st) % 8];
              x[i / 8][i % 8] = p + m;
              x[(i + st) / 8][(i + st) % 8] = p - m;
            }
#pragma unroll
        for (int i = 0; i < D / 2; ++i) {
          const float o = __shfl_xor(x[i / 8][i % 8], 32);
          x[i / 8][i % 8] = hh != 0 ? o - x[i / 8][i % 8] : x[i / 8][i % 8] + o;
        }
        qs *= (float)(1.0 / __builtin_sqrt((double)D));
      }
      float most = 0.0f;
#pragma unroll
      for (int i = 0; i < D / 2; ++i) most = fmaxf(most, fabsf(x[i / 8][i % 8]));
      most = fmaxf(most, __shfl_xor(most, 32));
      int ex = most > 0.0f && most < __builtin_inff() ? __builtin_amdgcn_frexp_expf(most) : 0;
      ex = kv_max(ex, -100) - kQUp;
      float down = __builtin_amdgcn_ldexpf(1.0f, -ex);
      qs = __builtin_amdgcn_ldexpf(qs, ex);
      if (neg != 0) down = -down;
      if (keep == 0) down = 0.0f;
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const v2u w = query2<FMT>(x[s][slot_of<FMT>(2 * i)] * down, x[s][slot_of<FMT>(2 * i + 1)] * down);
          q[s][i] = w[0];
          if (kTwo) q2[kTwo ? s : 0][i] = w[1];
        }
    }
  }
  // Scores are compared before their factor, which must not be zero for it.
  qs = fmaxf(qs, 0x1p-120f);
  const float iqs = __fdiv_rn(1.0f, qs);

  v16f acc[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) acc[i] = v16f{0};
  float m = kLowest, l = 0.0f;
  constexpr float kFar = 0x1p20f;
  // What a score (quantized: a score times its factor, plus its scale's
  // exponent) may be before m moves.
  float lim = (m + kMost<FMT>) * (kQuant ? 1.0f : iqs);
  // K row of lane r32: token bits 2 and 3 exchanged.
  const int krow = (r32 & 19) | (r32 >> 1 & 4) | (r32 << 1 & 8);
  auto scores = [&](int st, v16f (&s)[TT]) KV_INLINE {
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) {
      s[tt] = v16f{0};
      const int row = tt * 32 + krow;
      const int sw = (row / RS) & (ROWC - 1);
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const v4u x = lk[st][row * ROWC + ((2 * k + hh) ^ sw)];
        s[tt] = mfma32<FMT>(x, q[k], s[tt]);
        if constexpr (kTwo) s[tt] = mfma32<FMT>(x, q2[k], s[tt]);
      }
    }
  };
  // One stage: `s` are its scores, `next` becomes those of the following one.
  auto step = [&](int st, int tb, v16f (&s)[TT], v16f (&next)[TT]) KV_INLINE {
    const bool has1 = tb + NK < end, has2 = tb + 2 * NK < end;
    if (has1) load_v(st ^ 1, tb + NK, pid1, ok1);
    if (has2) {
      ok2 = resolve(tb + 2 * NK, pid2);
      load_k(st, tb + 2 * NK, pid2);
    }
    if (tb < w_hi && tb + NK > w_lo) {
      const bool masked = tb + NK > w_all_hi || tb < w_all_lo || ok0 != (1 << BLK) - 1;
      if constexpr (kQuant) {
#pragma unroll
        for (int tt = 0; tt < TT; ++tt)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[tt][i] *= lsc[st][0][32 * tt + 16 * (i / 8) + 8 * hh + i % 8];
      }
      if (masked) {
#pragma unroll
        for (int tt = 0; tt < TT; ++tt)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int key = tb + 32 * tt + 16 * (i / 8) + 8 * hh + i % 8;
            if (!(key >= lo_c && key < hi_c && (ok0 >> (2 * tt + i / 8) & 1) != 0))
              s[tt][i] = -__builtin_inff();
          }
      }
      float mx = -__builtin_inff();
#pragma unroll
      for (int tt = 0; tt < TT; ++tt)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float y = s[tt][i];
          if constexpr (kQuant) y = __builtin_fmaf(y, qs, lsc[st][2][32 * tt + 16 * (i / 8) + 8 * hh + i % 8]);
          mx = fmaxf(mx, y);
        }
      float from = m;
      if (__any(mx > lim)) {
        const float nm = fmaxf(m, fmaxf(mx, __shfl_xor(mx, 32)) * (kQuant ? 1.0f : qs) - kTop<FMT>);
        const float f = __builtin_amdgcn_exp2f(m - nm);
        l = kQuant ? decay(l, m - nm) : l * f;
        m = from = nm;
        lim = (m + kMost<FMT>) * (kQuant ? 1.0f : iqs);
#pragma unroll
        for (int i = 0; i < NT; ++i) acc[i] *= f;
        // Scores so large that a product's rounding is no longer small beside 1:
        // they are rounded before they are compared with m, as m was, stage by
        // stage (any score passes this limit).
        const bool far = fabsf(m) > kFar && m > kLowest;
        if (far) lim = -__builtin_inff();
        if (__any(far)) {
#pragma unroll
          for (int tt = 0; tt < TT; ++tt)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float most = kMost<FMT>;
              if constexpr (kQuant) most -= lsc[st][2][32 * tt + 16 * (i / 8) + 8 * hh + i % 8];
              const float d = s[tt][i] * qs - m;
              s[tt][i] = (d > most ? most : d) * iqs;
            }
          from = 0.0f;
        }
      }
      scores(st ^ 1, next);
      v4u pf[2 * TT];
#pragma unroll
      for (int kk = 0; kk < 2 * TT; ++kk) {
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float x = s[kk / 2][8 * (kk % 2) + i];
          p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x, qs, -from));
          l += p[i];
          // (a masked key's scale may be NaN: it must not reach the row)
          if constexpr (kQuant)
            p[i] = x == -__builtin_inff() ? 0.0f : p[i] * lsc[st][1][16 * kk + 8 * hh + i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          pf[kk][i] = pack2<FMT>(p[slot_of<FMT>(2 * i)], p[slot_of<FMT>(2 * i + 1)]);
      }
#pragma unroll
      for (int kk = 0; kk < 2 * TT; ++kk)
#pragma unroll
        for (int n = 0; n < NT; ++n)
          acc[n] = mfma32<FMT>(lv[st][(2 * kk + hh) * D + 32 * n + r32], pf[kk], acc[n]);
    } else {
      scores(st ^ 1, next);
    }
    if (has1) store_v(st ^ 1, tb + NK, pid1, ok1);
    if (has2) store_k(st);
    if constexpr (!kQuant) lds_wait();
    __syncthreads();
    ok0 = ok1;
    ok1 = ok2;
    pid1 = pid2;
  };
  if (begin < end) {
    store_k(0);
    store_v(0, begin, pid2, ok0);
    if (begin + NK < end) {
      ok1 = resolve(begin + NK, pid1);
      load_k(1, begin + NK, pid1);
      store_k(1);
    }
    if constexpr (!kQuant) lds_wait();
  }
  __syncthreads();
  if (begin < end) {
    v16f sa[TT], sb[TT];
    scores(0, sa);
    for (int tb = begin;;) {
      step(0, tb, sa, sb);
      if ((tb += NK) >= end) break;
      step(1, tb, sb, sa);
      if ((tb += NK) >= end) break;
    }
  }

  if (!kQuant && lodd != 0) {
    // The values of V that were left out, for the rows that see them.
    constexpr uint32_t kOne = FMT == kKvF16 ? 0x3c00u : 0x3f80u;
    for (int tb = begin; tb < end; tb += 16) {
      const int stage = begin + (tb - begin) / NK * NK;
      if (stage + NK <= all_hi && stage >= all_lo) {
        bool there = true;
#pragma unroll
        for (int i = 0; i < BLK; ++i) there &= kv_page(c, seq, stage + 16 * i) >= 0;
        if (there) continue;
      }
      const int page = kv_page(c, seq, tb), key = tb + 8 * hh;
      uint32_t see[4] = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (key + i >= lo_c && key + i < hi_c && page >= 0) see[i / 2] |= kOne << (16 * (i & 1));
      const v4u sees = v4u{see[0], see[1], see[2], see[3]};
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        v4u v = *reinterpret_cast<const v4u*>(
            c.v + ((size_t)kv_max(page, 0) * c.kv_heads + h) * head_bytes +
            ((size_t)((key & (P - 1)) / kKvGroup) * D + 32 * n + r32) * 16);
        v4u pos, neg;
        split_odd<FMT>(v, pos, neg);
        const v16f up = mfma32<FMT>(pos, sees, v16f{0}), down = mfma32<FMT>(neg, sees, v16f{0});
#pragma unroll
        for (int k = 0; k < 16; ++k) acc[n][k] += odd_sum(up[k], down[k]);
      }
    }
  }
  l += __shfl_xor(l, 32);
  if (a.splits > 1) {
    if (!real) return;
    const size_t at = (((size_t)u * c.kv_heads + h) * a.splits + split) * kKvPromptRows + 32 * wave + r32;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        *reinterpret_cast<v4f*>(a.part + at * D + 32 * n + 8 * k + 4 * hh) =
            v4f{acc[n][4 * k], acc[n][4 * k + 1], acc[n][4 * k + 2], acc[n][4 * k + 3]};
    if (hh == 0) {
      a.part_ml[at * 2] = m;
      a.part_ml[at * 2 + 1] = l;
    }
    return;
  }
  float inv = l != 0.0f ? __fdiv_rn(1.0f, l) : 0.0f;
  if constexpr (FMT == kKvTq4) {
    // The rotation back, over the dimensions as a lane holds them: 32 n + 8
    // (k / 4) + 4 half + k % 4.
    auto both = [&](int n0, int k0, int n1, int k1) {
      const float p = acc[n0][k0], o = acc[n1][k1];
      acc[n0][k0] = p + o;
      acc[n1][k1] = p - o;
    };
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int b = 1; b < 16; b *= 2)
#pragma unroll
        for (int k = 0; k < 16; ++k)
          if ((k & b) == 0) both(n, k, n, k + b);
#pragma unroll
    for (int b = 1; b < NT; b *= 2)
#pragma unroll
      for (int n = 0; n < NT; ++n)
        if ((n & b) == 0)
#pragma unroll
          for (int k = 0; k < 16; ++k) both(n, k, n + b, k);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const float o = __shfl_xor(acc[n][k], 32);
        acc[n][k] = (hh != 0 ? o - acc[n][k] : acc[n][k] + o) *
                    c.t.signs[32 * n + 8 * (k / 4) + 4 * hh + k % 4];
      }
    inv *= (float)(1.0 / __builtin_sqrt((double)D));
  }
  if (!real) return;
  const long long row = t.s.row0 + qrow;
  const int head = h * a.group + rr % a.group;
  uint8_t* dst = a.out + ((size_t)row * a.out_stride + (size_t)head * D) * 2;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = acc[n][4 * k + i] * inv;
      v2u w;
      if (a.dtype == kKvRowF16)
        w = v2u{f32_to_f16(o[0]) | f32_to_f16(o[1]) << 16, f32_to_f16(o[2]) | f32_to_f16(o[3]) << 16};
      else
        w = v2u{f32_to_bf16(o[0]) | f32_to_bf16(o[1]) << 16, f32_to_bf16(o[2]) | f32_to_bf16(o[3]) << 16};
      *reinterpret_cast<v2u*>(dst + (32 * n + 8 * k + 4 * hh) * 2) = w;
    }
  if (a.lse != nullptr && hh == 0)
    a.lse[(size_t)row * a.heads + head] =
        l != 0.0f ? (m + __log2f(l)) * 0.69314718056f : -__builtin_inff();
}

// One split's part of a row, D / 8 lanes.
struct Part {
  v4f lo, hi;
  float m, l;
};
template <int D>
EOS_DEV Part load_part(const KvAttnArgs& a, size_t p) {
  const int l8 = threadIdx.x % (D / 8);
  Part x;
  x.lo = reinterpret_cast<const v4f*>(a.part + p * D + l8 * 8)[0];
  x.hi = reinterpret_cast<const v4f*>(a.part + p * D + l8 * 8)[1];
  x.m = a.part_ml[p * 2];
  x.l = a.part_ml[p * 2 + 1];
  return x;
}

// A row from its n parts, part(i) loading the i-th and `first` holding a lane
// group's first one: each lane group its own parts with a running reference
// as in attn_segment, then the groups.
template <int FMT, int D, class F>
EOS_DEV void join_parts(const KvAttnArgs& a, const KvSeq& s, int r, int h, int n, Part first, F part) {
  constexpr int LANES = D / 8, NG = 256 / LANES;
  __shared__ __align__(16) float so[NG][D];
  __shared__ float sl[NG], sm[NG];
  const int tid = threadIdx.x, l8 = tid % LANES, grp = tid / LANES;
  float x[8] = {}, m = kLowest, l = 0.0f;
  for (int i = grp; i < n; i += NG) {
    const Part p = i == grp ? first : part(i);
    const float nm = fmaxf(m, p.m), fo = __builtin_amdgcn_exp2f(m - nm), fn = __builtin_amdgcn_exp2f(p.m - nm);
    l = decay(l, m - nm) + decay(p.l, p.m - nm);
    m = nm;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      x[k] = x[k] * fo + p.lo[k] * fn;
      x[4 + k] = x[4 + k] * fo + p.hi[k] * fn;
    }
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) so[grp][l8 * 8 + k] = x[k];
  if (l8 == 0) {
    sl[grp] = l;
    sm[grp] = m;
  }
  __syncthreads();
  if (tid >= LANES) return;
  const int used = kv_min(n, NG);
  float top = kLowest;
  for (int i = 0; i < used; ++i) top = fmaxf(top, sm[i]);
  l = 0.0f;
#pragma unroll
  for (int k = 0; k < 8; ++k) x[k] = 0.0f;
  for (int i = 0; i < used; ++i) {
    const float f = __builtin_amdgcn_exp2f(sm[i] - top);
    l += decay(sl[i], sm[i] - top);
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] += so[i][l8 * 8 + k] * f;
  }
  finish_row<FMT, D>(a, s, r, h, l8, true, x, top, l);
}

// Joins a row's splits: one workgroup a row and head, D / 8 lanes a split. The
// first splits' parts are loaded before it is known how many there are, so
// that they do not wait for the sequence's numbers.
template <int FMT, int D>
EOS_DEV void attn_join(const KvAttnArgs& a) {
  const KvCacheArgs& c = a.c;
  const int grp = threadIdx.x / (D / 8), head = blockIdx.y, h = head / a.group, rows = a.tile_rows;
  KvTile t;
  size_t at;
  int r;
  Part first = {v4f{0, 0, 0, 0}, v4f{0, 0, 0, 0}, kLowest, 0.0f};
  if (c.offsets == nullptr) {
    r = head % a.group;
    at = (((size_t)blockIdx.x * ((a.group + rows - 1) / rows) + r / rows) * c.kv_heads + h) * a.splits * rows + r % rows;
    if (grp < a.splits) first = load_part<D>(a, at + (size_t)grp * rows);
    t.s = kv_seq(c, blockIdx.x);
  } else {
    long long within = 0;
    if (!find_seq(c, blockIdx.x, 1, 1, 0, t.s, within)) return;
    if (within < 0 || within >= t.s.n) return;
    r = (int)within * a.group + head % a.group;
    const long long u = kv_unit_base(c, t.s.b, a.group, rows, 1) + r / rows;
    at = ((size_t)u * c.kv_heads + h) * a.splits * rows + r % rows;
    if (grp < a.splits) first = load_part<D>(a, at + (size_t)grp * rows);
  }
  kv_tile(t, r / rows, rows, a.group, a.window, a.splits);
  join_parts<FMT, D>(a, t.s, r, h, t.splits, first,
                     [&](int i) KV_INLINE { return load_part<D>(a, at + (size_t)i * rows); });
}

// The same for few splits: a workgroup has as many heads of a row as it has
// lane groups, each of which goes through its head's splits (1,024 rows x 8
// heads in two splits: 5 us, by one workgroup a row and head 20).
template <int FMT, int D>
EOS_DEV void attn_join_few(const KvAttnArgs& a) {
  constexpr int LANES = D / 8, NG = 256 / LANES;
  const KvCacheArgs& c = a.c;
  const int l8 = threadIdx.x % LANES, rows = a.tile_rows;
  const int head = blockIdx.y * NG + threadIdx.x / LANES, h = head / a.group;
  KvTile t;
  long long within = 0;
  if (c.offsets == nullptr) {
    t.s = kv_seq(c, blockIdx.x);
  } else if (!find_seq(c, blockIdx.x, 1, 1, 0, t.s, within)) {
    return;
  }
  if (within < 0 || within >= t.s.n) return;
  const bool live = head < a.heads;
  const int r = (int)within * a.group + head % a.group;
  kv_tile(t, r / rows, rows, a.group, a.window, a.splits);
  const long long u = (c.offsets == nullptr ? (long long)t.s.b * ((a.group + rows - 1) / rows)
                                            : kv_unit_base(c, t.s.b, a.group, rows, 1)) +
                      r / rows;
  const size_t at = ((size_t)u * c.kv_heads + h) * a.splits * rows + r % rows;
  float x[8] = {}, m = kLowest, l = 0.0f;
  const int n = live ? t.splits : 0;
  Part p[kKvFewSplits];
#pragma unroll
  for (int i = 0; i < kKvFewSplits; ++i)
    if (i < n) p[i] = load_part<D>(a, at + (size_t)i * rows);
#pragma unroll
  for (int i = 0; i < kKvFewSplits; ++i)
    if (i < n) {
      const float nm = fmaxf(m, p[i].m);
      const float fo = __builtin_amdgcn_exp2f(m - nm), fn = __builtin_amdgcn_exp2f(p[i].m - nm);
      l = decay(l, m - nm) + decay(p[i].l, p[i].m - nm);
      m = nm;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        x[k] = x[k] * fo + p[i].lo[k] * fn;
        x[4 + k] = x[4 + k] * fo + p[i].hi[k] * fn;
      }
    }
  finish_row<FMT, D>(a, t.s, r, h, l8, live, x, m, l);
}

// Joins what the stream's workgroups left of a row, where more than one had
// it, and writes the rows that have no key.
template <int FMT, int D>
EOS_DEV void attn_stream_join(const KvAttnArgs& a) {
  __shared__ long long pre[kKvStreamBatch + 1];
  const KvCacheArgs& c = a.c;
  const int grp = threadIdx.x / (D / 8), b = blockIdx.x, head = blockIdx.y, h = head / a.group;
  const int tiles = kv_tiles_of(a.group), r = head % a.group;
  const KvSeq s = kv_seq(c, b);
  flag(c, s.bad);
  stream_steps(a, pre);
  const long long total = pre[c.batch], share = kv_share(total * c.kv_heads, a.workgroups);
  const int steps = (int)((pre[b + 1] - pre[b]) / tiles);
  const long long tile = h * total + pre[b] + (long long)(r / kKvTileRows) * steps;
  const long long w0 = tile / share, w1 = steps > 0 ? (tile + steps - 1) / share : w0 - 1;
  if (w0 == w1) return;
  auto part = [&](int i) KV_INLINE {
    return load_part<D>(a, (size_t)kv_part(w0 + i, (w0 + i) * share, tile) + r % kKvTileRows);
  };
  const int n = (int)(w1 - w0 + 1);
  Part first = {v4f{0, 0, 0, 0}, v4f{0, 0, 0, 0}, kLowest, 0.0f};
  if (grp < n) first = part(grp);
  join_parts<FMT, D>(a, s, r, h, n, first, part);
}

}  // namespace

#define KV_KERNELS(NAME, FMT, D)                                                             \
  extern "C" __global__ __launch_bounds__(FMT == kKvTq4 ? 256 : 2 * D, D == 256 ? 2 : 4) void eos_kv_append_##NAME##_##D( \
      KvRowsArgs a) {                                                                        \
    if constexpr (FMT == kKvTq4)                                                             \
      append_tq4_run<D>(a);                                                                  \
    else                                                                                     \
      append_run<FMT, D, kKvRun>(a);                                                         \
  }                                                                                          \
  extern "C" __global__ __launch_bounds__(2 * D) void eos_kv_append1_##NAME##_##D(KvRowsArgs a) { \
    append_run<FMT, D, kKvGroup>(a);                                                         \
  }                                                                                          \
  extern "C" __global__ __launch_bounds__(FMT == kKvTq4 ? 256 : 2 * D) void eos_kv_read_##NAME##_##D( \
      KvRowsArgs a) {                                                                        \
    if constexpr (FMT == kKvTq4)                                                             \
      read_tq4_run<D>(a);                                                                    \
    else                                                                                     \
      read_run<FMT, D, kKvRun>(a);                                                           \
  }                                                                                          \
  extern "C" __global__ __launch_bounds__(2 * D) void eos_kv_read1_##NAME##_##D(KvRowsArgs a) {  \
    read_run<FMT, D, kKvGroup>(a);                                                           \
  }                                                                                          \
  extern "C" __global__ __launch_bounds__(256, D * bits_of(FMT) > 2048 ? 1 : 2) void eos_kv_split_##NAME##_##D(KvAttnArgs a) {    \
    attn_split<FMT, D>(a);                                                                   \
  }                                                                                          \
  extern "C" __global__ __launch_bounds__(256, D == 256 ? 1 : 2) void eos_kv_prompt_##NAME##_##D(  \
      KvAttnArgs a) {                                                                        \
    attn_prompt<FMT, D>(a);                                                               \
  }                                                                                          \
  extern "C" __global__ __launch_bounds__(256, D * bits_of(FMT) > 2048 ? 1 : 2) void eos_kv_stream_##NAME##_##D( \
      KvAttnArgs a) {                                                                        \
    attn_stream<FMT, D>(a);                                                                  \
  }                                                                                          \
  extern "C" __global__ __launch_bounds__(256) void eos_kv_stream_join_##NAME##_##D(KvAttnArgs a) { \
    attn_stream_join<FMT, D>(a);                                                             \
  }                                                                                          \
  extern "C" __global__ __launch_bounds__(256) void eos_kv_join_##NAME##_##D(KvAttnArgs a) {     \
    attn_join<FMT, D>(a);                                                                    \
  }                                                                                          \
  extern "C" __global__ __launch_bounds__(256) void eos_kv_join_few_##NAME##_##D(KvAttnArgs a) { \
    attn_join_few<FMT, D>(a);                                                                \
  }
#define KV_FORMATS(D)           \
  KV_KERNELS(f16, kKvF16, D)    \
  KV_KERNELS(bf16, kKvBf16, D)  \
  KV_KERNELS(q8, kKvQ8, D)      \
  KV_KERNELS(tq4, kKvTq4, D)

KV_FORMATS(32)
KV_FORMATS(64)
KV_FORMATS(128)
KV_FORMATS(256)
