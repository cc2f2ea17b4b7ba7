// Rows in microscaled 4-bit floating point on gfx950: quantised, taken back,
// and multiplied.
//
// A block is 32 consecutive values of a row; it has the scale 2^e, held as the
// byte e + 127, with e = floor(log2(max |x|)) - 2 in -127..127, and codes of
// four bits, sign and one of 0, .5, 1, 1.5, 2, 3, 4, 6: x / 2^e rounded to the
// nearest (ties to the even code), saturating. A block with an infinity or a
// NaN has scale byte 255 and stands for NaN.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mx_args.h"

#define EOS_DEV __device__ __forceinline__

namespace {

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef __bf16 v2b __attribute__((ext_vector_type(2)));
typedef uint16_t v2s __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));

constexpr int size_of(int type) { return type == kMxF32 ? 4 : 2; }

// The value of lane ^ 1 or ^ 2.
template <int CTRL>
EOS_DEV uint32_t dpp(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true);
}

EOS_DEV float bits_f(uint32_t u) { return __builtin_bit_cast(float, u); }

// Eight consecutive values of a row as they stand in memory, zeros from
// `left` on.
template <int T>
struct Eight {
  uint32_t u[T == kMxF32 ? 8 : 4];
};
template <int T>
EOS_DEV Eight<T> load8(const uint8_t* p, int left) {
  Eight<T> e = {};
  if (left >= 8) {
    const v4u a = *reinterpret_cast<const v4u*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) e.u[i] = a[i];
    if constexpr (T == kMxF32) {
      const v4u b = reinterpret_cast<const v4u*>(p)[1];
#pragma unroll
      for (int i = 0; i < 4; ++i) e.u[4 + i] = b[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) {
        if constexpr (T == kMxF32) e.u[i] = reinterpret_cast<const uint32_t*>(p)[i];
        else e.u[i / 2] |= (uint32_t) reinterpret_cast<const uint16_t*>(p)[i] << 16 * (i % 2);
      }
  }
  return e;
}

// The largest magnitude's bits (of its own type: they order as the values do,
// infinity and NaN last).
template <int T>
EOS_DEV uint32_t most8(const Eight<T>& e) {
  if constexpr (T == kMxF32) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, e.u[i] & 0x7fffffffu);
    return m;
  } else {
    v2s m = {};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      m = __builtin_elementwise_max(m, __builtin_bit_cast(v2s, e.u[i] & 0x7fff7fffu));
    return max(m[0], m[1]);
  }
}

// A block's scale byte from its largest magnitude's bits.
template <int T>
EOS_DEV uint32_t scale_byte(uint32_t most) {
  uint32_t e;
  if constexpr (T == kMxBf16) e = most >> 7;
  else if constexpr (T == kMxF32) e = most >> 23;
  else e = most >= 0x7c00u ? 255u
                           : __builtin_bit_cast(uint32_t, (float)__builtin_bit_cast(_Float16, (uint16_t)most)) >> 23;
  return e == 255 ? 255u : e > 2 ? e - 2 : 0u;
}
// The scale as a float (255: any, its codes do not matter).
EOS_DEV float scale_value(uint32_t byte) { return byte ? bits_f(byte << 23) : 0x1p-127f; }

// Codes of eight values, element j at bits 4 j.
template <int T>
EOS_DEV uint32_t codes8(const Eight<T>& e, float scale) {
  uint32_t c = 0;
  if constexpr (T == kMxF32) {
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, bits_f(e.u[0]), bits_f(e.u[1]), scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, bits_f(e.u[2]), bits_f(e.u[3]), scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, bits_f(e.u[4]), bits_f(e.u[5]), scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, bits_f(e.u[6]), bits_f(e.u[7]), scale, 3);
  } else if constexpr (T == kMxBf16) {
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(v2b, e.u[0]), scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(v2b, e.u[1]), scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(v2b, e.u[2]), scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(v2b, e.u[3]), scale, 3);
  } else {
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(v2h, e.u[0]), scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(v2h, e.u[1]), scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(v2h, e.u[2]), scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(v2h, e.u[3]), scale, 3);
  }
  return c;
}

// A quarter of a block, by four lanes side by side: its scale byte and codes.
template <int T>
EOS_DEV uint32_t quarter(const Eight<T>& e, uint32_t& byte) {
  uint32_t m = most8<T>(e);
  m = max(m, dpp<0xb1>(m));  // quad_perm 1 0 3 2
  m = max(m, dpp<0x4e>(m));  // quad_perm 2 3 0 1
  byte = scale_byte<T>(m);
  return byte == 255 ? 0u : codes8<T>(e, scale_value(byte));
}

// ------------------------------------------------------------ quantised rows

// Four lanes a block, eight values a lane: every load and store of a wavefront
// is of consecutive bytes.
template <int T>
EOS_DEV void quantize(const MxQuantArgs& a) {
  const long long first = (long long)blockIdx.x * 64;  // blocks of all rows in order
  const long long row0 = first / a.blocks;
  const uint32_t in = (uint32_t)(first - row0 * a.blocks) + threadIdx.x / 4;
  const uint32_t over = in / (uint32_t)a.blocks;
  const long long row = row0 + over;
  if (row >= a.rows) return;
  const int block = (int)(in - over * a.blocks);
  const int at = block * kMxBlock + (threadIdx.x & 3) * 8;
  const Eight<T> e = load8<T>(a.x + row * a.stride + (long long)at * size_of(T), a.k - at);
  uint32_t byte;
  const uint32_t c = quarter<T>(e, byte);
  const long long b = row * a.blocks + block;
  reinterpret_cast<uint32_t*>(a.codes)[b * 4 + (threadIdx.x & 3)] = c;
  if ((threadIdx.x & 3) == 0) a.scales[b] = (uint8_t)byte;
}

// The same into laid-out tiles: a wavefront a tile and step, four steps a
// workgroup.
template <int T>
EOS_DEV void lay(const MxQuantArgs& a) {
  const MxLaid& o = a.laid;
  const int wave = threadIdx.x / 64, lane = threadIdx.x & 63;
  const long long tile = blockIdx.x / (unsigned)o.quads;
  const int quad = (int)(blockIdx.x - tile * o.quads);
  const int step = quad * 4 + wave;
  uint8_t* scales = o.scales + (tile * o.quads + quad) * kMxScaleBytes + wave;
  if constexpr (T == kMxCodes) {
    const long long row = tile * kMxTile + lane % 16;
    const int block = step * 4 + lane / 16;
    v4u c = {};
    uint32_t byte = 0;
    if (row < a.rows && block < a.blocks) {
      c = *reinterpret_cast<const v4u*>(a.x + (row * a.blocks + block) * 16);
      byte = a.xs[row * a.blocks + block];
    }
    if (step < o.steps)
      *reinterpret_cast<v4u*>(o.codes + (tile * o.steps + step) * kMxTileBytes + lane * 16) = c;
    scales[lane * 4] = (uint8_t)byte;
  } else {
    const int at = step * kMxStep + (lane % 16) * 8;
    Eight<T> e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long row = tile * kMxTile + i * 4 + lane / 16;
      e[i] = Eight<T>{};
      if (row < a.rows) e[i] = load8<T>(a.x + row * a.stride + (long long)at * size_of(T), a.k - at);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int l = lane % 16 / 4 * 16 + i * 4 + lane / 16;  // the lane that multiplies it
      uint32_t byte;
      const uint32_t c = quarter<T>(e[i], byte);
      if (step < o.steps)
        reinterpret_cast<uint32_t*>(o.codes + (tile * o.steps + step) * kMxTileBytes)[l * 4 + (lane & 3)] = c;
      if ((lane & 3) == 0) scales[l * 4] = (uint8_t)byte;
    }
  }
}

EOS_DEV uint32_t pack_bf16(float x, float y) {
  return (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)x) | (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)y) << 16;
}
EOS_DEV uint32_t pack_f16(float x, float y) {
  return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)x) | (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)y) << 16;
}

// The value of a code times a power of two, exactly: sign, two bits of exponent
// and one of fraction, put where a float has its own, are 2^-126 of it.
EOS_DEV float level(uint32_t code, float unit) {
  const float f = bits_f((code & 8u) << 28 | (code & 7u) << 22);
  return f * 0x1p126f * unit;
}

// Eight values a lane.
template <int T>
EOS_DEV void dequantize(const MxDequantArgs& a) {
  const long long first = (long long)blockIdx.x * 64;
  const long long row0 = first / a.blocks;
  const uint32_t in = (uint32_t)(first - row0 * a.blocks) + threadIdx.x / 4;
  const uint32_t over = in / (uint32_t)a.blocks;
  const long long row = row0 + over;
  if (row >= a.rows) return;
  const int block = (int)(in - over * a.blocks);
  const long long b = row * a.blocks + block;
  const uint32_t c = reinterpret_cast<const uint32_t*>(a.codes)[b * 4 + (threadIdx.x & 3)];
  const uint32_t byte = a.scales[b];
  const float unit = byte == 255 ? __builtin_nanf("") : scale_value(byte);
  const int at = block * kMxBlock + (threadIdx.x & 3) * 8;
  const int left = a.k - at;
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = level(c >> (4 * i), unit);
  uint8_t* p = a.out + row * a.stride + (long long)at * size_of(T);
  uint32_t u[T == kMxF32 ? 8 : 4];
  if constexpr (T == kMxF32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = __builtin_bit_cast(uint32_t, x[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      u[i] = T == kMxF16 ? pack_f16(x[2 * i], x[2 * i + 1]) : pack_bf16(x[2 * i], x[2 * i + 1]);
  }
  if (left >= 8) {
    reinterpret_cast<v4u*>(p)[0] = v4u{u[0], u[1], u[2], u[3]};
    if constexpr (T == kMxF32) reinterpret_cast<v4u*>(p)[1] = v4u{u[4], u[5], u[6], u[7]};
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) {
        if constexpr (T == kMxF32) reinterpret_cast<uint32_t*>(p)[i] = u[i];
        else reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)(u[i / 2] >> 16 * (i % 2));
      }
  }
}

// ------------------------------------------------------------------ products

EOS_DEV v8i operand(v4u u) {
  return v8i{(int)u[0], (int)u[1], (int)u[2], (int)u[3], 0, 0, 0, 0};
}
// acc += w x^T over 128 values of K: lane l gets outputs 4 (l / 16) .. + 3 of
// w's 16 rows for row l % 16 of x.
EOS_DEV v4f mfma(v4u w, uint32_t ws, v4u x, uint32_t xs, v4f acc) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(w), operand(x), acc, 4, 4, 0,
                                                          (int)ws, 0, (int)xs);
}

// Four consecutive outputs of a row, of which the matrix has `left`.
template <int T>
EOS_DEV void store4(uint8_t* p, v4f y, int left) {
  if constexpr (T == kMxF32) {
    if (left >= 4) {
      *reinterpret_cast<v4f*>(p) = y;
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) reinterpret_cast<float*>(p)[i] = y[i];
  } else {
    const v2u u = T == kMxF16 ? v2u{pack_f16(y[0], y[1]), pack_f16(y[2], y[3])}
                              : v2u{pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3])};
    if (left >= 4) {
      *reinterpret_cast<v2u*>(p) = u;
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)(u[i / 2] >> 16 * (i % 2));
  }
}

// Four wavefronts, each a tile of 32 x 32 outputs, operands straight from memory.
template <int T>
EOS_DEV void linear(const MxLinearArgs& a) {
  constexpr int MT = 2, NT = 2;
  const int wave = threadIdx.x / 64, lane = threadIdx.x & 63;
  const long long bm = blockIdx.x / (unsigned)a.tiles_n;
  const int bn = (int)(blockIdx.x - bm * a.tiles_n);
  const long long m0 = (bm * 2 + wave / 2) * MT;
  const int n0 = (bn * 2 + wave % 2) * NT;
  const long long last_m = (a.rows - 1) / kMxTile;
  const int last_n = (a.n - 1) / kMxTile;
  const uint8_t *x[MT], *xs[MT], *w[NT], *ws[NT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const long long t = m0 + i < last_m ? m0 + i : last_m;
    x[i] = a.x.codes + t * a.x.steps * kMxTileBytes + lane * 16;
    xs[i] = a.x.scales + t * a.x.quads * kMxScaleBytes + lane * 4;
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const long long t = n0 + i < last_n ? n0 + i : last_n;
    w[i] = a.w.codes + t * a.w.steps * kMxTileBytes + lane * 16;
    ws[i] = a.w.scales + t * a.w.quads * kMxScaleBytes + lane * 4;
  }
  v4f acc[NT][MT] = {};
  for (int s = 0; s < a.x.steps; ++s) {
    v4u xv[MT], wv[NT];
    uint32_t xe[MT], we[NT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      xv[i] = *reinterpret_cast<const v4u*>(x[i] + (long long)s * kMxTileBytes);
      xe[i] = *reinterpret_cast<const uint32_t*>(xs[i] + (s / 4) * kMxScaleBytes) >> 8 * (s % 4);
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      wv[i] = *reinterpret_cast<const v4u*>(w[i] + (long long)s * kMxTileBytes);
      we[i] = *reinterpret_cast<const uint32_t*>(ws[i] + (s / 4) * kMxScaleBytes) >> 8 * (s % 4);
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < MT; ++j) acc[i][j] = mfma(wv[i], we[i], xv[j], xe[j], acc[i][j]);
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int n = (n0 + i) * kMxTile + lane / 16 * 4;
    if (n >= a.n) continue;
    v4f b = {};
    if (a.bias != nullptr) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (n + r < a.n) b[r] = a.bias[n + r];
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      const long long m = (m0 + j) * kMxTile + lane % 16;
      if (m < a.rows)
        store4<T>(a.out + m * a.out_stride + (long long)n * size_of(T), acc[i][j] + b, a.n - n);
    }
  }
}

}  // namespace

#define MX_KERNELS(NAME, T)                                                                     \
  extern "C" __global__ __launch_bounds__(256) void eos_mx_quantize_##NAME(MxQuantArgs a) {     \
    quantize<T>(a);                                                                             \
  }                                                                                             \
  extern "C" __global__ __launch_bounds__(256) void eos_mx_lay_##NAME(MxQuantArgs a) {          \
    lay<T>(a);                                                                                  \
  }                                                                                             \
  extern "C" __global__ __launch_bounds__(256) void eos_mx_dequantize_##NAME(MxDequantArgs a) { \
    dequantize<T>(a);                                                                           \
  }                                                                                             \
  extern "C" __global__ __launch_bounds__(256) void eos_mx_linear_##NAME(MxLinearArgs a) {      \
    linear<T>(a);                                                                               \
  }
MX_KERNELS(f16, kMxF16)
MX_KERNELS(bf16, kMxBf16)
MX_KERNELS(f32, kMxF32)
extern "C" __global__ __launch_bounds__(256) void eos_mx_lay_codes(MxQuantArgs a) { lay<kMxCodes>(a); }
