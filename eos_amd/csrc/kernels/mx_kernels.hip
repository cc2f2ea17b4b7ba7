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
  } else if (left > 0) {
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
// is of consecutive bytes. Bound by them: 16,384 rows of 4,096 bf16 in 35 us and
// back in 31, 170 MB each (4.9 and 5.5 TB/s; a copy reaches 4.7 to 5.2).
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

// The same into laid-out tiles: a workgroup a tile and quad, a wavefront a step.
// 8,192 rows of 8,192 bf16: 39 us, 4.4 TB/s; of a small call 3, its latency.
template <int T>
EOS_DEV void lay(const MxQuantArgs& a) {
  const MxLaid& o = a.laid;
  const int step = threadIdx.x / 64, lane = threadIdx.x & 63;
  const long long tile = blockIdx.x / (unsigned)o.quads;
  const int quad = (int)(blockIdx.x - tile * o.quads);
  uint8_t* codes = o.codes + (long long)blockIdx.x * kMxTileBytes + step * 1024;
  uint8_t* scales = o.scales + (long long)blockIdx.x * kMxScaleBytes + step;
  if constexpr (T == kMxCodes) {
    const long long row = tile * kMxTile + lane % 32;
    const int block = quad * 8 + step * 2 + lane / 32;
    v4u c = {};
    uint32_t byte = 0;
    if (row < a.rows && block < a.blocks) {
      c = *reinterpret_cast<const v4u*>(a.x + (row * a.blocks + block) * 16);
      byte = a.xs[row * a.blocks + block];
    }
    *reinterpret_cast<v4u*>(codes + lane * 16) = c;
    scales[lane * 4] = (uint8_t)byte;
  } else {
    const int at = quad * kMxQuad + step * 64 + lane % 8 * 8;
    Eight<T> e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long row = tile * kMxTile + i * 8 + lane / 8;
      e[i] = Eight<T>{};
      if (row < a.rows) e[i] = load8<T>(a.x + row * a.stride + (long long)at * size_of(T), a.k - at);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int l = lane % 8 / 4 * 32 + i * 8 + lane / 8;  // the lane that multiplies it
      uint32_t byte;
      const uint32_t c = quarter<T>(e[i], byte);
      reinterpret_cast<uint32_t*>(codes)[l * 4 + (lane & 3)] = c;
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

typedef float v16f __attribute__((ext_vector_type(16)));

EOS_DEV v8i operand(v4u u) {
  return v8i{(int)u[0], (int)u[1], (int)u[2], (int)u[3], 0, 0, 0, 0};
}
// acc += w x^T over 64 values of K: lane l gets outputs 8 g + 4 (l / 32) .. + 3
// of w's 32 rows, g = 0..3, for row l % 32 of x. S: which byte of the scales.
template <int S>
EOS_DEV v16f mfma(v4u w, uint32_t ws, v4u x, uint32_t xs, v16f acc) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(w), operand(x), acc, 4, 4, S,
                                                         (int)ws, S, (int)xs);
}
// acc += w x^T over 128 values: lane l gets outputs 4 (l / 16) .. + 3 of w's
// 16 rows for row l % 16 of x.
EOS_DEV v4f mfma16(v4u w, uint32_t ws, v4u x, uint32_t xs, v4f acc) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(w), operand(x), acc, 4, 4, 0,
                                                          (int)ws, 0, (int)xs);
}

// Four consecutive outputs of a row, of which the matrix has `left`.
EOS_DEV void store4(uint8_t* p, int type, v4f y, int left) {
  if (type == kMxF32) {
    if (left >= 4) {
      *reinterpret_cast<v4f*>(p) = y;
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) reinterpret_cast<float*>(p)[i] = y[i];
  } else {
    const v2u u = type == kMxF16 ? v2u{pack_f16(y[0], y[1]), pack_f16(y[2], y[3])}
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
// A barrier that LDS accesses are complete at, loads from memory not.
EOS_DEV void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// The tile of a workgroup: consecutive workgroups go to the 8 XCDs in turn, so
// each XCD gets a run of tiles, in columns of eight (of x) by eight, whose
// operands its L2 keeps.
EOS_DEV void place(const MxLinearArgs& a, int& bm, int& bn) {
  const unsigned total = gridDim.x, xcd = blockIdx.x % 8, q = total / 8, r = total % 8;
  const unsigned t = xcd * q + min(xcd, r) + blockIdx.x / 8;
  const unsigned column = 8u * (unsigned)a.tiles_n;
  const unsigned group = t / column, in = t - group * column;
  const unsigned high = min(8u, (unsigned)a.tiles_m - group * 8);
  bn = (int)(in / high);
  bm = (int)(group * 8 + in - bn * high);
}

// A wavefront's NF tiles of outputs of 32 rows from row m0 and output n0 on: through
// its part of LDS, so that a store writes whole lines. (One wavefront a SIMD
// issues an instruction every four cycles or five: what counts is how many these
// are.)
template <int T, int MF, int NF>
EOS_DEV void put(const MxLinearArgs& a, const v16f (&acc)[NF][MF], int j, uint8_t* mine, long long m0,
                 int n0) {
  constexpr int kSize = size_of(T), kEach = 16 / kSize;       // outputs of a store
  constexpr int kRow = NF * 32 * kSize + 16;                  // bytes of a row in LDS
  constexpr int kLanes = NF * 32 / kEach, kRows = 64 / kLanes;  // lanes of a row, rows of a store
  const int lane = threadIdx.x & 63;
  uint8_t* to = mine + lane % 32 * kRow + lane / 32 * 4 * kSize;
#pragma unroll
  for (int i = 0; i < NF; ++i)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const v4f y = {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
      store4(to + (i * 32 + 8 * g) * kSize, T, y, 4);
    }
  __builtin_amdgcn_wave_barrier();
  const uint8_t* from = mine + lane / kLanes * kRow + lane % kLanes * 16;
  const int n = n0 + lane % kLanes * kEach;
  uint8_t* p = a.out + (m0 + lane / kLanes) * a.out_stride + (long long)n * kSize;
  if (m0 + 32 <= a.rows && n0 + NF * 32 <= a.n) {
#pragma unroll 4
    for (int r = 0; r < 32; r += kRows, p += kRows * a.out_stride)
      *reinterpret_cast<v4u*>(p) = *reinterpret_cast<const v4u*>(from + r * kRow);
  } else if (n < a.n) {
#pragma unroll 1
    for (int r = 0; r < 32 && m0 + lane / kLanes + r < a.rows; r += kRows, p += kRows * a.out_stride) {
      if (n + kEach <= a.n) {
        *reinterpret_cast<v4u*>(p) = *reinterpret_cast<const v4u*>(from + r * kRow);
        continue;
      }
#pragma unroll 1
      for (int i = 0; n + i < a.n; ++i) {
        if constexpr (T == kMxF32)
          reinterpret_cast<uint32_t*>(p)[i] = reinterpret_cast<const uint32_t*>(from + r * kRow)[i];
        else
          reinterpret_cast<uint16_t*>(p)[i] = reinterpret_cast<const uint16_t*>(from + r * kRow)[i];
      }
    }
  }
  __builtin_amdgcn_wave_barrier();
}

typedef __amdgpu_buffer_rsrc_t Buffer;

// Memory from p on (uniform), as far as 32-bit offsets reach.
EOS_DEV Buffer buffer(const uint8_t* p) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, 0xffffffffu, 0x00027000);
}
EOS_DEV v4u load16(Buffer b, int lane_offset, int offset) {
  return __builtin_amdgcn_raw_buffer_load_b128(b, lane_offset, offset, 0);
}
EOS_DEV uint32_t load4(Buffer b, int lane_offset, int offset) {
  return __builtin_amdgcn_raw_buffer_load_b32(b, lane_offset, offset, 0);
}

// 16 bytes a lane from memory straight into LDS: lane i's at lds + 16 i. loads_wait
// and a barrier stand before their first use. Written out because the compiler,
// which cannot tell the two buffers apart, would wait for the builtin's before
// every read of the other.
EOS_DEV void load_lds16(v4u memory, int lane_offset, int offset, uint32_t lds) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %1, %2, %3 offen lds"
      :
      : "s"(lds), "v"(lane_offset), "s"(memory), "s"(offset)
      : "memory", "m0");
}
EOS_DEV void loads_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
EOS_DEV v4u descriptor(const uint8_t* p) {
  const uint64_t u = (uint64_t)(uintptr_t)p;
  return v4u{(uint32_t)u, (uint32_t)(u >> 32), 0xffffffffu, 0x00027000u};
}

// 2 x 2 wavefronts, each MF x NF tiles of 32 x 32 outputs. Quads of K go from
// memory into one of two LDS buffers while the other is multiplied. The order of
// the instructions is the one written: between any two matrix instructions of a
// step stand a read of an operand of the next step (the quad's last step: of the
// next quad's first) and a load.
// DIRECT: loads straight into LDS, in the quad's first step and the one before it,
// for which the barrier of the quad before has made room; they have two steps to
// arrive. Otherwise through registers, which are stored in the first two steps and
// at once loaded again, a quad ahead; a load that comes back so takes 29 clocks of
// the matrix unit's. The 256 tile's steps are long enough for the former (8,192^3
// through registers in the compiler's order 298 us, in the written one 263, straight
// into LDS 230), those of 64 and 128 not (512 by 4,096 x 4,096 from HBM 13.7 us
// direct, 12.3 through registers; 1,024 17.1 and 15.1).
//
// Tiles of 32 x 32 x 64: on values as they come these reach 6.5 PFLOP/s of the
// card, 16 x 16 x 128 5.6 (on zeros 9.5 and 6.9: it is the power that they draw).
// MF = NF = 4: a wavefront's 128 x 128 outputs read 16 KB of LDS for 128 values of
// K, half of what 64 x 64 read for as many products. 8,192^3: 230 to 241 us by the
// card, 4.6 to 4.8 PFLOP/s. A quad is 2,480 clocks, 2,048 of them matrix
// instructions; the clock is 2.4 GHz for one workgroup, 1.45 when all multiply (2.2
// on zeros): power. 7 us of each of four turns are the first loads and the stores.
template <int MF, int NF>
struct Product {
  static constexpr int TM = 2 * MF, TN = 2 * NF, TILES = TM + TN, SLOTS = MF + NF;
  static constexpr bool DIRECT = MF * NF >= 16;
  v4u lds_x, lds_w;  // descriptors of the codes
  Buffer codes_x, codes_w, scales_x, scales_w;
  int at[TILES], scale_at[SLOTS];  // offsets of tiles (x, then w), of the wavefront's scales
  v4u stage[TILES];
  v4u xv[2][MF], wv[2][NF];
  uint32_t sc[SLOTS], next[SLOTS];  // scales of x, then w
  v16f acc[NF][MF];

  // Direct scales that have arrived: their registers are taken here, where all
  // loads are waited for, or the compiler would wait at their use, for later loads
  // too.
  EOS_DEV void scales_here() {
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) asm volatile("" : "+v"(next[i]));
  }
  // The thread's 16 bytes of tile i of quad q to a register, or to the buffer whose
  // part for the wavefront begins at `lds`.
  EOS_DEV void fetch(int i, int q) {
    stage[i] = load16(i < TM ? codes_x : codes_w, threadIdx.x * 16, at[i] + q * kMxTileBytes);
  }
  EOS_DEV void fetch_lds(int i, int q, uint32_t lds) {
    load_lds16(i < TM ? lds_x : lds_w, threadIdx.x * 16, at[i] + q * kMxTileBytes, lds + i * kMxTileBytes);
  }
  EOS_DEV void fetch_scales(int i, int q) {
    next[i] = load4(i < MF ? scales_x : scales_w, (threadIdx.x & 63) * 4,
                    scale_at[i] + q * kMxScaleBytes);
  }
  // Operand k of a step in the order in which the step needs them.
  EOS_DEV void read(int to, int k, const v4u* x, const v4u* w, int step) {
    if (k == 0) wv[to][0] = w[step * 64];
    else if (k <= MF) xv[to][k - 1] = x[(k - 1) * 256 + step * 64];
    else wv[to][k - MF] = w[(k - MF) * 256 + step * 64];
  }
  // x, w: where the next step's operands are read, from its step `step`; to: the
  // buffer that is loaded or stored.
  template <int S>
  EOS_DEV void step(const v4u* x, const v4u* w, int step, v4u* to, uint32_t to_lds, int q, int last) {
#pragma unroll
    for (int k = 0; k < SLOTS; ++k) {
      read((S + 1) & 1, k, x, w, step);
      if constexpr (DIRECT) {
        if constexpr (S == 3) fetch_lds(k, min(q + 2, last), to_lds);
        if constexpr (S == 0) fetch_lds(SLOTS + k, min(q + 1, last), to_lds);
      } else if constexpr (S < 2) {
        to[(S * SLOTS + k) * 256 + threadIdx.x] = stage[S * SLOTS + k];
        fetch(S * SLOTS + k, min(q + 2, last));
      }
      if constexpr (S == 0) fetch_scales(k, min(q + 1, last));
#pragma unroll
      for (int m = k * MF * NF / SLOTS; m < (k + 1) * MF * NF / SLOTS; ++m)
        acc[m / MF][m % MF] = mfma<S>(wv[S & 1][m / MF], sc[MF + m / MF], xv[S & 1][m % MF],
                                      sc[m % MF], acc[m / MF][m % MF]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};

template <int T, int MF, int NF>
EOS_DEV void product(const MxLinearArgs& a) {
  typedef Product<MF, NF> P;
  constexpr int TM = P::TM, TN = P::TN, TILES = P::TILES;
  __shared__ v4u lds[2][TILES * 256];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x & 63;
  const int wm = wave / 2 * MF, wn = wave % 2 * NF;
  int bm, bn;
  place(a, bm, bn);
  // (offsets within a workgroup's tiles stay below 2^31: 8 tiles of 2^16 quads)
  const int last_m = (int)((a.rows - 1) / kMxTile) - bm * TM, last_n = (a.n - 1) / kMxTile - bn * TN;
  const int quads = a.w.quads, last = quads - 1;
  P p;
  const uint8_t* codes_x = a.x.codes + (long long)bm * TM * quads * kMxTileBytes;
  const uint8_t* codes_w = a.w.codes + (long long)bn * TN * quads * kMxTileBytes;
  p.lds_x = descriptor(codes_x);
  p.lds_w = descriptor(codes_w);
  p.codes_x = buffer(codes_x);
  p.codes_w = buffer(codes_w);
  p.scales_x = buffer(a.x.scales + (long long)bm * TM * quads * kMxScaleBytes);
  p.scales_w = buffer(a.w.scales + (long long)bn * TN * quads * kMxScaleBytes);
#pragma unroll
  for (int i = 0; i < TILES; ++i)
    p.at[i] = (i < TM ? min(i, last_m) : min(i - TM, last_n)) * quads * kMxTileBytes;
#pragma unroll
  for (int i = 0; i < MF + NF; ++i)
    p.scale_at[i] = (i < MF ? min(wm + i, last_m) : min(wn + i - MF, last_n)) * quads * kMxScaleBytes;
#pragma unroll
  for (int i = 0; i < NF; ++i) {
    v16f b = {};  // the sums begin with the bias
    if (a.bias != nullptr) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        b[r] = a.bias[min((bn * TN + wn + i) * kMxTile + r / 4 * 8 + lane / 32 * 4 + r % 4, a.n - 1)];
    }
#pragma unroll
    for (int j = 0; j < MF; ++j) p.acc[i][j] = b;
  }
  // (a wavefront's part of a tile: 1024 bytes)
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)lds[0] + wave * 1024;
  constexpr uint32_t kBuffer = sizeof(lds[0]);
#pragma unroll
  for (int i = 0; i < MF + NF; ++i) p.fetch_scales(i, 0);
  if constexpr (P::DIRECT) {
#pragma unroll
    for (int i = 0; i < TILES; ++i) p.fetch_lds(i, 0, lds0);
    loads_wait();
    p.scales_here();
#pragma unroll
    for (int i = 0; i < TILES / 2; ++i) p.fetch_lds(i, min(1, last), lds0 + kBuffer);
  } else {
#pragma unroll
    for (int i = 0; i < TILES; ++i) p.fetch(i, 0);
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
      lds[0][i * 256 + threadIdx.x] = p.stage[i];
      p.fetch(i, min(1, last));
    }
  }
#pragma unroll
  for (int i = 0; i < MF + NF; ++i) p.sc[i] = p.next[i];
  lds_barrier();
  const int x0 = wm * 256 + lane, w0 = (TM + wn) * 256 + lane;
#pragma unroll
  for (int k = 0; k < MF + NF; ++k) p.read(0, k, lds[0] + x0, lds[0] + w0, 0);
  for (int q = 0; q < quads; ++q) {
    v4u *now = lds[q & 1], *then = lds[(q + 1) & 1];
    const uint32_t lds_now = lds0 + (q & 1) * kBuffer, lds_then = lds0 + ((q + 1) & 1) * kBuffer;
    p.template step<0>(now + x0, now + w0, 1, then, lds_then, q, last);
    p.template step<1>(now + x0, now + w0, 2, then, 0, q, last);
    p.template step<2>(now + x0, now + w0, 3, nullptr, 0, q, last);
    if constexpr (P::DIRECT) {
      loads_wait();
      p.scales_here();
    }
    lds_barrier();
    p.template step<3>(then + x0, then + w0, 0, nullptr, lds_now, q, last);
#pragma unroll
    for (int i = 0; i < MF + NF; ++i) p.sc[i] = p.next[i];
  }
  if constexpr (P::DIRECT) loads_wait();  // the outputs take the buffers' place
  lds_barrier();
  const long long m0 = (long long)(bm * TM + wm) * kMxTile;
  const int n0 = (bn * TN + wn) * kMxTile;
  uint8_t* mine = reinterpret_cast<uint8_t*>(lds) + wave * (sizeof(lds) / 4);
#pragma unroll
  for (int j = 0; j < MF; ++j) put<T, MF, NF>(a, p.acc, j, mine, m0 + j * 32, n0);
}

// ------------------------------------------------------------------ few rows

constexpr int kMxRowsLaid = 4;  // x laid out by an earlier kernel

// A lane's block as an operand.
struct Piece {
  v4u c;
  uint32_t byte;
};

// A lane's block of 16 laid-out rows (tile16 counts those) in 128 values of K.
EOS_DEV Piece load_laid(const MxLaid& m, int tile16, int op) {
  const int lane = threadIdx.x & 63;
  const int at = (lane & 16) * 2 + (tile16 & 1) * 16 + lane % 16;  // its lane in the layout
  const int step = op % 2 * 2 + lane / 32;
  const long long t = (long long)(tile16 >> 1) * m.quads + op / 2;
  Piece p;
  p.c = *reinterpret_cast<const v4u*>(m.codes + t * kMxTileBytes + step * 1024 + at * 16);
  p.byte = reinterpret_cast<const uint32_t*>(m.scales + t * kMxScaleBytes)[at] >> 8 * step;
  return p;
}

// 16 rows of x on their way to operands: a wavefront's own part of LDS, codes and
// scales of U times 128 values. Offsets in words, so that a row's 64 stores (four
// blocks of four words, U of them) hit 64 banks.
template <int U>
struct Rows16 {
  uint32_t codes[U * 272];
  uint32_t scales[U * 68];
  EOS_DEV static int code_at(int u, int block, int row) { return u * 272 + block * 68 + row * 4; }
  EOS_DEV static int scale_at(int u, int block, int row) { return u * 68 + block * 16 + row; }
};

// Quantises the rows' values first * 128 .. + 127, and u * 8 * 128 further on.
// Up to four rows a row at a time, eight values a lane as they lie in memory;
// more of them a block a lane, four rows at a time, which loads parts of lines
// but takes 0.6 of the instructions (16,384 values by 4,096 weights: one row 9.2
// us against 11.8; 4,096 by 6,144: 16 rows 9.2 against 8.2; from HBM).
template <int X, bool FOUR, int U>
EOS_DEV void quantize_rows(const MxLinearArgs& a, Rows16<U>& to, int first) {
  static_assert(U == 4, "64 lanes take four times 16 lanes' or 16 blocks");
  const int lane = threadIdx.x & 63, rows = (int)a.rows;
  if constexpr (FOUR) {
    const int u = lane / 16, block = lane % 16 / 4;
    const int at = (first + u * 8) * 128 + lane % 16 * 8;
    const uint8_t* from = a.rows_x + (long long)at * size_of(X);
    Eight<X> e[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      e[r] = Eight<X>{};
      if (r < rows) e[r] = load8<X>(from + r * a.x_stride, a.k - at);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (r >= rows) break;
      uint32_t byte;
      const uint32_t c = quarter<X>(e[r], byte);
      to.codes[to.code_at(u, block, r) + (lane & 3)] = c;
      if ((lane & 3) == 0) to.scales[to.scale_at(u, block, r)] = byte;
    }
  } else {
    constexpr int kBatch = X == kMxF32 ? 1 : 2;  // times four rows whose loads are in flight
    const int u = lane % 16 / 4, block = lane % 4;
    const int at = (first + u * 8) * 128 + block * kMxBlock, left = a.k - at;
    const uint8_t* from = a.rows_x + (long long)at * size_of(X);
    for (int r0 = lane / 16; r0 - lane / 16 < rows; r0 += 4 * kBatch) {
      Eight<X> e[kBatch][4];
#pragma unroll
      for (int r = 0; r < kBatch; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          e[r][i] = load8<X>(from + (r0 + 4 * r) * a.x_stride + i * 8 * size_of(X),
                             r0 + 4 * r < rows ? left - i * 8 : 0);
#pragma unroll
      for (int r = 0; r < kBatch; ++r) {
        if (r0 + 4 * r >= rows) break;
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) m = max(m, most8<X>(e[r][i]));
        const uint32_t byte = scale_byte<X>(m);
        v4u c;
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = byte == 255 ? 0u : codes8<X>(e[r][i], scale_value(byte));
        *reinterpret_cast<v4u*>(&to.codes[to.code_at(u, block, r0 + 4 * r)]) = c;
        to.scales[to.scale_at(u, block, r0 + 4 * r)] = byte;
      }
    }
  }
}

// Up to 16 MT rows of x (16, where they are not laid out) by 16 NT rows of w a
// workgroup: its eight wavefronts take 128 values of K in turn, U at a time, so
// that the weights, read once, arrive in long runs; their sums meet in LDS, in
// the wavefronts' order. Bound by the weights: 16,384 x 16,384 by one row in 26
// us, 5.5 TB/s; 48 rows by 4,096 x 16,384 11.1 from HBM, 8.6 (4.4 TB/s) where the
// weights are still on the chip; one by 4,096 x 6,144 5.5 and 4.4, a chain of launch,
// loads, sums. 16 rows by it 8.2; as codes, without their quantisation, 6.0.
template <int X, bool FOUR, int MT, int NT, int U>
EOS_DEV void few(const MxLinearArgs& a) {
  constexpr bool kRows = X < kMxCodes;
  constexpr size_t kSums = 8 * MT * NT * 64 * sizeof(v4f), kRowBytes = kRows ? 8 * sizeof(Rows16<U>) : 0;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kSums > kRowBytes ? kSums : kRowBytes];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x & 63;
  const int n0 = blockIdx.x * NT, last_n = (a.n - 1) / 16, ops = a.w.quads * 2;
  Rows16<U>& rows = reinterpret_cast<Rows16<U>*>(lds)[kRows ? wave : 0];
  if constexpr (kRows) {  // rows that x lacks stay zero
    uint32_t* z = reinterpret_cast<uint32_t*>(&rows);
    for (int i = lane; i < (int)(sizeof(rows) / 4); i += 64) z[i] = 0;
  }
  v4f acc[NT][MT] = {};
  for (int first = wave; first < ops; first += 8 * U) {
    Piece w[U][NT];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < NT; ++i) w[u][i] = load_laid(a.w, min(n0 + i, last_n), min(first + 8 * u, ops - 1));
    Piece x[U][MT];
    if constexpr (kRows) {
      quantize_rows<X, FOUR, U>(a, rows, first);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int op = min(first + 8 * u, ops - 1);
        if constexpr (X == kMxRowsLaid) {
#pragma unroll
          for (int j = 0; j < MT; ++j) x[u][j] = load_laid(a.x, j, op);
        } else {
          const int row = lane % 16, block = op * 4 + lane / 16;
          x[u][0] = Piece{};
          if (row < a.rows && block < a.x.blocks) {
            const long long b = (long long)row * a.x.blocks + block;
            x[u][0].c = *reinterpret_cast<const v4u*>(a.rows_x + b * 16);
            x[u][0].byte = a.scales_x[b];
          }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (first + 8 * u >= ops) break;
      if constexpr (kRows) {
        x[u][0].c = *reinterpret_cast<const v4u*>(&rows.codes[rows.code_at(u, lane / 16, lane % 16)]);
        x[u][0].byte = rows.scales[rows.scale_at(u, lane / 16, lane % 16)];
      }
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int i = 0; i < NT; ++i)
          acc[i][j] = mfma16(w[u][i].c, w[u][i].byte, x[u][j].c, x[u][j].byte, acc[i][j]);
    }
  }
  if constexpr (kRows) __syncthreads();  // the sums take the rows' place
  v4f(*sums)[MT * NT * 64] = reinterpret_cast<v4f(*)[MT * NT * 64]>(lds);
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) sums[wave][(i * MT + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  for (int e = threadIdx.x; e < MT * NT * 64; e += 512) {
    const int tile = e / 64, l = e % 64;
    const int m = tile % MT * 16 + l % 16, n = (n0 + tile / MT) * 16 + l / 16 * 4;
    if (m >= a.rows || n >= a.n) continue;
    v4f y = sums[0][e];
#pragma unroll
    for (int v = 1; v < 8; ++v) y += sums[v][e];
    if (a.bias != nullptr) {
#pragma unroll
      for (int r = 0; r < 4; ++r) y[r] += a.bias[min(n + r, a.n - 1)];
    }
    const int size = a.out_type == kMxF32 ? 4 : 2;
    store4(a.out + m * a.out_stride + (long long)n * size, a.out_type, y, a.n - n);
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
  }
MX_KERNELS(f16, kMxF16)
MX_KERNELS(bf16, kMxBf16)
MX_KERNELS(f32, kMxF32)
extern "C" __global__ __launch_bounds__(256) void eos_mx_lay_codes(MxQuantArgs a) { lay<kMxCodes>(a); }

#define MX_PRODUCT(NAME, T, MF, NF, WAVES)                                                         \
  extern "C" __global__ __launch_bounds__(256, WAVES) void eos_mx_product_##NAME(MxLinearArgs a) { \
    product<T, MF, NF>(a);                                                                         \
  }
#define MX_PRODUCTS(TYPE, T)          \
  MX_PRODUCT(64_##TYPE, T, 1, 1, 2)   \
  MX_PRODUCT(128_##TYPE, T, 2, 2, 2)  \
  MX_PRODUCT(256_##TYPE, T, 4, 4, 1)
MX_PRODUCTS(f16, kMxF16)
MX_PRODUCTS(bf16, kMxBf16)
MX_PRODUCTS(f32, kMxF32)

#define MX_FEW(NAME, X, FOUR, MT, NT, U)                                                       \
  extern "C" __global__ __launch_bounds__(512) void eos_mx_few_##NAME##_##NT(MxLinearArgs a) { \
    few<X, FOUR, MT, NT, U>(a);                                                                \
  }
#define MX_FEW_ROWS(NAME, X)               \
  MX_FEW(NAME##_4, X, true, 1, 1, 4)       \
  MX_FEW(NAME##_4, X, true, 1, 2, 4)       \
  MX_FEW(NAME##_16, X, false, 1, 1, 4)     \
  MX_FEW(NAME##_16, X, false, 1, 2, 4)     \
  MX_FEW(NAME##_16, X, false, 1, 4, 4)
MX_FEW_ROWS(f16, kMxF16)
MX_FEW_ROWS(bf16, kMxBf16)
MX_FEW_ROWS(f32, kMxF32)
#define MX_FEW_N(NAME, X, MT, U2)         \
  MX_FEW(NAME, X, false, MT, 1, 4)        \
  MX_FEW(NAME, X, false, MT, 2, U2)
MX_FEW_N(codes_16, kMxCodes, 1, 4)
MX_FEW_N(laid_32, kMxRowsLaid, 2, 4)
MX_FEW_N(laid_48, kMxRowsLaid, 3, 2)
MX_FEW_N(laid_64, kMxRowsLaid, 4, 2)
