// What a decoding step does around the paged cache, on gfx950: rotary
// positions of its queries and keys, and the page tables, row ranges and slots
// of its batch from the lengths of its requests.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "step_args.h"

#define EOS_DEV __device__ __forceinline__

namespace {

typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------- rotary positions

constexpr int size_of(int type) { return type == kRotF32 ? 4 : 2; }

EOS_DEV float to_f32(uint16_t u, int type) {
  return type == kRotF16 ? (float)__builtin_bit_cast(_Float16, u)
                         : __builtin_bit_cast(float, (uint32_t)u << 16);
}
EOS_DEV uint32_t from_f32(float f, int type) {
  return type == kRotF16 ? __builtin_bit_cast(uint16_t, (_Float16)f)
                         : __builtin_bit_cast(uint16_t, (__bf16)f);
}

template <int T>
EOS_DEV void load8(const uint8_t* p, float (&x)[8]) {
  if constexpr (T == kRotF32) {
    const v4f a = reinterpret_cast<const v4f*>(p)[0], b = reinterpret_cast<const v4f*>(p)[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
  } else {
    const v4u u = *reinterpret_cast<const v4u*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = to_f32((uint16_t)u[i], T);
      x[2 * i + 1] = to_f32((uint16_t)(u[i] >> 16), T);
    }
  }
}
template <int T>
EOS_DEV void store8(uint8_t* p, const float (&x)[8]) {
  if constexpr (T == kRotF32) {
    reinterpret_cast<v4f*>(p)[0] = v4f{x[0], x[1], x[2], x[3]};
    reinterpret_cast<v4f*>(p)[1] = v4f{x[4], x[5], x[6], x[7]};
  } else {
    v4u u;
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = from_f32(x[2 * i], T) | from_f32(x[2 * i + 1], T) << 16;
    *reinterpret_cast<v4u*>(p) = u;
  }
}
template <int T>
EOS_DEV float load1(const uint8_t* p, int i) {
  if constexpr (T == kRotF32) return reinterpret_cast<const float*>(p)[i];
  else return to_f32(reinterpret_cast<const uint16_t*>(p)[i], T);
}
template <int T>
EOS_DEV void store1(uint8_t* p, int i, float x) {
  if constexpr (T == kRotF32) reinterpret_cast<float*>(p)[i] = x;
  else reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)from_f32(x, T);
}

// A row's position in its sequence, by a whole wavefront; -1: not a row of the
// batch, or padding.
EOS_DEV int row_position(const RotArgs& a, long long row) {
  if (row >= a.rows) return -1;
  if (a.positions != nullptr) return a.positions[row];
  if (a.offsets == nullptr) return a.lengths[row] - 1;
  // How many sequences end at or before the row: 64 probes a turn.
  const int lane = threadIdx.x & 63;
  const int32_t* ends = a.offsets + 1;
  int base = 0, size = a.batch;
  while (size > 0) {
    const int step = (size + 63) / 64;
    const bool before = lane * (long long)step < size && ends[base + lane * step] <= row;
    const int c = __popcll(__ballot(before));
    if (c == 0) break;
    const int skip = (c - 1) * step + 1;
    base += skip;
    size = min(step - 1, size - skip);
  }
  if (base >= a.batch) return -1;
  const int lo = a.offsets[base], hi = ends[base];
  if (lo < 0 || row < lo || row >= hi || hi > a.rows) return -1;
  const long long pos = (long long)a.lengths[base] - hi + row;
  return pos < 0 || pos > INT32_MAX ? -1 : (int)pos;
}

// Cosine and sine of 2 pi p f for a frequency in turns a position: the product
// and its distance from whole turns in f64 (2^-52 of p f), the functions in f32.
EOS_DEV v2f turn(const RotArgs& a, int pos, int i) {
  const double t = (double)pos * a.turns[i];
  const float r = 2.0f * (float)(t - rint(t));
  float s, c;
  sincospif(r, &s, &c);
  return v2f{c * a.factor, s * a.factor * a.sign};
}

// A few rows a workgroup: their positions, then the cosines and sines that all
// heads of a row share, then the heads, eight (halves: twice eight) values a lane.
template <int T, int LAYOUT, bool WIDE>
EOS_DEV void rotate(const RotArgs& a) {
  __shared__ int pos[kRotRows];
  __shared__ __attribute__((aligned(16))) v2f cs[kRotAngles * 2];
  const int half = a.rotary_dim / 2;
  const long long row0 = (long long)blockIdx.x * a.each;
  for (int r = threadIdx.x / 64; r < a.each; r += 4) {
    const int p = row_position(a, row0 + r);
    if ((threadIdx.x & 63) == 0) pos[r] = p;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.each * half; i += 256) {
    const int r = i / half;
    if (pos[r] >= 0) cs[i] = turn(a, pos[r], i - r * half);
  }
  __syncthreads();
  const int lane = threadIdx.x & ((1 << a.lanes_shift) - 1);
  const int heads = a.heads + a.kv_heads, step = 256 >> a.lanes_shift;
  for (int r = 0; r < a.each; ++r) {
    if (pos[r] < 0) continue;
    const v2f* turns = cs + r * half;
    for (int h = threadIdx.x >> a.lanes_shift; h < heads; h += step) {
      const bool key = h >= a.heads;
      const long long row = row0 + r;
      const long long at = (long long)(key ? h - a.heads : h) * a.head_dim * size_of(T);
      const uint8_t* x = (key ? a.k + row * a.k_stride : a.q + row * a.q_stride) + at;
      uint8_t* y = (key ? a.k_out + row * a.k_out_stride : a.q_out + row * a.q_out_stride) + at;
      if constexpr (WIDE && LAYOUT == kRotHalves) {
        if (lane < half / 8) {
          float u[8], v[8];
          load8<T>(x + lane * 8 * size_of(T), u);
          load8<T>(x + (half + lane * 8) * size_of(T), v);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const v2f t = turns[lane * 8 + i];
            const float p = u[i] * t[0] - v[i] * t[1];
            v[i] = u[i] * t[1] + v[i] * t[0];
            u[i] = p;
          }
          store8<T>(y + lane * 8 * size_of(T), u);
          store8<T>(y + (half + lane * 8) * size_of(T), v);
        } else {
          const int i = a.rotary_dim + (lane - half / 8) * 8;
          if (i < a.head_dim && x != y) {
            float u[8];
            load8<T>(x + i * size_of(T), u);
            store8<T>(y + i * size_of(T), u);
          }
        }
      } else if constexpr (WIDE) {
        const int i = lane * 8;
        if (i < a.rotary_dim) {
          float u[8];
          load8<T>(x + i * size_of(T), u);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const v2f t = turns[lane * 4 + j];
            const float p = u[2 * j] * t[0] - u[2 * j + 1] * t[1];
            u[2 * j + 1] = u[2 * j] * t[1] + u[2 * j + 1] * t[0];
            u[2 * j] = p;
          }
          store8<T>(y + i * size_of(T), u);
        } else if (i < a.head_dim && x != y) {
          float u[8];
          load8<T>(x + i * size_of(T), u);
          store8<T>(y + i * size_of(T), u);
        }
      } else {
        for (int i = lane; i < half; i += 1 << a.lanes_shift) {
          const int i0 = LAYOUT == kRotPairs ? 2 * i : i, i1 = LAYOUT == kRotPairs ? 2 * i + 1 : i + half;
          const v2f t = turns[i];
          const float u = load1<T>(x, i0), v = load1<T>(x, i1);
          store1<T>(y, i0, u * t[0] - v * t[1]);
          store1<T>(y, i1, u * t[1] + v * t[0]);
        }
        if (x != y)
          for (int i = a.rotary_dim + lane; i < a.head_dim; i += 1 << a.lanes_shift)
            store1<T>(y, i, load1<T>(x, i));
      }
    }
  }
}

// --------------------------------------------------------------- page tables

constexpr int kThreads = 1024;
constexpr int kEach = kPagerSlots / kThreads;  // slots of a thread

// Sum over the threads in front of this one, and of all.
EOS_DEV long long before(long long x, long long* sums, long long& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x / 64;
  long long upto = x;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const long long y = __shfl_up(upto, d);
    if (lane >= d) upto += y;
  }
  __syncthreads();
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  long long base = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    if (w < wave) base += sums[w];
    total += sums[w];
  }
  return base + upto - x;
}

EOS_DEV long long room_of(const PagerArgs& a) {
  const long long room = (long long)a.stride << a.page_shift;
  return room < 1 << 30 ? room : 1 << 30;
}
EOS_DEV int pages_of(int tokens, int shift) {
  return (int)(((long long)tokens + (1 << shift) - 1) >> shift);
}
EOS_DEV int free_pages(const PagerArgs& a, int& bad) {
  const int count = *a.free_count;
  if (count >= 0 && count <= a.pages) return count;
  bad |= kPagerBadNumber;
  return count < 0 ? 0 : (int)a.pages;
}

// True in every thread of the workgroup that is done last: all others have
// read the state that it is about to write.
EOS_DEV bool last_one(const PagerArgs& a, int* flag) {
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    *flag = atomicAdd(&a.state[1], 1) == (int)gridDim.x - 1;
  }
  __syncthreads();
  return *flag != 0;
}

// Every workgroup sums the requests of all slots up by itself (16 bytes a slot
// from the L2, no second launch), keeps the batch's ranges in LDS and fills its
// share of rows and table entries; the last one brings lengths and stack up to date.
EOS_DEV void extend(const PagerArgs& a) {
  extern __shared__ int lds[];
  __shared__ long long sums[kThreads / 64];
  __shared__ int flag;
  int* row_of = lds;                 // [batch + 1] first row
  int* len_of = row_of + a.slots + 1;  // [batch] tokens before, -1: refused
  int* page_of = len_of + a.slots;     // [batch] first new page's place below the stack's top
  int* slot_of = page_of + a.slots;    // [batch]
  const long long room = room_of(a);
  int bad = 0;
  const int count = free_pages(a, bad);
  int len[kEach], fresh[kEach], need[kEach];
  long long mine = 0;  // rows << 13 | requests
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int s = threadIdx.x * kEach + i;
    len[i] = fresh[i] = 0;
    if (s < a.slots) {
      fresh[i] = a.ask[s];
      len[i] = a.lengths[s];
      if (fresh[i] < 0) {
        bad |= kPagerBadNumber;
        fresh[i] = 0;
      }
    }
    mine += fresh[i] > 0 ? ((long long)fresh[i] << 13) + 1 : 0;
  }
  long long all;
  long long at = before(mine, sums, all);
  const int batch = (int)(all & 8191);
  const long long rows = all >> 13;
  // A request has room if its table row holds it and its rows are the caller's.
  long long want = 0, row = at >> 13;
  bool ok[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    need[i] = 0;
    ok[i] = false;
    if (fresh[i] > 0) {
      row += fresh[i];
      if (len[i] < 0 || len[i] > room || row > a.rows) bad |= kPagerBadNumber;
      else if (len[i] + (long long)fresh[i] > room) bad |= kPagerNoRoom;
      else {
        ok[i] = true;
        need[i] = pages_of(len[i] + fresh[i], a.page_shift) - pages_of(len[i], a.page_shift);
      }
    }
    want += need[i];
  }
  long long asked;
  long long page = before(want, sums, asked);
  // Pages go to slots in order until one asks for more than there are.
  long long given = 0;
  int j = (int)(at & 8191);
  row = at >> 13;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    if (ok[i] && need[i] > 0 && page + need[i] > count) {
      ok[i] = false;
      bad |= kPagerNoPages;
    }
    if (fresh[i] > 0) {
      const int s = threadIdx.x * kEach + i;
      row_of[j] = (int)min(row, a.rows);
      len_of[j] = ok[i] ? len[i] : -1;
      page_of[j] = (int)min(page, (long long)count);
      slot_of[j] = s;
      if (blockIdx.x == 0) {
        a.b_slots[j] = s;
        a.b_lengths[j] = ok[i] ? len[i] + fresh[i] : 0;
        a.b_offsets[j] = row_of[j];
      }
      row += fresh[i];
      ++j;
    }
    page += need[i];
    if (ok[i] && need[i] > 0) given = page;
  }
  if (threadIdx.x == 0) {
    row_of[batch] = (int)min(rows, a.rows);
    if (blockIdx.x == 0) a.b_offsets[batch] = row_of[batch];
  }
  __syncthreads();
  // Rows: their positions and slots.
  const int upto = row_of[batch];
  for (long long r = (long long)blockIdx.x * kThreads + threadIdx.x; r < upto;
       r += (long long)gridDim.x * kThreads) {
    int lo = 0, hi = batch - 1;  // the request whose range holds it
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (row_of[mid] <= r) lo = mid;
      else hi = mid - 1;
    }
    int p = -1;
    long long place = -1;
    if (len_of[lo] >= 0) {
      p = len_of[lo] + (int)(r - row_of[lo]);
      const int i = p >> a.page_shift, held = pages_of(len_of[lo], a.page_shift);
      const int id = i < held ? a.table[(long long)slot_of[lo] * a.stride + i]
                              : a.free_list[count - 1 - (page_of[lo] + i - held)];
      place = ((long long)id << a.page_shift) + (p & ((1 << a.page_shift) - 1));
    }
    if (a.positions != nullptr) a.positions[r] = p;
    if (a.slot_map != nullptr) a.slot_map[r] = place;
  }
  // Table rows, by wavefronts: what a slot has, then its new pages.
  const int segments = (a.stride + kPagerSegment - 1) / kPagerSegment;
  const long long units = (long long)batch * segments;
  for (long long u = (long long)blockIdx.x * (kThreads / 64) + threadIdx.x / 64; u < units;
       u += (long long)gridDim.x * (kThreads / 64)) {
    const int b = (int)(u / segments), first = (int)(u - (long long)b * segments) * kPagerSegment;
    if (len_of[b] < 0) continue;
    const int tokens = len_of[b] + row_of[b + 1] - row_of[b];
    const int held = pages_of(len_of[b], a.page_shift), end = pages_of(tokens, a.page_shift);
    int32_t* t = a.table + (long long)slot_of[b] * a.stride;
    for (int i = first + (threadIdx.x & 63); i < min(end, first + kPagerSegment); i += 64) {
      int id;
      if (i < held) {
        id = t[i];
      } else {
        id = a.free_list[count - 1 - (page_of[b] + i - held)];
        t[i] = id;
      }
      if (a.b_table != nullptr) a.b_table[(long long)b * a.stride + i] = id;
    }
  }
  if (blockIdx.x == 0 && bad != 0) atomicOr(&a.state[0], bad);
  if (!last_one(a, &flag)) return;
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    if (ok[i]) a.lengths[threadIdx.x * kEach + i] = len[i] + fresh[i];
  // The last granted request's end is what the stack has given.
  __shared__ int taken;
  if (threadIdx.x == 0) taken = 0;
  __syncthreads();
  if (given > 0) atomicMax(&taken, (int)given);
  __syncthreads();
  if (threadIdx.x == 0) {
    *a.free_count = count - taken;
    a.state[1] = 0;
  }
}

// Pages behind the tokens to keep go back onto the stack, the last slot's last
// page first: extends undone leave it as it was.
EOS_DEV void trim(const PagerArgs& a) {
  extern __shared__ int lds[];
  __shared__ long long sums[kThreads / 64];
  __shared__ int flag;
  int* page_of = lds;                // [slots] pages in front of a slot's
  int* gone_of = page_of + a.slots;  // [slots] its pages
  int* left_of = gone_of + a.slots;  // [slots] pages that stay
  const long long room = room_of(a);
  int bad = 0;
  const int count = free_pages(a, bad);
  int keep[kEach], gone[kEach];
  long long mine = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int s = threadIdx.x * kEach + i;
    keep[i] = -1;
    gone[i] = 0;
    if (s < a.slots) {
      const int len = a.lengths[s], k = a.ask[s];
      if (len < 0 || len > room) {
        bad |= kPagerBadNumber;
      } else if (k >= 0 && k < len) {
        keep[i] = k;
        left_of[s] = pages_of(k, a.page_shift);
        gone[i] = pages_of(len, a.page_shift) - left_of[s];
      }
      gone_of[s] = gone[i];
    }
    mine += gone[i];
  }
  long long total;
  long long at = before(mine, sums, total);
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int s = threadIdx.x * kEach + i;
    if (s < a.slots) page_of[s] = (int)min(at, (long long)INT32_MAX);
    at += gone[i];
  }
  if (count + total > a.pages) bad |= kPagerBadNumber;
  __syncthreads();
  const int segments = (a.stride + kPagerSegment - 1) / kPagerSegment;
  const long long units = (long long)a.slots * segments;
  for (long long u = (long long)blockIdx.x * (kThreads / 64) + threadIdx.x / 64; u < units;
       u += (long long)gridDim.x * (kThreads / 64)) {
    const int s = (int)(u / segments), first = (int)(u - (long long)s * segments) * kPagerSegment;
    if (first >= gone_of[s]) continue;
    int32_t* t = a.table + (long long)s * a.stride + left_of[s];
    for (int i = first + (threadIdx.x & 63); i < min(gone_of[s], first + kPagerSegment); i += 64) {
      const long long to = count + total - 1 - (page_of[s] + (long long)i);
      if (to >= 0 && to < a.pages) a.free_list[to] = t[i];
      t[i] = -1;
    }
  }
  if (blockIdx.x == 0 && bad != 0) atomicOr(&a.state[0], bad);
  if (!last_one(a, &flag)) return;
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    if (keep[i] >= 0) a.lengths[threadIdx.x * kEach + i] = keep[i];
  if (threadIdx.x == 0) {
    *a.free_count = (int)min(count + total, a.pages);
    a.state[1] = 0;
  }
}

}  // namespace

#define ROT_KERNELS(NAME, T)                                                                      \
  extern "C" __global__ __launch_bounds__(256) void eos_rot_pairs_##NAME(RotArgs a) {             \
    rotate<T, kRotPairs, true>(a);                                                                \
  }                                                                                               \
  extern "C" __global__ __launch_bounds__(256) void eos_rot_halves_##NAME(RotArgs a) {            \
    rotate<T, kRotHalves, true>(a);                                                               \
  }                                                                                               \
  extern "C" __global__ __launch_bounds__(256) void eos_rot_pairs_odd_##NAME(RotArgs a) {         \
    rotate<T, kRotPairs, false>(a);                                                               \
  }                                                                                               \
  extern "C" __global__ __launch_bounds__(256) void eos_rot_halves_odd_##NAME(RotArgs a) {        \
    rotate<T, kRotHalves, false>(a);                                                              \
  }
ROT_KERNELS(f16, kRotF16)
ROT_KERNELS(bf16, kRotBf16)
ROT_KERNELS(f32, kRotF32)

extern "C" __global__ __launch_bounds__(kThreads) void eos_pager_extend(PagerArgs a) { extend(a); }
extern "C" __global__ __launch_bounds__(kThreads) void eos_pager_trim(PagerArgs a) { trim(a); }

extern "C" __global__ __launch_bounds__(256) void eos_pager_reset(PagerArgs a) {
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x, all = (long long)gridDim.x * 256;
  for (long long i = id; i < (long long)a.slots * a.stride; i += all) a.table[i] = -1;
  for (long long i = id; i < a.pages; i += all) a.free_list[i] = (int)(a.pages - 1 - i);
  if (id < a.slots) a.lengths[id] = 0;
  if (id < 2) a.state[id] = 0;
  if (id == 0) *a.free_count = (int)a.pages;
}
