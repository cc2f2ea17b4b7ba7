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
  const int heads = a.heads + a.kv_heads, step = 256 >> a.lanes_shift, all = a.each * heads;
  // A head of a row: where it stands and goes, and its row's turns.
  const auto head = [&](int i, const uint8_t*& x, uint8_t*& y, int& r) {
    r = a.each == 1 ? 0 : i / heads;
    const int h = i - r * heads;
    const bool key = h >= a.heads;
    const long long row = row0 + r, at = (long long)(key ? h - a.heads : h) * a.head_dim * size_of(T);
    x = (key ? a.k + row * a.k_stride : a.q + row * a.q_stride) + at;
    y = (key ? a.k_out + row * a.k_out_stride : a.q_out + row * a.q_out_stride) + at;
  };
  if constexpr (WIDE) {
    // The lane's eight values, of halves also the eight that they turn with. Pairs:
    // four heads' loads are in flight (9,000 ragged rows of 40 heads of 128, a
    // quarter turned: 48 -> 42 us, 4.3 TB/s), halves have two already (16,384 rows of
    // 64 heads: 101 us, 5.3 TB/s; with four heads' 107).
    constexpr bool kHalves = LAYOUT == kRotHalves;
    constexpr int kHeads = kHalves ? 1 : 4;
    const int turning = kHalves ? half / 8 : a.rotary_dim / 8;  // lanes
    const bool turns = lane < turning;
    const int at0 = (turns || !kHalves ? lane * 8 : a.rotary_dim + (lane - turning) * 8) * size_of(T);
    const bool any = at0 < a.head_dim * size_of(T);
    const v2f* my = cs + (kHalves ? lane * 8 : lane * 4);
    for (int i0 = threadIdx.x >> a.lanes_shift; i0 < all; i0 += kHeads * step) {
      float u[kHeads][8], v[kHeads][kHalves ? 8 : 1];
      uint8_t* y[kHeads];
      int r[kHeads];
      bool live[kHeads];
#pragma unroll
      for (int c = 0; c < kHeads; ++c) {
        live[c] = false;
        if (i0 + c * step >= all) continue;
        const uint8_t* x;
        head(i0 + c * step, x, y[c], r[c]);
        live[c] = any && pos[r[c]] >= 0 && (turns || x != y[c]);
        if (!live[c]) continue;
        load8<T>(x + at0, u[c]);
        if constexpr (kHalves) {
          if (turns) load8<T>(x + at0 + half * size_of(T), v[c]);
        }
      }
#pragma unroll
      for (int c = 0; c < kHeads; ++c) {
        if (!live[c]) continue;
        const v2f* t = my + r[c] * half;
        if constexpr (kHalves) {
          if (turns) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float p = u[c][i] * t[i][0] - v[c][i] * t[i][1];
              v[c][i] = u[c][i] * t[i][1] + v[c][i] * t[i][0];
              u[c][i] = p;
            }
            store8<T>(y[c] + at0 + half * size_of(T), v[c]);
          }
        } else if (turns) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float p = u[c][2 * i] * t[i][0] - u[c][2 * i + 1] * t[i][1];
            u[c][2 * i + 1] = u[c][2 * i] * t[i][1] + u[c][2 * i + 1] * t[i][0];
            u[c][2 * i] = p;
          }
        }
        store8<T>(y[c] + at0, u[c]);
      }
    }
  } else {
    // Halves or pairs that do not begin at such: a value at a time (16,384 rows of 40
    // heads of 128 bf16 in place: 122 of the head turned in 128 us by halves and 114
    // by pairs, all of it eight at a time in 67 and 71; one row a sequence takes as
    // long either way).
    for (int i0 = threadIdx.x >> a.lanes_shift; i0 < all; i0 += step) {
      const uint8_t* x;
      uint8_t* y;
      int r;
      head(i0, x, y, r);
      if (pos[r] < 0) continue;
      const v2f* turns = cs + r * half;
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

// --------------------------------------------------------------- page tables

constexpr int kThreads = 1024, kWaves = kThreads / 64;

// A barrier that LDS accesses are complete at, stores to memory not.
EOS_DEV void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

template <int CTRL, int ROWS>
EOS_DEV long long from_lane(long long x) {
  const int lo = __builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, true);
  const int hi = __builtin_amdgcn_update_dpp(0, (int)(x >> 32), CTRL, ROWS, 0xf, true);
  return (long long)hi << 32 | (uint32_t)lo;
}
// Sum of a wavefront's lanes up to and with this one, by the vector unit's own
// lane moves (a shuffle goes through LDS: a fifth as fast here).
EOS_DEV long long upto_lane(long long x) {
  x += from_lane<0x111, 0xf>(x);  // rows of 16 shifted by 1, 2, 4, 8
  x += from_lane<0x112, 0xf>(x);
  x += from_lane<0x114, 0xf>(x);
  x += from_lane<0x118, 0xf>(x);
  x += from_lane<0x142, 0xa>(x);  // a row's last to the next row, the second's to the last two
  return x + from_lane<0x143, 0xc>(x);
}
EOS_DEV long long of_lane(long long x, int lane) {
  return (long long)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)x, lane);
}
// The sum of the threads in front of this one, and of all; where FEW, every
// wavefront has the same numbers and needs no other.
template <bool FEW>
EOS_DEV long long before(long long x, long long* sums, long long& total) {
  const long long in = upto_lane(x);
  long long at = in - x;
  total = of_lane(in, 63);
  if constexpr (!FEW) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    lds_barrier();
    if (lane == 0) sums[wave] = total;
    lds_barrier();
    const long long all = upto_lane(lane < kWaves ? sums[lane] : 0);
    if (wave > 0) at += of_lane(all, wave - 1);
    total = of_lane(all, kWaves - 1);
  }
  return at;
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
// read the state that it is about to write. (Nothing that they wrote is read:
// their loads have returned, for what they loaded has been used.)
// Many workgroups count in eight groups first: additions to one place follow
// each other by 10 ns.
template <bool GROUPS>
EOS_DEV bool last_one(const PagerArgs& a, int* flag) {
  lds_barrier();
  if (gridDim.x == 1) return true;
  if (threadIdx.x == 0) {
    int* all = a.state + kPagerLine;
    const auto arrive = [](int* at, int of) {
      if (__hip_atomic_fetch_add(at, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != of - 1) return false;
      __hip_atomic_store(at, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      return true;
    };
    const int n = gridDim.x, g = blockIdx.x % 8;
    *flag = !GROUPS || n < 64 ? arrive(all, n)
                              : arrive(all + (1 + g) * kPagerLine, (n - g + 7) / 8) && arrive(all, 8);
  }
  lds_barrier();
  return *flag != 0;
}

// Every workgroup sums the requests of all slots up by itself, E a thread (8 bytes
// a slot from the L2, no second launch); where there are FEW, 64 at most, every
// wavefront does, without a barrier. The rows of a short request its thread
// writes; for the others and for the table entries, which the workgroups share,
// the batch's ranges are left in LDS. The last one that is done brings lengths
// and stack up to date. What these kernels wait for is a chain of loads and, each
// instruction running once, the instructions: hence loops, not unrolled ones. A
// token for each of 64 slots of 8,000: 8.3 -> 5.8 us, trimmed again 5.7 -> 3.3;
// 1.9 million rows for 4,096 slots 34.6 -> 18.9 (27 MB, 1.4 TB/s) and 13.1 -> 8.1
// (1.5 MB: loads, a scan and the count of workgroups, one behind the other).
template <bool FEW, int E>
EOS_DEV void extend(const PagerArgs& a) {
  extern __shared__ int lds[];
  __shared__ long long sums[kWaves];
  __shared__ int flag, taken, any_long;
  int* row_of = lds;                 // [batch + 1] first row
  int* len_of = row_of + a.slots + 1;  // [batch] tokens before, -1: refused
  int* page_of = len_of + a.slots;     // [batch] first new page's place below the stack's top
  int* slot_of = page_of + a.slots;    // [batch]
  const int lane = threadIdx.x & 63, wave_in = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int wave = blockIdx.x * kWaves + wave_in, waves = gridDim.x * kWaves;
  const int one = (1 << a.page_shift) - 1;
  if (threadIdx.x == 0) taken = any_long = 0;
  lds_barrier();
  const long long room = room_of(a);
  const int slot0 = (FEW ? lane : (int)threadIdx.x) * E;
  int bad = 0, len[E], fresh[E], need[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    len[i] = fresh[i] = 0;
    if (slot0 + i < a.slots) {
      fresh[i] = a.ask[slot0 + i];
      len[i] = a.lengths[slot0 + i];
    }
  }
  const int count = free_pages(a, bad);
  long long all, mine = 0;  // rows << 13 | requests
#pragma unroll
  for (int i = 0; i < E; ++i) {
    if (fresh[i] < 0) {
      bad |= kPagerBadNumber;
      fresh[i] = 0;
    }
    mine += fresh[i] > 0 ? ((long long)fresh[i] << 13) + 1 : 0;
  }
  const long long at0 = before<FEW>(mine, sums, all);
  // A request has room if its table row holds it and its rows are the caller's.
  long long at = at0;
  bool ok[E];
  mine = 0;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    need[i] = 0;
    ok[i] = false;
    if (fresh[i] > 0) {
      at += ((long long)fresh[i] << 13) + 1;
      if (len[i] < 0 || len[i] > room || (at >> 13) > a.rows) bad |= kPagerBadNumber;
      else if (len[i] + (long long)fresh[i] > room) bad |= kPagerNoRoom;
      else {
        ok[i] = true;
        need[i] = pages_of(len[i] + fresh[i], a.page_shift) - pages_of(len[i], a.page_shift);
        mine += need[i];
      }
    }
  }
  // Pages go to slots in order until one asks for more than there are.
  long long asked;
  long long page = before<FEW>(mine, sums, asked);
  at = at0;
  int given = 0;
  bool rows_left = false;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    if (need[i] > 0) {
      if (page + need[i] > count) {
        ok[i] = false;
        bad |= kPagerNoPages;
      } else {
        given = (int)page + need[i];
      }
    }
    if (fresh[i] > 0) {
      const int s = slot0 + i, j = (int)(at & 8191), r0 = (int)min(at >> 13, a.rows);
      const int n = (int)min((long long)fresh[i], a.rows - r0);
      if (!FEW || wave_in == 0) {
        row_of[j] = r0;
        len_of[j] = ok[i] ? len[i] : -1;
        page_of[j] = (int)min(page, (long long)count);
        slot_of[j] = s;
        if (blockIdx.x == 0) {
          a.b_slots[j] = s;
          a.b_lengths[j] = ok[i] ? len[i] + fresh[i] : 0;
          a.b_offsets[j] = r0;
        }
      }
      rows_left |= n > kPagerShort;
      if (n <= kPagerShort && (FEW ? wave == waves - 1 : (wave_in * E + i) % (int)gridDim.x == (int)blockIdx.x)) {
        const int held = pages_of(len[i], a.page_shift);
#pragma unroll 1
        for (int c = 0; c < n; ++c) {
          const int p = len[i] + c, e = p >> a.page_shift;
          long long place = -1;
          if (ok[i] && a.slot_map != nullptr) {
            const int id = e < held ? a.table[(long long)s * a.stride + e]
                                    : a.free_list[count - 1 - ((int)page + e - held)];
            place = ((long long)id << a.page_shift) + (p & one);
          }
          if (a.positions != nullptr) a.positions[r0 + c] = ok[i] ? p : -1;
          if (a.slot_map != nullptr) a.slot_map[r0 + c] = place;
        }
      }
      at += ((long long)fresh[i] << 13) + 1;
    }
    page += need[i];
  }
  // The last granted request's end is what the stack has given.
  const unsigned long long gave = __ballot(given > 0), left = __ballot(rows_left);
  if (gave != 0) given = __builtin_amdgcn_readlane(given, 63 - __builtin_clzll(gave));
  if (lane == 0 && gave != 0) atomicMax(&taken, given);
  if (lane == 0 && left != 0) any_long = 1;
  const int batch = (int)(all & 8191), upto = (int)min(all >> 13, a.rows);
  if (threadIdx.x == 0) {
    row_of[batch] = upto;
    if (blockIdx.x == 0) a.b_offsets[batch] = upto;
  }
  lds_barrier();
  // The rows of the others, 256 a wavefront: between the requests that the first
  // and the last belong to lies each row's.
  if (any_long != 0 && (a.positions != nullptr || a.slot_map != nullptr))
    for (long long first = (long long)wave * kPagerUnit; first < upto; first += (long long)waves * kPagerUnit) {
      const int end = (int)min(first + kPagerUnit, (long long)upto) - 1;
      int j0 = 0, size = batch;  // 64 probes a turn
      while (size > 1) {
        const int step = (size + 63) / 64, probe = j0 + lane * step;
        const int c = __popcll(__ballot(lane * step < size && row_of[min(probe, batch)] <= (int)first)) - 1;
        j0 += c * step;
        size = min(step, size - c * step);
      }
      const int more = __popcll(__ballot(j0 + 1 + lane < batch && row_of[min(j0 + 1 + lane, batch)] <= end));
      const int j1 = more < 64 ? j0 + more : min(batch - 1, j0 + kPagerUnit);
      int p[kPagerUnit / 64], id[kPagerUnit / 64];
      bool set[kPagerUnit / 64];
#pragma unroll
      for (int k = 0; k < kPagerUnit / 64; ++k) {
        const int r = (int)first + k * 64 + lane;
        p[k] = id[k] = -1;
        set[k] = false;
        if (r <= end) {
          int b = j0, hi = j1;  // the last of them that begins at or before r
          while (b < hi) {
            const int mid = (b + hi + 1) / 2;
            if (row_of[mid] <= r) b = mid;
            else hi = mid - 1;
          }
          const int t = len_of[b];
          set[k] = row_of[b + 1] - row_of[b] > kPagerShort;
          if (set[k] && t >= 0) {
            p[k] = t + (r - row_of[b]);
            const int i = p[k] >> a.page_shift, held = pages_of(t, a.page_shift);
            id[k] = i < held ? a.table[(long long)slot_of[b] * a.stride + i]
                             : a.free_list[count - 1 - (page_of[b] + i - held)];
          }
        }
      }
#pragma unroll
      for (int k = 0; k < kPagerUnit / 64; ++k) {
        const long long r = first + k * 64 + lane;
        if (!set[k]) continue;
        if (a.positions != nullptr) a.positions[r] = p[k];
        if (a.slot_map != nullptr)
          a.slot_map[r] = p[k] < 0 ? -1 : ((long long)id[k] << a.page_shift) + (p[k] & one);
      }
    }
  // Table rows: what a slot has, then its new pages; a wavefront a slot and
  // kPagerEntries of its entries.
  const int pieces = (a.stride + kPagerEntries - 1) / kPagerEntries;
  for (int u = wave; u < batch * pieces; u += waves) {
    const int b = pieces == 1 ? u : u / pieces, first = (u - b * pieces) * kPagerEntries;
    const int t = len_of[b], held = pages_of(t, a.page_shift);
    const int end = min(pages_of(t + row_of[b + 1] - row_of[b], a.page_shift), first + kPagerEntries);
    if (t < 0 || first >= end || (a.b_table == nullptr && held >= end)) continue;
    int32_t* from = a.table + (long long)slot_of[b] * a.stride;
    int32_t* to = a.b_table != nullptr ? a.b_table + (long long)b * a.stride : nullptr;
    const int32_t* top = a.free_list + (count - 1 - page_of[b] + held);
    int id[kPagerEntries / 64];
#pragma unroll
    for (int k = 0; k < kPagerEntries / 64; ++k) {
      const int i = first + k * 64 + lane;
      if (i < end) id[k] = *(i < held ? from + i : top - i);
    }
#pragma unroll
    for (int k = 0; k < kPagerEntries / 64; ++k) {
      const int i = first + k * 64 + lane;
      if (i < end && i >= held) from[i] = id[k];
      if (i < end && to != nullptr) to[i] = id[k];
    }
  }
  if (blockIdx.x == 0 && bad != 0) atomicOr(&a.state[0], bad);
  if (!last_one<!FEW>(a, &flag)) return;
  for (int j = threadIdx.x; j < batch; j += kThreads)
    if (len_of[j] >= 0) a.lengths[slot_of[j]] = len_of[j] + row_of[j + 1] - row_of[j];
  if (threadIdx.x == 0) *a.free_count = count - taken;
}

// Pages behind the tokens to keep go back onto the stack, the last slot's last
// page first: extends undone leave it as it was.
template <bool FEW, int E>
EOS_DEV void trim(const PagerArgs& a) {
  extern __shared__ int lds[];
  __shared__ long long sums[kWaves];
  __shared__ int flag;
  int* page_of = lds;                // [slots] pages in front of a slot's
  int* gone_of = page_of + a.slots;  // [slots] its pages
  int* keep_of = gone_of + a.slots;  // [slots] tokens that stay, -1: as they are
  const int lane = threadIdx.x & 63, wave_in = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int wave = blockIdx.x * kWaves + wave_in, waves = gridDim.x * kWaves;
  const long long room = room_of(a);
  const int slot0 = (FEW ? lane : (int)threadIdx.x) * E;
  int bad = 0, len[E], keep[E], gone[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    len[i] = 0;
    keep[i] = -1;
    if (slot0 + i < a.slots) {
      len[i] = a.lengths[slot0 + i];
      keep[i] = a.ask[slot0 + i];
    }
  }
  const int count = free_pages(a, bad);
  long long all, mine = 0;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    gone[i] = 0;
    if (len[i] < 0 || len[i] > room) {
      bad |= kPagerBadNumber;
      keep[i] = -1;
    } else if (keep[i] >= len[i]) {
      keep[i] = -1;
    } else if (keep[i] >= 0) {
      gone[i] = pages_of(len[i], a.page_shift) - pages_of(keep[i], a.page_shift);
    }
    mine += gone[i];
  }
  long long at = before<FEW>(mine, sums, all);
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int s = slot0 + i;
    if (s < a.slots && (!FEW || wave_in == 0)) {
      page_of[s] = (int)min(at, (long long)INT32_MAX);
      gone_of[s] = gone[i];
      keep_of[s] = keep[i];
    }
    at += gone[i];
  }
  if (count + all > a.pages) bad |= kPagerBadNumber;
  lds_barrier();
  if (all > 0) {
    const int pieces = (a.stride + kPagerEntries - 1) / kPagerEntries;
    for (int u = wave; u < a.slots * pieces; u += waves) {
      const int s = pieces == 1 ? u : u / pieces, first = (u - s * pieces) * kPagerEntries;
      const int end = min(gone_of[s], first + kPagerEntries);
      if (first >= end) continue;
      int32_t* from = a.table + (long long)s * a.stride + pages_of(keep_of[s], a.page_shift);
      const long long top = count + all - 1 - page_of[s];
      int id[kPagerEntries / 64];
#pragma unroll
      for (int k = 0; k < kPagerEntries / 64; ++k) {
        const int i = first + k * 64 + lane;
        if (i < end) id[k] = from[i];
      }
#pragma unroll
      for (int k = 0; k < kPagerEntries / 64; ++k) {
        const int i = first + k * 64 + lane;
        if (i >= end) continue;
        if (top - i >= 0 && top - i < a.pages) a.free_list[top - i] = id[k];
        from[i] = -1;
      }
    }
  }
  if (blockIdx.x == 0 && bad != 0) atomicOr(&a.state[0], bad);
  if (!last_one<!FEW>(a, &flag)) return;
  for (int s = threadIdx.x; s < a.slots; s += kThreads)
    if (keep_of[s] >= 0) a.lengths[s] = keep_of[s];
  if (threadIdx.x == 0) *a.free_count = (int)min(count + all, a.pages);
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

#define PAGER_KERNELS(NAME, FEW, E)                                                                \
  extern "C" __global__ __launch_bounds__(kThreads) void eos_pager_extend_##NAME(PagerArgs a) {    \
    extend<FEW, E>(a);                                                                             \
  }                                                                                                \
  extern "C" __global__ __launch_bounds__(kThreads) void eos_pager_trim_##NAME(PagerArgs a) {      \
    trim<FEW, E>(a);                                                                               \
  }
PAGER_KERNELS(few, true, 1)
PAGER_KERNELS(some, false, 1)
PAGER_KERNELS(many, false, kPagerSlots / kThreads)

extern "C" __global__ __launch_bounds__(256) void eos_pager_reset(PagerArgs a) {
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x, all = (long long)gridDim.x * 256;
  for (long long i = id; i < (long long)a.slots * a.stride; i += all) a.table[i] = -1;
  for (long long i = id; i < a.pages; i += all) a.free_list[i] = (int)(a.pages - 1 - i);
  if (id < a.slots) a.lengths[id] = 0;
  if (id == 0) a.state[0] = 0;
  if (id == 0) *a.free_count = (int)a.pages;
}
