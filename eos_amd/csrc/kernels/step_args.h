// Kernel argument blocks of the decoding step's code object (rotary positions,
// page tables), shared with the host shim.
#ifndef EOSHIP_STEP_ARGS_H
#define EOSHIP_STEP_ARGS_H

#include <stdint.h>

enum { kRotF16 = 0, kRotBf16 = 1, kRotF32 = 2 };
enum { kRotPairs = 0, kRotHalves = 1 };

constexpr int kRotAngles = 256;  // cosines and sines that a workgroup computes at once
constexpr int kRotRows = 16;     // rows of a workgroup at most

struct RotArgs {
  const uint8_t *q, *k;
  uint8_t *q_out, *k_out;
  long long q_stride, k_stride, q_out_stride, k_out_stride;  // bytes between rows
  const double* turns;      // [rotary_dim / 2] frequencies in turns a position
  const int32_t* positions;  // [rows], or the batch's
  const int32_t* lengths;    // [batch]
  const int32_t* offsets;    // [batch + 1] or NULL: one row each
  long long rows;
  int batch, heads, kv_heads, head_dim, rotary_dim, layout;
  int each;                  // rows of a workgroup
  int lanes_shift;           // log2 of the lanes of a head
  float factor, sign;        // sign -1: turned back
};

// Status bits of a pager.
enum { kPagerNoPages = 1, kPagerNoRoom = 2, kPagerBadNumber = 4 };
constexpr int kPagerSlots = 4096;    // slots that every workgroup sums up
constexpr int kPagerFew = 64;       // ... and every wavefront
constexpr int kPagerShort = 4;      // rows of a request that one thread writes
constexpr int kPagerUnit = 256;    // rows that a wavefront takes at a time
constexpr int kPagerEntries = 256;  // table entries that it does

constexpr int kPagerLine = 32;      // words of a cache line
constexpr int kPagerState = 10 * kPagerLine;  // status; workgroups done, of eight groups

struct PagerArgs {
  int32_t* table;     // [slots][stride]
  int32_t* lengths;   // [slots]
  int32_t* free_list;  // [pages], a stack
  int32_t* free_count;
  int32_t* state;
  const int32_t* ask;  // extend: new tokens, trim: tokens to keep, of every slot
  int32_t *b_slots, *b_table, *b_lengths, *b_offsets, *positions;
  int64_t* slot_map;
  long long pages, rows;
  int slots, stride, page_shift;
};

#endif
