// Kernel argument blocks of the key-value cache code object, shared with the
// host shim.
#ifndef EOSHIP_KV_ARGS_H
#define EOSHIP_KV_ARGS_H

#include <stdint.h>

// Storage formats and element types of the rows a caller passes.
enum { kKvF16 = 0, kKvBf16 = 1, kKvQ8 = 2, kKvTq4 = 3 };
enum { kKvRowF16 = 0, kKvRowBf16 = 1, kKvRowF32 = 2 };

constexpr int kKvFewSplits = 8;        // splits that one lane group joins by itself
constexpr int kKvStreamBatch = 512;   // sequences whose steps every workgroup sums up

// Status bits a kernel sets when what it read from the device was out of
// range (nothing outside the pool and the rows is touched).
enum { kKvBadPage = 1, kKvBadLength = 2, kKvBadOffset = 4 };

constexpr int kKvMostKeys = 1 << 30;  // tokens of a sequence: positions and steps stay in 32 bits
constexpr int kKvGroup = 8;       // tokens of V stored side by side
constexpr int kKvRun = 32;         // positions of a workgroup of append and read
constexpr int kKvTileRows = 16;    // query rows of a workgroup of the split kernel
constexpr int kKvPromptRows = 128;  // query rows of a workgroup of the prompt kernel

struct KvTables {
  uint32_t hi[2], lo[2];  // tq4: high and low bytes of the 8 f16 magnitudes
  float edges[7];         // tq4: thresholds between them
  float mags[8];          // tq4: the magnitudes
  const float* signs;     // tq4: [head_dim]
};

// The cache and a batch of sequences over it.
struct KvCacheArgs {
  uint8_t *k, *v;           // page pools
  float *k_scale, *v_scale;  // [pages][kv_heads][page_tokens]
  const int32_t* table;     // [batch][table_stride] page ids
  const int32_t* lengths;   // [batch] tokens, the call's rows included
  const int32_t* offsets;   // [batch + 1] row ranges, or NULL: one row each
  int32_t* status;
  KvTables t;
  long long rows;
  int pages, kv_heads, page_shift, table_stride, batch;
};

struct KvRowsArgs {
  KvCacheArgs c;
  uint8_t *k, *v;               // caller's rows (append reads, read writes)
  long long k_stride, v_stride;  // elements between rows
  int dtype;
};

struct KvAttnArgs {
  KvCacheArgs c;
  const uint8_t* q;
  uint8_t* out;
  float* lse;       // [rows][heads] or NULL
  float* part;      // [tiles][kv_heads][splits][tile_rows][head_dim] unnormalised sums
  float* part_ml;   // [tiles][kv_heads][splits][tile_rows][2] reference and weight sum
                    // (stream kernels: [workgroups][2][16] of both)
  long long q_stride, out_stride;
  float scale;      // of q . k, times log2(e)
  long long tiles;
  int heads, group, window, splits, dtype, tile_rows, workgroups;
};

#endif
