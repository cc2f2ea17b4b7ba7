// Kernel argument blocks of the microscaled 4-bit code object, shared with the
// host shim.
#ifndef EOSHIP_MX_ARGS_H
#define EOSHIP_MX_ARGS_H

#include <stdint.h>

// Element types of the rows a caller passes.
enum { kMxF16 = 0, kMxBf16 = 1, kMxF32 = 2, kMxCodes = 3 };

constexpr int kMxBlock = 32;      // values of a scale
constexpr int kMxQuad = 256;      // values of K that are laid out together
constexpr int kMxTile = 32;       // rows that are laid out together
constexpr int kMxTileBytes = 4096;  // codes of both
constexpr int kMxScaleBytes = 256;  // and scales

// Rows in the order that matrix instructions read them. Tile t (32 rows) and
// quad q (four steps of 64 values) are 4096 bytes at (t * quads + q) * 4096:
// step s's 1024 hold, 16 bytes a lane, block 8 q + 2 s + l / 32 of row
// 32 t + l % 32. Their scales are byte s of the lanes' words at (t * quads + q)
// * 256. Rows and blocks that the matrix lacks are zero.
struct MxLaid {
  uint8_t* codes;
  uint8_t* scales;
  long long rows;
  int blocks;      // ceil(k / 32)
  int quads;       // ceil(k / 256)
};

struct MxQuantArgs {
  const uint8_t* x;    // caller's rows, or codes
  const uint8_t* xs;   // scales of codes
  long long stride;    // bytes between rows of x
  uint8_t* codes;      // [rows][blocks][16]
  uint8_t* scales;     // [rows][blocks]
  MxLaid laid;         // where laid out
  long long rows;
  int k, blocks;
};

struct MxDequantArgs {
  const uint8_t* codes;
  const uint8_t* scales;
  uint8_t* out;
  long long stride;    // bytes between rows of out
  long long rows;
  int k, blocks;
};

struct MxLinearArgs {
  MxLaid x, w;           // x where its rows are laid out
  const uint8_t* rows_x;   // and where they are not: rows, or codes
  const uint8_t* scales_x;
  long long x_stride;    // bytes
  const float* bias;     // [n] or NULL
  uint8_t* out;
  long long out_stride;  // bytes
  long long rows;
  int n, k, out_type;
  int tiles_m, tiles_n;  // workgroup tiles
};

#endif
