// Kernel argument blocks of the microscaled 4-bit code object, shared with the
// host shim.
#ifndef EOSHIP_MX_ARGS_H
#define EOSHIP_MX_ARGS_H

#include <stdint.h>

// Element types of the rows a caller passes.
enum { kMxF16 = 0, kMxBf16 = 1, kMxF32 = 2, kMxCodes = 3 };

constexpr int kMxBlock = 32;      // values of a scale
constexpr int kMxStep = 128;      // values of K a matrix instruction takes
constexpr int kMxTile = 16;       // rows of a laid-out tile
constexpr int kMxTileBytes = 1024;  // a tile's codes of a step: 64 lanes of 16 bytes
constexpr int kMxScaleBytes = 256;  // a tile's scales of four steps: 64 lanes of 4 bytes

// Rows in the order that matrix instructions read them. Tile t (16 rows) and
// step s (128 values) are 1024 bytes at (t * steps + s) * 1024: lane l holds
// block 4 s + l / 16 of row 16 t + l % 16. Its scales are byte s % 4 of the
// lanes' words at (t * quads + s / 4) * 256. Rows and blocks that the matrix
// lacks are zero.
struct MxLaid {
  uint8_t* codes;
  uint8_t* scales;
  long long rows;
  int blocks;      // ceil(k / 32)
  int steps;       // ceil(k / 128)
  int quads;       // ceil(steps / 4)
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
  MxLaid x, w;
  const float* bias;   // [n] or NULL
  uint8_t* out;
  long long out_stride;  // bytes
  long long rows;
  int n, k;
  int tiles_m, tiles_n;  // workgroup tiles
};

#endif
