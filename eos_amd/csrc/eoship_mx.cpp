// Microscaled 4-bit half of the eoship C ABI: rows quantised and taken back,
// and linear layers over weights held in that form. Beside the q8 encoder's
// matrix products (runtime/backend/tensor_ops.go:938-2208 on the host), the
// form that the matrix units of gfx950 multiply directly.
#include <algorithm>
#include <cstdint>
#include <string>

#include "eoship_internal.h"
#include "kernels/mx_args.h"
#include "row_ranges.h"

using eoship::bytes_of;
using eoship::guarded;
using eoship::hip_err;
using eoship::OnDevice;
using eoship::Rows;
using eoship::rows_meet;
using eoship::rows_of;
using eoship::set_err;

struct EosHipMX {
  EosHipRuntime* rt = nullptr;
  int n = 0, k = 0;
  MxLaid w{};
  const float* bias = nullptr;
  void* mem = nullptr;  // codes, scales, bias
  ~EosHipMX() {
    if (mem != nullptr) hipFree(mem);
  }
};

namespace {

constexpr int kMost = 1 << 24;  // values of a row, outputs of a layer
constexpr long long kGroups = (1 << 24) - 1;  // workgroups of 256 threads in a launch

// Which kernel takes a layer's rows (256 CUs; us of a call among others, 4,096
// values, bf16, weights from HBM).
// Up to 16 rows are quantised by the workgroups that multiply them, in one
// launch (16 rows by 6,144 weights 8.6, by 16,384 12.7; laid out first 10.2 and
// 13.1). A workgroup takes 16 weights, 32 where there are more of those than CUs
// (1 row by 6,144: 6.1 and 5.8, 16 rows 12.1 and 8.6; by 4,096: 5.4 and 5.4, 7.8
// and 7.9), 64 where there are more than twice as many and the rows' quantisation
// weighs (16 by 16,384: 20.5, 15.5 and 12.7; by 6,144 with 64 10.3).
constexpr int kFewRows = 16;
// Up to 64 are laid out by a launch before and multiplied in the same way (64 by
// 2,048 9.1, by tiles of 64 12.0; by 6,144 12.0 and 14.7, by 16,384 16.0 and 15.9).
constexpr int kSomeRows = 64;
// More go by tiles of outputs. Tiles of 64 while there are no more than two a CU
// (512 by 4,096: 17.0, by tiles of 128 18.9; 1,024 by 4,096: 26.4 and 22.0); then
// of 128, two workgroups a CU, or of 256, one, whose turn takes 3/2 the time of the
// two's or more (2,048 rows; a turn each, by 4,096: 32.4 and 38.6; two turns and
// one, by 8,192: 54.7 and 44.7; four and two, by 16,384: 102 and 83). At three
// turns and two, where both predict the same, those of 128: their last turn is
// shorter where it is not full (by 10,240: 65.5 and 74.1; full, by 12,288: 76.8 and
// 76.4).

const char* const kTypes[] = {"f16", "bf16", "f32", "codes"};

bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }
int size_of(int type) { return type == kMxF32 ? 4 : 2; }
int ceil_div(int a, int b) { return (a + b - 1) / b; }

MxLaid laid(long long rows, int k) {
  MxLaid m{};
  m.rows = rows;
  m.blocks = ceil_div(k, kMxBlock);
  m.quads = ceil_div(k, kMxQuad);
  return m;
}
size_t tiles(const MxLaid& m) { return (size_t)((m.rows + kMxTile - 1) / kMxTile); }
size_t code_bytes(const MxLaid& m) { return tiles(m) * m.quads * kMxTileBytes; }
size_t scale_bytes(const MxLaid& m) { return tiles(m) * m.quads * kMxScaleBytes; }
void place(MxLaid* m, void* mem) {
  m->codes = static_cast<uint8_t*>(mem);
  m->scales = m->codes + code_bytes(*m);
}

int check_shape(int64_t rows, int32_t k, const char* what, char** err) {
  if (rows < 0 || rows > INT32_MAX)
    return set_err(err, "%s: rows must be in 0..2^31-1, got %lld", what, (long long)rows);
  if (k < 1 || k > kMost) return set_err(err, "%s: k must be in 1..2^24, got %d", what, k);
  return 0;
}

int check_blocks(int64_t rows, int32_t k, const char* what, char** err) {
  if (rows * ceil_div(k, kMxBlock) <= 64 * kGroups) return 0;
  return set_err(err, "%s: %lld rows of %d values are more than 2^30 - 64 blocks", what,
                 (long long)rows, k);
}

int check_tiles(int64_t rows, int32_t k, const char* what, char** err) {
  if ((rows + kMxTile - 1) / kMxTile * ceil_div(k, kMxQuad) <= kGroups) return 0;
  return set_err(err, "%s: %lld rows of %d values are more than 2^24 - 1 tiles of 32 rows by 256",
                 what, (long long)rows, k);
}

int check_type(int32_t type, int most, const char* what, char** err) {
  if (type < 0 || type > most)
    return set_err(err, "%s: dtype must be 0 (f16), 1 (bf16)%s, got %d", what,
                   most == kMxF32 ? " or 2 (f32)" : ", 2 (f32) or 3 (mxfp4)", type);
  return 0;
}

int check_rows(const void* p, int64_t stride, int64_t width, const char* name, const char* what,
               char** err) {
  if (p == nullptr) return set_err(err, "%s: %s is NULL", what, name);
  if (!aligned(p)) return set_err(err, "%s: %s is not 16-byte aligned", what, name);
  if (stride < width || stride % 8 != 0 || stride > 1LL << 40)
    return set_err(err,
                   "%s: the row stride of %s must be a multiple of 8 and at least %lld (at most "
                   "2^40), got %lld",
                   what, name, (long long)width, (long long)stride);
  return 0;
}

int check_codes(const void* codes, const void* scales, const char* what, char** err) {
  if (codes == nullptr || scales == nullptr)
    return set_err(err, "%s: NULL codes or scales", what);
  if (!aligned(codes)) return set_err(err, "%s: codes are not 16-byte aligned", what);
  return 0;
}

int launch(EosHipRuntime* rt, const std::string& name, long long blocks, void* args,
           const char* what, char** err) {
  if (blocks > kGroups) return set_err(err, "%s: too many outputs for one call", what);
  return rt->launch(name.c_str(), dim3((unsigned)blocks), dim3(256), 0, args, err);
}

// Rows (or codes) into a laid-out matrix.
int lay(EosHipRuntime* rt, const MxLaid& to, const void* x, int64_t stride, int type,
        const void* scales, int k, const char* what, char** err) {
  MxQuantArgs a{};
  a.x = static_cast<const uint8_t*>(x);
  a.xs = static_cast<const uint8_t*>(scales);
  a.stride = type == kMxCodes ? 0 : stride * size_of(type);
  a.laid = to;
  a.rows = to.rows;
  a.k = k;
  a.blocks = to.blocks;
  return launch(rt, std::string("eos_mx_lay_") + kTypes[type], (long long)tiles(to) * to.quads, &a,
                what, err);
}

// Few rows by 16 `tiles` rows of weights a workgroup.
int few(EosHipRuntime* rt, const std::string& kind, int tiles, MxLinearArgs* a, char** err) {
  const std::string name = "eos_mx_few_" + kind + "_" + std::to_string(tiles);
  return rt->launch(name.c_str(), dim3((unsigned)ceil_div(a->n, 16 * tiles)), dim3(512), 0, a, err);
}

}  // namespace

extern "C" {

int eoship_mx_bytes(int64_t rows, int32_t k, int64_t* code_bytes, int64_t* scale_bytes,
                    char** err) {
  if (check_shape(rows, k, "eoship_mx_bytes", err) != 0) return 1;
  const int64_t blocks = rows * ceil_div(k, kMxBlock);
  if (code_bytes) *code_bytes = blocks * 16;
  if (scale_bytes) *scale_bytes = blocks;
  return 0;
}

int eoship_mx_quantize_device(EosHipRuntime* rt, const void* d_x, int64_t x_stride, int32_t dtype,
                              int64_t rows, int32_t k, uint8_t* d_codes, uint8_t* d_scales,
                              char** err) {
  const char* what = "eoship_mx_quantize_device";
  return guarded(what, err, [&]() -> int {
    if (check_shape(rows, k, what, err) != 0 || check_type(dtype, kMxF32, what, err) != 0 ||
        check_blocks(rows, k, what, err) != 0)
      return 1;
    if (rt == nullptr) return set_err(err, "%s: NULL runtime", what);
    if (rows == 0) return 0;
    if (check_rows(d_x, x_stride, k, "x", what, err) != 0 ||
        check_codes(d_codes, d_scales, what, err) != 0)
      return 1;
    const int64_t blocks = rows * ceil_div(k, kMxBlock);
    const Rows x = rows_of(d_x, rows, x_stride * size_of(dtype), (int64_t)k * size_of(dtype));
    const Rows codes = bytes_of(d_codes, blocks * 16), scales = bytes_of(d_scales, blocks);
    if (rows_meet(x, codes) || rows_meet(x, scales))
      return set_err(err, "%s: codes or scales overlap x", what);
    if (rows_meet(codes, scales)) return set_err(err, "%s: scales overlap codes", what);
    OnDevice on(rt->device);
    if (rt->load(eoship::Runtime::kMx, err) != 0) return 1;
    MxQuantArgs a{};
    a.x = static_cast<const uint8_t*>(d_x);
    a.stride = x_stride * size_of(dtype);
    a.codes = d_codes;
    a.scales = d_scales;
    a.rows = rows;
    a.k = k;
    a.blocks = ceil_div(k, kMxBlock);
    return launch(rt, std::string("eos_mx_quantize_") + kTypes[dtype], (rows * a.blocks + 63) / 64,
                  &a, what, err);
  });
}

int eoship_mx_dequantize_device(EosHipRuntime* rt, const uint8_t* d_codes, const uint8_t* d_scales,
                                int64_t rows, int32_t k, void* d_out, int64_t out_stride,
                                int32_t dtype, char** err) {
  const char* what = "eoship_mx_dequantize_device";
  return guarded(what, err, [&]() -> int {
    if (check_shape(rows, k, what, err) != 0 || check_type(dtype, kMxF32, what, err) != 0 ||
        check_blocks(rows, k, what, err) != 0)
      return 1;
    if (rt == nullptr) return set_err(err, "%s: NULL runtime", what);
    if (rows == 0) return 0;
    if (check_codes(d_codes, d_scales, what, err) != 0 ||
        check_rows(d_out, out_stride, k, "out", what, err) != 0)
      return 1;
    const int64_t blocks = rows * ceil_div(k, kMxBlock);
    const Rows out = rows_of(d_out, rows, out_stride * size_of(dtype), (int64_t)k * size_of(dtype));
    if (rows_meet(out, bytes_of(d_codes, blocks * 16)) || rows_meet(out, bytes_of(d_scales, blocks)))
      return set_err(err, "%s: out overlaps codes or scales", what);
    OnDevice on(rt->device);
    if (rt->load(eoship::Runtime::kMx, err) != 0) return 1;
    MxDequantArgs a{};
    a.codes = d_codes;
    a.scales = d_scales;
    a.out = static_cast<uint8_t*>(d_out);
    a.stride = out_stride * size_of(dtype);
    a.rows = rows;
    a.k = k;
    a.blocks = ceil_div(k, kMxBlock);
    return launch(rt, std::string("eos_mx_dequantize_") + kTypes[dtype],
                  (rows * a.blocks + 63) / 64, &a, what, err);
  });
}

int eoship_mx_bind(EosHipRuntime* rt, const uint8_t* d_codes, const uint8_t* d_scales, int32_t n,
                   int32_t k, const float* d_bias, EosHipMX** out, char** err) {
  const char* what = "eoship_mx_bind";
  return guarded(what, err, [&]() -> int {
    if (out != nullptr) *out = nullptr;
    if (n < 1 || n > kMost) return set_err(err, "%s: n must be in 1..2^24, got %d", what, n);
    if (check_shape(n, k, what, err) != 0 || check_tiles(n, k, what, err) != 0 ||
        check_codes(d_codes, d_scales, what, err) != 0)
      return 1;
    if (((uintptr_t)d_bias & 3) != 0) return set_err(err, "%s: bias is not 4-byte aligned", what);
    if (rt == nullptr || out == nullptr) return set_err(err, "%s: NULL argument", what);
    OnDevice on(rt->device);
    if (rt->load(eoship::Runtime::kMx, err) != 0) return 1;
    auto* mx = new EosHipMX();
    mx->rt = rt;
    mx->n = n;
    mx->k = k;
    mx->w = laid(n, k);
    const size_t held = code_bytes(mx->w) + scale_bytes(mx->w);
    int rc = rt->alloc(held + (d_bias != nullptr ? (size_t)n * 4 : 0), &mx->mem, err);
    if (rc == 0) {
      place(&mx->w, mx->mem);
      rc = lay(rt, mx->w, d_codes, 0, kMxCodes, d_scales, k, what, err);
    }
    if (rc == 0 && d_bias != nullptr) {
      float* b = reinterpret_cast<float*>(static_cast<char*>(mx->mem) + held);
      const hipError_t e = rt->copy_async(b, d_bias, (size_t)n * 4, hipMemcpyDeviceToDevice);
      if (e != hipSuccess) rc = hip_err(err, what, e);
      mx->bias = b;
    }
    // Done with the caller's memory when the call returns.
    if (rc == 0) rc = rt->sync(err);
    if (rc != 0) {
      delete mx;
      return rc;
    }
    *out = mx;
    return 0;
  });
}

int eoship_mx_release(EosHipRuntime* rt, EosHipMX* mx, char** err) {
  if (mx == nullptr) return 0;
  if (rt == nullptr || mx->rt != rt) return set_err(err, "eoship_mx_release: wrong runtime");
  OnDevice on(rt->device);
  if (rt->sync(err) != 0) return 1;
  delete mx;
  return 0;
}

int eoship_mx_linear_device(EosHipRuntime* rt, EosHipMX* mx, const void* d_x, int64_t x_stride,
                            int32_t dtype, const uint8_t* d_x_scales, int64_t rows, void* d_out,
                            int64_t out_stride, int32_t out_dtype, char** err) {
  const char* what = "eoship_mx_linear_device";
  return guarded(what, err, [&]() -> int {
    if (rt == nullptr || mx == nullptr) return set_err(err, "%s: NULL argument", what);
    if (mx->rt != rt) return set_err(err, "%s: the layer is bound to another runtime", what);
    if (check_shape(rows, mx->k, what, err) != 0 || check_tiles(rows, mx->k, what, err) != 0 ||
        check_type(dtype, kMxCodes, what, err) != 0 ||
        check_type(out_dtype, kMxF32, what, err) != 0)
      return 1;
    if (rows == 0) return 0;
    if (dtype == kMxCodes ? check_codes(d_x, d_x_scales, what, err) != 0
                          : check_rows(d_x, x_stride, mx->k, "x", what, err) != 0)
      return 1;
    if (check_rows(d_out, out_stride, mx->n, "out", what, err) != 0) return 1;
    const int64_t blocks = rows * ceil_div(mx->k, kMxBlock), size = size_of(out_dtype);
    const Rows out = rows_of(d_out, rows, out_stride * size, mx->n * size);
    const Rows in = dtype == kMxCodes
                        ? bytes_of(d_x, blocks * 16)
                        : rows_of(d_x, rows, x_stride * size_of(dtype), (int64_t)mx->k * size_of(dtype));
    if (rows_meet(out, in)) return set_err(err, "%s: out overlaps x", what);
    if (dtype == kMxCodes && rows_meet(out, bytes_of(d_x_scales, blocks)))
      return set_err(err, "%s: out overlaps x's scales", what);
    OnDevice on(rt->device);
    MxLinearArgs a{};
    a.w = mx->w;
    a.x = laid(rows, mx->k);
    a.bias = mx->bias;
    a.out = static_cast<uint8_t*>(d_out);
    a.out_stride = out_stride * size_of(out_dtype);
    a.rows = rows;
    a.n = mx->n;
    a.k = mx->k;
    a.out_type = out_dtype;
    const int cus = rt->compute_units, n16 = ceil_div(mx->n, 16);
    if (rows <= kFewRows) {
      a.rows_x = static_cast<const uint8_t*>(d_x);
      a.scales_x = d_x_scales;
      a.x_stride = dtype == kMxCodes ? 0 : x_stride * size_of(dtype);
      const bool four = dtype != kMxCodes && rows <= 4;
      const int tiles = n16 <= cus ? 1 : n16 <= 2 * cus || four || dtype == kMxCodes ? 2 : 4;
      return few(rt, std::string(kTypes[dtype]) + (four ? "_4" : "_16"), tiles, &a, err);
    }
    void* ws = nullptr;
    if (rt->workspace(code_bytes(a.x) + scale_bytes(a.x), &ws, err) != 0) return 1;
    place(&a.x, ws);
    if (lay(rt, a.x, d_x, x_stride, dtype, d_x_scales, mx->k, what, err) != 0) return 1;
    if (rows <= kSomeRows)
      return few(rt, "laid_" + std::to_string((rows + 15) / 16 * 16), n16 <= cus ? 1 : 2, &a, err);
    const auto count = [&](int t) { return ((rows + t - 1) / t) * ceil_div(mx->n, t); };
    const auto turns = [&](long long tiles, int at_once) {
      return (tiles + (long long)at_once * cus - 1) / ((long long)at_once * cus);
    };
    const int t = count(64) <= 2 * cus ? 64 : 3 * turns(count(256), 1) >= 2 * turns(count(128), 2) ? 128 : 256;
    a.tiles_m = (int)((rows + t - 1) / t);
    a.tiles_n = ceil_div(mx->n, t);
    return launch(rt, "eos_mx_product_" + std::to_string(t) + "_" + kTypes[out_dtype],
                  (long long)a.tiles_m * a.tiles_n, &a, what, err);
  });
}

}  // extern "C"
