// Rotary positions half of the eoship C ABI: queries and keys turned by their
// positions in a paged cache's batch. The reference's ropeRows
// (runtime/backend/tensor_ops.go:1936-1965) turns whole rows by pairs; this is
// the form that heads of a decoder take.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>
#include <vector>

#include "eoship_internal.h"
#include "kernels/step_args.h"
#include "row_ranges.h"

using eoship::bytes_of;
using eoship::guarded;
using eoship::hip_err;
using eoship::OnDevice;
using eoship::Rows;
using eoship::rows_meet;
using eoship::rows_of;
using eoship::set_err;

struct EosHipRotary {
  EosHipRuntime* rt = nullptr;
  int head_dim = 0, rotary_dim = 0, layout = 0;
  float factor = 1.0f;
  double* turns = nullptr;
  ~EosHipRotary() {
    if (turns != nullptr) hipFree(turns);
  }
};

namespace {

const char* const kTypes[] = {"f16", "bf16", "f32"};

int check_rows(const void* p, int64_t stride, int64_t width, const char* name, const char* what,
               char** err) {
  if (p == nullptr) return set_err(err, "%s: %s is NULL", what, name);
  if (((uintptr_t)p & 15) != 0) return set_err(err, "%s: %s is not 16-byte aligned", what, name);
  if (stride < width || stride % 8 != 0 || stride > 1LL << 40)
    return set_err(err,
                   "%s: the row stride of %s must be a multiple of 8 and at least %lld (at most "
                   "2^40), got %lld",
                   what, name, (long long)width, (long long)stride);
  return 0;
}

}  // namespace

extern "C" {

int eoship_rotary_bind(EosHipRuntime* rt, const EosHipRotaryDesc* desc, EosHipRotary** out,
                       char** err) {
  const char* what = "eoship_rotary_bind";
  return guarded(what, err, [&]() -> int {
    if (out != nullptr) *out = nullptr;
    if (desc == nullptr) return set_err(err, "%s: desc is NULL", what);
    if (desc->head_dim < 8 || desc->head_dim > 1024 || desc->head_dim % 8 != 0)
      return set_err(err, "%s: head_dim must be a multiple of 8 in 8..1024, got %d", what,
                     desc->head_dim);
    if (desc->rotary_dim < 2 || desc->rotary_dim > desc->head_dim || desc->rotary_dim % 2 != 0)
      return set_err(err, "%s: rotary_dim must be even and in 2..head_dim, got %d", what,
                     desc->rotary_dim);
    if (desc->layout != kRotPairs && desc->layout != kRotHalves)
      return set_err(err, "%s: layout must be 0 (pairs) or 1 (halves), got %d", what, desc->layout);
    if (!std::isfinite(desc->factor)) return set_err(err, "%s: factor must be finite", what);
    if (desc->frequencies == nullptr) return set_err(err, "%s: frequencies is NULL", what);
    std::vector<double> turns(desc->rotary_dim / 2);
    for (size_t i = 0; i < turns.size(); ++i) {
      // (2^31 positions of it stay within the 52 bits of a product)
      if (!(std::fabs(desc->frequencies[i]) <= 64.0))
        return set_err(err, "%s: frequencies[%zu] must be a number of at most 64", what, i);
      turns[i] = (double)((long double)desc->frequencies[i] / 6.283185307179586476925286766559L);
    }
    if (rt == nullptr || out == nullptr) return set_err(err, "%s: NULL argument", what);
    OnDevice on(rt->device);
    if (rt->load(eoship::Runtime::kStep, err) != 0) return 1;
    auto* rot = new EosHipRotary();
    rot->rt = rt;
    rot->head_dim = desc->head_dim;
    rot->rotary_dim = desc->rotary_dim;
    rot->layout = desc->layout;
    rot->factor = desc->factor;
    void* mem = nullptr;
    if (rt->alloc(turns.size() * sizeof(double), &mem, err) != 0) {
      delete rot;
      return 1;
    }
    rot->turns = static_cast<double*>(mem);
    const hipError_t e =
        rt->copy_sync(mem, turns.data(), turns.size() * sizeof(double), hipMemcpyHostToDevice);
    if (e != hipSuccess) {
      delete rot;
      return hip_err(err, "hipMemcpy(frequencies)", e);
    }
    *out = rot;
    return 0;
  });
}

int eoship_rotary_release(EosHipRuntime* rt, EosHipRotary* rot, char** err) {
  if (rot == nullptr) return 0;
  if (rt == nullptr || rot->rt != rt) return set_err(err, "eoship_rotary_release: wrong runtime");
  OnDevice on(rt->device);
  if (rt->sync(err) != 0) return 1;
  delete rot;
  return 0;
}

int eoship_rotary_device(EosHipRuntime* rt, EosHipRotary* rot, const EosHipKVBatch* batch,
                         const int32_t* d_positions, int64_t rows, int32_t inverse, int32_t dtype,
                         const void* d_q, int64_t q_stride, int32_t heads, void* d_q_out,
                         int64_t q_out_stride, const void* d_k, int64_t k_stride, int32_t kv_heads,
                         void* d_k_out, int64_t k_out_stride, char** err) {
  const char* what = "eoship_rotary_device";
  return guarded(what, err, [&]() -> int {
    if (rt == nullptr || rot == nullptr) return set_err(err, "%s: NULL argument", what);
    if (rot->rt != rt) return set_err(err, "%s: bound to another runtime", what);
    if ((batch == nullptr) == (d_positions == nullptr))
      return set_err(err, "%s: either a batch or positions", what);
    if (dtype < kRotF16 || dtype > kRotF32)
      return set_err(err, "%s: dtype must be 0 (f16), 1 (bf16) or 2 (f32), got %d", what, dtype);
    if (heads < 0 || heads > 65535 || kv_heads < 0 || kv_heads > 65535 || heads + kv_heads == 0)
      return set_err(err, "%s: heads and kv_heads must be in 0..65535, not both 0", what);
    RotArgs a{};
    a.rows = rows;
    a.positions = d_positions;
    if (batch != nullptr) {
      a.rows = batch->rows;
      a.batch = batch->batch;
      a.lengths = batch->d_lengths;
      a.offsets = batch->d_offsets;
      if (batch->batch < 0) return set_err(err, "%s: negative batch", what);
      if (batch->batch == 0) a.rows = std::min<int64_t>(a.rows, 0);
      if (a.rows > 0 && a.lengths == nullptr) return set_err(err, "%s: NULL lengths", what);
      if (a.rows > 0 && a.offsets == nullptr && a.rows != a.batch)
        return set_err(err, "%s: without offsets every sequence has one row: rows %lld, batch %d",
                       what, (long long)a.rows, a.batch);
    }
    if (a.rows < 0 || a.rows > INT32_MAX)
      return set_err(err, "%s: rows must be in 0..2^31-1, got %lld", what, (long long)a.rows);
    if (a.rows == 0) return 0;
    if ((((uintptr_t)d_positions | (uintptr_t)a.lengths | (uintptr_t)a.offsets) & 3) != 0)
      return set_err(err, "%s: positions, lengths and offsets must be 4-byte aligned", what);
    const int64_t d = rot->head_dim;
    if (heads > 0 && (check_rows(d_q, q_stride, heads * d, "q", what, err) != 0 ||
                      check_rows(d_q_out, q_out_stride, heads * d, "q_out", what, err) != 0))
      return 1;
    if (kv_heads > 0 && (check_rows(d_k, k_stride, kv_heads * d, "k", what, err) != 0 ||
                         check_rows(d_k_out, k_out_stride, kv_heads * d, "k_out", what, err) != 0))
      return 1;
    if ((heads > 0 && d_q == d_q_out && q_stride != q_out_stride) ||
        (kv_heads > 0 && d_k == d_k_out && k_stride != k_out_stride))
      return set_err(err, "%s: rows turned in place keep their stride", what);
    const int size = dtype == kRotF32 ? 4 : 2;
    const auto rows_at = [&](const void* p, int64_t stride, int n) {
      return rows_of(p, n > 0 ? a.rows : 0, stride * size, n * d * size);
    };
    const Rows q = rows_at(d_q, q_stride, heads), q_out = rows_at(d_q_out, q_out_stride, heads);
    const Rows k = rows_at(d_k, k_stride, kv_heads), k_out = rows_at(d_k_out, k_out_stride, kv_heads);
    if (d_q != d_q_out && rows_meet(q_out, q)) return set_err(err, "%s: q_out overlaps q", what);
    if (d_k != d_k_out && rows_meet(k_out, k)) return set_err(err, "%s: k_out overlaps k", what);
    if (d_k != d_k_out && rows_meet(q_out, k)) return set_err(err, "%s: q_out overlaps k", what);
    if (d_q != d_q_out && rows_meet(k_out, q)) return set_err(err, "%s: k_out overlaps q", what);
    if (rows_meet(q_out, k_out)) return set_err(err, "%s: q_out overlaps k_out", what);
    const Rows read[] = {bytes_of(d_positions, d_positions != nullptr ? 4 * a.rows : 0),
                         bytes_of(a.lengths, a.lengths != nullptr ? 4LL * a.batch : 0),
                         bytes_of(a.offsets, a.offsets != nullptr ? 4LL * a.batch + 4 : 0)};
    for (const Rows& r : read)
      if (rows_meet(q_out, r) || rows_meet(k_out, r))
        return set_err(err, "%s: an output overlaps positions, lengths or offsets", what);
    OnDevice on(rt->device);
    a.q = static_cast<const uint8_t*>(d_q);
    a.k = static_cast<const uint8_t*>(d_k);
    a.q_out = static_cast<uint8_t*>(d_q_out);
    a.k_out = static_cast<uint8_t*>(d_k_out);
    a.q_stride = q_stride * size;
    a.k_stride = k_stride * size;
    a.q_out_stride = q_out_stride * size;
    a.k_out_stride = k_out_stride * size;
    a.turns = rot->turns;
    a.heads = heads;
    a.kv_heads = kv_heads;
    a.head_dim = rot->head_dim;
    a.rotary_dim = rot->rotary_dim;
    a.layout = rot->layout;
    a.factor = rot->factor;
    a.sign = inverse != 0 ? -1.0f : 1.0f;
    const int half = rot->rotary_dim / 2;
    // Eight values at a time where both halves, or all pairs, begin at such.
    const bool wide = half % (rot->layout == kRotHalves ? 8 : 4) == 0;
    const int lanes = !wide ? 64
                      : rot->layout == kRotHalves ? half / 8 + (rot->head_dim - rot->rotary_dim) / 8
                                                  : rot->head_dim / 8;
    while ((1 << a.lanes_shift) < lanes) ++a.lanes_shift;
    // A workgroup computes up to 256 angles at once, of as many rows; of fewer
    // where there are not rows enough for every CU.
    const long long most = std::max(1, std::min(kRotAngles / half, kRotRows));
    a.each = (int)std::max(1LL, std::min(most, a.rows / (4 * rt->compute_units)));
    const long long blocks = (a.rows + a.each - 1) / a.each, groups = (1 << 24) - 1;
    if (blocks > groups)
      return set_err(err, "%s: %lld rows are more than %lld rows of one call", what,
                     (long long)a.rows, groups * most);
    const std::string name = std::string(rot->layout == kRotHalves ? "eos_rot_halves_" : "eos_rot_pairs_") +
                             (wide ? "" : "odd_") + kTypes[dtype];
    return rt->launch(name.c_str(), dim3((unsigned)blocks), dim3(256), 0, &a, err);
  });
}

}  // extern "C"
