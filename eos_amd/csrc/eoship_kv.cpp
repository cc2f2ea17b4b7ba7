// Key-value cache half of the eoship C ABI: binds a caller's paged cache and
// enqueues its writes, reads and attention. The counterpart of the kv_cache
// capability that the reference's CUDA backend advertises
// (runtime/backend/backend.go:1428-1431), with the Hadamard TurboQuant
// quantizer (runtime/backends/cuda/native_linux.go:1812-2004) as one of its
// storage formats.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <string>
#include <vector>

#include "eoship_internal.h"
#include "kernels/kv_index.h"

using eoship::guarded;
using eoship::hip_err;
using eoship::OnDevice;
using eoship::set_err;

struct EosHipKVCache {
  EosHipRuntime* rt = nullptr;
  EosHipKVDesc d{};
  KvTables tables{};
  int page_shift = 0;
  void* mem = nullptr;  // status word, then the signs
  ~EosHipKVCache() {
    if (mem != nullptr) hipFree(mem);
  }
};

namespace {

// Query rows a sequence (heads of a group counted) from which the prompt
// kernel takes a call, by format. Below, 16 rows at a time, each wavefront with
// keys of its own, are faster: the prompt kernel's stage has a latency of its
// own, and quantized stages are expanded by few wavefronts. 8 sequences, heads
// 32 to 8 of 128, us (16 rows / 128 rows at a time): behind 8,000 keys bf16 2
// rows each 65 / 59, 8 rows 116 / 66; q8 8 rows 65 / 96, 16 rows 107 / 119;
// behind 2,000 keys q8 32 rows 58 / 56, 128 rows 124 / 104; tq4 32 rows 52 /
// 71, 128 rows 133 / 128.
constexpr int kPromptFrom[] = {8, 8, 96, 384};
// ... and not while the 16-row workgroups are on the CUs at once over so few
// keys (4 prompts of 256, 8 heads of 64: 10 / 17). Here and for the equal shares
// below, keys are those that the page table has room for: lengths are on the
// device, so short sequences under a wide table take the kernels of long ones.
constexpr int kPromptKeys = 1024;

const char* const kFormats[] = {"f16", "bf16", "q8", "tq4"};

bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

int bits_of(int format) { return format == kKvQ8 ? 8 : format == kKvTq4 ? 4 : 16; }

// The f16 bits of a float that f16 holds exactly and normally, or 0.
uint16_t exact_f16(float f) {
  uint32_t u;
  std::memcpy(&u, &f, 4);
  const int ex = (int)(u >> 23 & 255) - 127;
  if ((u & 0x1fff) != 0 || ex < -14 || ex > 15) return 0;
  return (uint16_t)((u >> 31) << 15 | (uint32_t)(ex + 15) << 10 | (u >> 13 & 0x3ff));
}

int check_desc(const EosHipKVDesc* d, const char* what, char** err) {
  if (d == nullptr) return set_err(err, "%s: desc is NULL", what);
  if (d->format < kKvF16 || d->format > kKvTq4)
    return set_err(err, "%s: format must be 0 (f16), 1 (bf16), 2 (q8) or 3 (tq4), got %d", what,
                   d->format);
  if (d->kv_heads < 1 || d->kv_heads > 1024)
    return set_err(err, "%s: kv_heads must be in 1..1024, got %d", what, d->kv_heads);
  if (d->head_dim != 32 && d->head_dim != 64 && d->head_dim != 128 && d->head_dim != 256)
    return set_err(err, "%s: head_dim must be 32, 64, 128 or 256, got %d", what, d->head_dim);
  const int p = d->page_tokens;
  if (p < 16 || p > 256 || (p & (p - 1)) != 0)
    return set_err(err, "%s: page_tokens must be 16, 32, 64, 128 or 256, got %d", what, p);
  if (d->pages < 1 || d->pages > INT32_MAX)
    return set_err(err, "%s: pages must be in 1..2^31-1, got %lld", what, (long long)d->pages);
  return 0;
}

int check_tables(const EosHipKVDesc* d, const char* what, char** err) {
  if (d->format != kKvTq4) return 0;
  if (d->codebook == nullptr || d->signs == nullptr)
    return set_err(err, "%s: tq4 needs a codebook and signs", what);
  for (int i = 0; i < 8; ++i) {
    if (!(d->codebook[i] > 0.0f) || exact_f16(d->codebook[i]) == 0)
      return set_err(err, "%s: codebook[%d] must be a positive f16 number", what, i);
    if (i > 0 && d->codebook[i] <= d->codebook[i - 1])
      return set_err(err, "%s: codebook must be ascending", what);
  }
  for (int i = 0; i < d->head_dim; ++i)
    if (d->signs[i] != 1.0f && d->signs[i] != -1.0f)
      return set_err(err, "%s: signs must be 1 or -1", what);
  return 0;
}

int check_batch(const EosHipRuntime* rt, const EosHipKVCache* kv, const EosHipKVBatch* b,
                const char* what, char** err) {
  if (rt == nullptr || kv == nullptr || b == nullptr)
    return set_err(err, "%s: NULL argument", what);
  if (kv->rt != rt) return set_err(err, "%s: the cache is bound to another runtime", what);
  if (b->batch < 0 || b->rows < 0) return set_err(err, "%s: negative batch or rows", what);
  if (b->rows > INT32_MAX) return set_err(err, "%s: more than 2^31-1 rows", what);
  if (b->batch == 0 || b->rows == 0) return 0;
  if (b->d_page_table == nullptr || b->d_lengths == nullptr)
    return set_err(err, "%s: NULL page table or lengths", what);
  if (b->table_stride < 1) return set_err(err, "%s: table_stride must be positive", what);
  if (b->d_offsets == nullptr && b->rows != b->batch)
    return set_err(err, "%s: without offsets every sequence has one row: rows %lld, batch %d",
                   what, (long long)b->rows, b->batch);
  return 0;
}

int check_rows(const void* p, int64_t stride, int64_t width, const char* name, const char* what,
               char** err) {
  if (p == nullptr) return set_err(err, "%s: %s is NULL", what, name);
  if (!aligned(p)) return set_err(err, "%s: %s is not 16-byte aligned", what, name);
  if (stride < width || stride % 8 != 0)
    return set_err(err, "%s: the row stride of %s must be a multiple of 8 and at least %lld, got %lld",
                   what, name, (long long)width, (long long)stride);
  return 0;
}

KvCacheArgs cache_args(const EosHipKVCache* kv, const EosHipKVBatch* b) {
  KvCacheArgs c{};
  c.k = static_cast<uint8_t*>(kv->d.d_k);
  c.v = static_cast<uint8_t*>(kv->d.d_v);
  c.k_scale = kv->d.d_k_scale;
  c.v_scale = kv->d.d_v_scale;
  c.table = b->d_page_table;
  c.lengths = b->d_lengths;
  c.offsets = b->d_offsets;
  c.status = static_cast<int32_t*>(kv->mem);
  c.t = kv->tables;
  c.rows = b->rows;
  c.pages = (int)kv->d.pages;
  c.kv_heads = kv->d.kv_heads;
  c.page_shift = kv->page_shift;
  c.table_stride = b->table_stride;
  c.batch = b->batch;
  return c;
}

int launch(EosHipRuntime* rt, const EosHipKVCache* kv, const char* op, long long gx, int gy,
           int threads, void* args, const char* what, char** err) {
  if (gx * threads > UINT32_MAX)
    return set_err(err, "%s: too many rows for one call", what);
  char name[64];
  snprintf(name, sizeof(name), "eos_kv_%s_%s_%d", op, kFormats[kv->d.format], kv->d.head_dim);
  return rt->launch(name, dim3((unsigned)gx, (unsigned)gy), dim3((unsigned)threads), 0, args, err);
}

int rows_call(EosHipRuntime* rt, const EosHipKVCache* kv, const EosHipKVBatch* b, const void* d_k,
              int64_t k_stride, const void* d_v, int64_t v_stride, int32_t dtype, const char* op,
              const char* what, char** err) {
  const int64_t width = (int64_t)kv->d.kv_heads * kv->d.head_dim;
  if (check_rows(d_k, k_stride, width, "k", what, err) != 0 ||
      check_rows(d_v, v_stride, width, "v", what, err) != 0)
    return 1;
  OnDevice on(rt->device);
  KvRowsArgs a{};
  a.c = cache_args(kv, b);
  a.k = static_cast<uint8_t*>(const_cast<void*>(d_k));
  a.v = static_cast<uint8_t*>(const_cast<void*>(d_v));
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.dtype = dtype;
  if (b->d_offsets == nullptr) {
    const std::string one = std::string(op) + "1";
    return launch(rt, kv, one.c_str(), b->batch, kv->d.kv_heads, 2 * kv->d.head_dim, &a, what, err);
  }
  return launch(rt, kv, op, kv_units(b->rows, b->batch, 1, kKvRun, 2), kv->d.kv_heads,
                kv->d.format == kKvTq4 ? 256 : 2 * kv->d.head_dim, &a, what, err);
}

}  // namespace

extern "C" {

int eoship_kv_bytes(const EosHipKVDesc* desc, int64_t* pool_bytes, int64_t* scale_bytes,
                    char** err) {
  const char* what = "eoship_kv_bytes";
  if (check_desc(desc, what, err) != 0) return 1;
  const int64_t tokens = desc->pages * desc->kv_heads * desc->page_tokens;
  if (pool_bytes) *pool_bytes = tokens * (desc->head_dim * bits_of(desc->format) / 8);
  if (scale_bytes) *scale_bytes = desc->format >= kKvQ8 ? tokens * 4 : 0;
  return 0;
}

int eoship_kv_check_batch(const EosHipKVDesc* desc, const int32_t* page_table,
                          int32_t table_stride, int32_t batch, const int32_t* lengths,
                          const int32_t* offsets, int64_t rows, int32_t writes, char** err) {
  return eoship_kv_check_batch_window(desc, page_table, table_stride, batch, lengths, offsets, rows,
                                      0, writes, err);
}

int eoship_kv_check_batch_window(const EosHipKVDesc* desc, const int32_t* page_table,
                                 int32_t table_stride, int32_t batch, const int32_t* lengths,
                                 const int32_t* offsets, int64_t rows, int32_t window,
                                 int32_t writes, char** err) {
  const char* what = "eoship_kv_check_batch";
  return guarded(what, err, [&]() -> int {
    if (check_desc(desc, what, err) != 0) return 1;
    if (window < 0) return set_err(err, "%s: window must not be negative, got %d", what, window);
    if (batch < 0 || rows < 0 || rows > INT32_MAX)
      return set_err(err, "%s: batch and rows must be in 0..2^31-1", what);
    if (batch == 0 || rows == 0) return 0;
    if (page_table == nullptr || lengths == nullptr || table_stride < 1)
      return set_err(err, "%s: NULL page table or lengths, or no table columns", what);
    if (offsets == nullptr && rows != batch)
      return set_err(err, "%s: without offsets every sequence has one row: rows %lld, batch %d",
                     what, (long long)rows, batch);
    if (offsets != nullptr && offsets[0] != 0)
      return set_err(err, "%s: offsets[0] must be 0, got %d", what, offsets[0]);
    KvCacheArgs c{};
    c.table = page_table;
    c.lengths = lengths;
    c.offsets = offsets;
    c.rows = rows;
    c.pages = (int)desc->pages;
    c.table_stride = table_stride;
    c.batch = batch;
    while ((1 << c.page_shift) < desc->page_tokens) ++c.page_shift;
    // Where a page is written: the sequence, and which of its pages.
    std::vector<std::pair<int, std::pair<int, int>>> written;
    for (int b = 0; b < batch; ++b) {
      const KvSeq s = kv_seq(c, b);
      if (s.bad & kKvBadOffset)
        return set_err(err, "%s: sequence %d: offsets must ascend within 0..rows", what, b);
      if (s.bad & kKvBadLength)
        return set_err(err, "%s: sequence %d: length %d outside 0..%lld of its table row", what, b,
                       lengths[b], (long long)table_stride * desc->page_tokens);
      // (the first row's window reaches furthest back)
      const int from = window == 0 ? 0 : s.n == 0 ? s.keys : (int)std::max(0LL, (long long)s.len - s.n - window + 1);
      for (int i = from >> c.page_shift; from < s.keys && i << c.page_shift < s.keys; ++i)
        if (kv_page(c, b, i << c.page_shift) < 0)
          return set_err(err, "%s: sequence %d: page %d of its table row is %d, not in 0..%lld", what,
                         b, i, page_table[(size_t)b * table_stride + i], (long long)desc->pages - 1);
      if (writes != 0 && s.n > 0 && s.keys > 0)
        for (int i = std::max(0, s.len - s.n) >> c.page_shift; i <= (s.keys - 1) >> c.page_shift; ++i)
          written.push_back({page_table[(size_t)b * table_stride + i], {b, i}});
    }
    std::sort(written.begin(), written.end());
    for (size_t i = 1; i < written.size(); ++i)
      if (written[i].first == written[i - 1].first)
        return set_err(err, "%s: page %d is written twice, by sequences %d and %d", what,
                       written[i].first, written[i - 1].second.first, written[i].second.first);
    return 0;
  });
}

int eoship_kv_bind(EosHipRuntime* rt, const EosHipKVDesc* desc, EosHipKVCache** out, char** err) {
  const char* what = "eoship_kv_bind";
  return guarded(what, err, [&]() -> int {
    if (out != nullptr) *out = nullptr;
    if (check_desc(desc, what, err) != 0 || check_tables(desc, what, err) != 0) return 1;
    if (desc->d_k == nullptr || desc->d_v == nullptr)
      return set_err(err, "%s: NULL pool", what);
    if (!aligned(desc->d_k) || !aligned(desc->d_v))
      return set_err(err, "%s: pools must be 16-byte aligned", what);
    if (desc->format >= kKvQ8 &&
        (desc->d_k_scale == nullptr || desc->d_v_scale == nullptr || !aligned(desc->d_k_scale) ||
         !aligned(desc->d_v_scale)))
      return set_err(err, "%s: %s needs 16-byte aligned scale pools", what, kFormats[desc->format]);
    if (rt == nullptr || out == nullptr) return set_err(err, "%s: NULL argument", what);
    OnDevice on(rt->device);
    if (rt->load(eoship::Runtime::kKv, err) != 0) return 1;
    auto* kv = new EosHipKVCache();
    kv->rt = rt;
    kv->d = *desc;
    while ((1 << kv->page_shift) < desc->page_tokens) ++kv->page_shift;
    const size_t signs = desc->format == kKvTq4 ? (size_t)desc->head_dim * 4 : 0;
    std::vector<char> host(16 + signs, 0);
    if (rt->alloc(host.size(), &kv->mem, err) != 0) {
      delete kv;
      return 1;
    }
    if (desc->format == kKvTq4) {
      std::memcpy(host.data() + 16, desc->signs, signs);
      KvTables& t = kv->tables;
      t.signs = reinterpret_cast<const float*>(static_cast<char*>(kv->mem) + 16);
      for (int i = 0; i < 8; ++i) {
        const uint32_t u = exact_f16(desc->codebook[i]);
        t.mags[i] = desc->codebook[i];
        t.hi[i / 4] |= (u >> 8) << (8 * (i % 4));
        t.lo[i / 4] |= (u & 255) << (8 * (i % 4));
        if (i > 0) t.edges[i - 1] = 0.5f * (desc->codebook[i] + desc->codebook[i - 1]);
      }
    }
    kv->d.codebook = kv->d.signs = nullptr;  // the caller's host memory is not kept
    const hipError_t e = rt->copy_sync(kv->mem, host.data(), host.size(), hipMemcpyHostToDevice);
    if (e != hipSuccess) {
      delete kv;
      return hip_err(err, "hipMemcpy(cache tables)", e);
    }
    *out = kv;
    return 0;
  });
}

int eoship_kv_release(EosHipRuntime* rt, EosHipKVCache* kv, char** err) {
  if (kv == nullptr) return 0;
  if (rt == nullptr || kv->rt != rt) return set_err(err, "eoship_kv_release: wrong runtime");
  OnDevice on(rt->device);
  if (rt->sync(err) != 0) return 1;
  delete kv;
  return 0;
}

int eoship_kv_append_device(EosHipRuntime* rt, EosHipKVCache* kv, const EosHipKVBatch* batch,
                            const void* d_k, int64_t k_stride, const void* d_v, int64_t v_stride,
                            int32_t dtype, char** err) {
  const char* what = "eoship_kv_append_device";
  return guarded(what, err, [&]() -> int {
    if (check_batch(rt, kv, batch, what, err) != 0) return 1;
    if (dtype != kKvRowF16 && dtype != kKvRowBf16)
      return set_err(err, "%s: rows must be f16 (0) or bf16 (1), got %d", what, dtype);
    if (kv->d.format <= kKvBf16 && dtype != kv->d.format)
      return set_err(err, "%s: the cache holds %s, the rows are %s", what, kFormats[kv->d.format],
                     kFormats[dtype]);
    if (batch->batch == 0 || batch->rows == 0) return 0;
    return rows_call(rt, kv, batch, d_k, k_stride, d_v, v_stride, dtype, "append", what, err);
  });
}

int eoship_kv_read_device(EosHipRuntime* rt, EosHipKVCache* kv, const EosHipKVBatch* batch,
                          void* d_k, int64_t k_stride, void* d_v, int64_t v_stride, int32_t dtype,
                          char** err) {
  const char* what = "eoship_kv_read_device";
  return guarded(what, err, [&]() -> int {
    if (check_batch(rt, kv, batch, what, err) != 0) return 1;
    if (dtype < kKvRowF16 || dtype > kKvRowF32)
      return set_err(err, "%s: rows must be f16 (0), bf16 (1) or f32 (2), got %d", what, dtype);
    if (batch->batch == 0 || batch->rows == 0) return 0;
    return rows_call(rt, kv, batch, d_k, k_stride, d_v, v_stride, dtype, "read", what, err);
  });
}

int eoship_kv_attention_device(EosHipRuntime* rt, EosHipKVCache* kv, const EosHipKVBatch* batch,
                               const void* d_q, int64_t q_stride, int32_t heads, int32_t dtype,
                               float scale, int32_t window, void* d_out, int64_t out_stride,
                               float* d_lse, char** err) {
  const char* what = "eoship_kv_attention_device";
  return guarded(what, err, [&]() -> int {
    if (check_batch(rt, kv, batch, what, err) != 0) return 1;
    if (dtype != kKvRowF16 && dtype != kKvRowBf16)
      return set_err(err, "%s: rows must be f16 (0) or bf16 (1), got %d", what, dtype);
    if (kv->d.format <= kKvBf16 && dtype != kv->d.format)
      return set_err(err, "%s: the cache holds %s, the rows are %s", what, kFormats[kv->d.format],
                     kFormats[dtype]);
    if (heads < 1 || heads > 65535 || heads % kv->d.kv_heads != 0)
      return set_err(err, "%s: heads must be a multiple of kv_heads (%d) up to 65535, got %d", what,
                     kv->d.kv_heads, heads);
    if (!std::isfinite(scale)) return set_err(err, "%s: scale must be finite", what);
    if (window < 0) return set_err(err, "%s: window must not be negative, got %d", what, window);
    if (batch->batch == 0 || batch->rows == 0) return 0;
    if (batch->rows * (heads / kv->d.kv_heads) > 1 << 30)
      return set_err(err, "%s: too many rows for one call", what);
    const int64_t width = (int64_t)heads * kv->d.head_dim;
    if (check_rows(d_q, q_stride, width, "q", what, err) != 0 ||
        check_rows(d_out, out_stride, width, "out", what, err) != 0)
      return 1;
    OnDevice on(rt->device);
    KvAttnArgs a{};
    a.c = cache_args(kv, batch);
    a.q = static_cast<const uint8_t*>(d_q);
    a.out = static_cast<uint8_t*>(d_out);
    a.lse = d_lse;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.scale = scale * 1.44269504089f;
    a.heads = heads;
    a.group = heads / kv->d.kv_heads;
    a.window = window;
    a.dtype = dtype;
    const int kvh = kv->d.kv_heads, d = kv->d.head_dim;
    // A window that holds the whole table restricts nothing.
    if (window >= std::min<long long>((long long)batch->table_stride << kv->page_shift, kKvMostKeys))
      a.window = window = 0;
    const long long slots = 2LL * rt->compute_units;  // two workgroups a CU, by their registers
    long long keys = (long long)batch->table_stride << kv->page_shift;
    if (window > 0) keys = std::min(keys, (long long)window + batch->rows + 32);
    const auto tiles = [&](int rows) {
      return batch->d_offsets == nullptr ? (long long)batch->batch * ((a.group + rows - 1) / rows)
                                         : kv_units(batch->rows, batch->batch, a.group, rows, 1);
    };
    const int64_t from = kPromptFrom[kv->d.format];
    const bool prompt = batch->d_offsets != nullptr && batch->rows * a.group >= from * batch->batch &&
                        (tiles(kKvTileRows) * kvh > slots || keys > kPromptKeys);
    a.tile_rows = prompt ? kKvPromptRows : kKvTileRows;
    a.tiles = tiles(a.tile_rows);
    // Splits while the workgroups are on the CUs at once, none below 256 keys:
    // further ones cost more in prologues and joining than their balance gains
    // (64 x 2,000 tokens of tq4: 39 us at two workgroups a CU, 53 at four, 68 at
    // eight). Prompts, whose joins are few, fill the last slots too (8 x 128 rows
    // behind 2,000 keys in q8: 104 us, 156 without).
    const long long units = a.tiles * kvh;
    const long long want = prompt ? (slots + units - 1) / units : slots / units;
    a.splits = (int)std::max(1LL, std::min(want, (keys + 255) / 256));
    // Several sequences with room for enough keys: equal shares of all of them
    // instead, whatever the lengths. 64 sequences of 1,024 to 16,384 tokens in
    // tq4: 164 us, in splits 230; of 2,000 tokens each 46 and 39; 32 of 64 to
    // 4,096 in bf16: 66 and 79. Many workgroups balance by themselves (256
    // sequences of 1,000: 206 in shares, 185 in splits), few keys do not pay for
    // the prefix sum (4 of up to 3,000: 21 and 16), and more sequences lose to it
    // what balance gains, in the smaller formats sooner (one head, 64 to 4,096
    // tokens: 300 of bf16 77 and 116, 500 of bf16 114 and 135, 900 of f16 190 and
    // 202, but of 2,000 each 185 and 170; 300 of q8 51 and 54, 500 of q8 74 and
    // 63; 300 of tq4 51 and 60, 400 of tq4 65 and 58, 300 of 2,000 each 43 and 37).
    const long long steps = ((long long)batch->table_stride << kv->page_shift) / 128;
    const int most = kv->d.format <= kKvBf16 ? kKvStreamBatch : kKvStreamBatch / 2;
    if (batch->d_offsets == nullptr && batch->batch > 1 && batch->batch <= most &&
        units < 4 * slots && steps * units >= 4 * slots) {
      a.workgroups = (int)slots;
      const size_t parts = (size_t)a.workgroups * 2 * kKvTileRows;
      void* ws = nullptr;
      if (rt->workspace(parts * (size_t)(d + 2) * 4, &ws, err) != 0) return 1;
      a.part = static_cast<float*>(ws);
      a.part_ml = a.part + parts * (size_t)d;
      if (launch(rt, kv, "stream", a.workgroups, 1, 256, &a, what, err) != 0) return 1;
      return launch(rt, kv, "stream_join", batch->batch, heads, 256, &a, what, err);
    }
    if (a.splits > 1) {
      const size_t parts = (size_t)units * a.splits * a.tile_rows;
      void* ws = nullptr;
      if (rt->workspace(parts * (size_t)(d + 2) * 4, &ws, err) != 0) return 1;
      a.part = static_cast<float*>(ws);
      a.part_ml = a.part + parts * (size_t)d;
    }
    const long long items = a.tiles * a.splits;
    if (prompt ? launch(rt, kv, "prompt", kv_place_blocks(kvh, items), 1, 256, &a, what, err) != 0
               : launch(rt, kv, "split", items, kvh, 256, &a, what, err) != 0)
      return 1;
    if (a.splits == 1) return 0;
    if (a.splits <= kKvFewSplits) {
      const int each = 256 / (d / 8);
      return launch(rt, kv, "join_few", batch->rows, (heads + each - 1) / each, 256, &a, what, err);
    }
    return launch(rt, kv, "join", batch->rows, heads, 256, &a, what, err);
  });
}

int eoship_kv_status(EosHipRuntime* rt, EosHipKVCache* kv, int32_t* status, char** err) {
  const char* what = "eoship_kv_status";
  if (rt == nullptr || kv == nullptr || status == nullptr)
    return set_err(err, "%s: NULL argument", what);
  if (kv->rt != rt) return set_err(err, "%s: the cache is bound to another runtime", what);
  OnDevice on(rt->device);
  hipError_t e = rt->copy_async(status, kv->mem, 4, hipMemcpyDeviceToHost);
  if (e != hipSuccess) return hip_err(err, what, e);
  if (rt->sync(err) != 0) return 1;
  if (*status == 0) return 0;
  const int32_t zero = 0;
  e = rt->copy_async(kv->mem, &zero, 4, hipMemcpyHostToDevice);
  if (e != hipSuccess) return hip_err(err, what, e);
  return rt->sync(err);
}

}  // extern "C"
