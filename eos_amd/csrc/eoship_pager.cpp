// Page tables half of the eoship C ABI: which pages of a key-value cache the
// requests of a server hold, planned on the device from their lengths. Goes
// with the paged cache (the kv_cache capability, runtime/backend/backend.go:
// 1428-1431); the reference plans its buffers on the host.
#include <algorithm>
#include <cstdint>
#include <string>

#include "eoship_internal.h"
#include "kernels/step_args.h"

using eoship::guarded;
using eoship::hip_err;
using eoship::OnDevice;
using eoship::set_err;

struct EosHipKVPager {
  EosHipRuntime* rt = nullptr;
  EosHipKVPagerDesc d{};
  int page_shift = 0;
  void* mem = nullptr;  // status, workgroups done
  ~EosHipKVPager() {
    if (mem != nullptr) hipFree(mem);
  }
};

namespace {

constexpr int kThreads = 1024;

bool aligned(const void* p, int n) { return ((uintptr_t)p & (n - 1)) == 0; }

int check_desc(const EosHipKVPagerDesc* d, const char* what, char** err) {
  if (d == nullptr) return set_err(err, "%s: desc is NULL", what);
  if (d->slots < 1 || d->slots > kPagerSlots)
    return set_err(err, "%s: slots must be in 1..%d, got %d", what, kPagerSlots, d->slots);
  if (d->table_stride < 1 || d->table_stride > 1 << 26)
    return set_err(err, "%s: table_stride must be in 1..2^26, got %d", what, d->table_stride);
  const int p = d->page_tokens;
  if (p < 16 || p > 256 || (p & (p - 1)) != 0)
    return set_err(err, "%s: page_tokens must be 16, 32, 64, 128 or 256, got %d", what, p);
  if (d->pages < 1 || d->pages > INT32_MAX)
    return set_err(err, "%s: pages must be in 1..2^31-1, got %lld", what, (long long)d->pages);
  if (d->d_page_table == nullptr || d->d_lengths == nullptr || d->d_free == nullptr ||
      d->d_free_count == nullptr)
    return set_err(err, "%s: NULL page table, lengths, free pages or their count", what);
  if (!aligned(d->d_page_table, 4) || !aligned(d->d_lengths, 4) || !aligned(d->d_free, 4) ||
      !aligned(d->d_free_count, 4))
    return set_err(err, "%s: arrays must be 4-byte aligned", what);
  return 0;
}

int check(const EosHipRuntime* rt, const EosHipKVPager* pager, const char* what, char** err) {
  if (rt == nullptr || pager == nullptr) return set_err(err, "%s: NULL argument", what);
  if (pager->rt != rt) return set_err(err, "%s: the pager is bound to another runtime", what);
  return 0;
}

// An array's bytes, none where it is not given.
struct Span {
  uintptr_t at, end;
  Span(const void* p, int64_t bytes) : at((uintptr_t)p), end((uintptr_t)p + (p != nullptr ? bytes : 0)) {}
};
// (an empty one meets none)
bool meet(const Span& a, const Span& b) { return std::max(a.at, b.at) < std::min(a.end, b.end); }

// A pager's arrays.
struct Arrays {
  Span table, free, lengths, count;
  explicit Arrays(const EosHipKVPagerDesc& d)
      : table(d.d_page_table, 4LL * d.slots * d.table_stride), free(d.d_free, 4 * d.pages),
        lengths(d.d_lengths, 4LL * d.slots), count(d.d_free_count, 4) {}
};

PagerArgs args(const EosHipKVPager* p) {
  PagerArgs a{};
  a.table = p->d.d_page_table;
  a.lengths = p->d.d_lengths;
  a.free_list = p->d.d_free;
  a.free_count = p->d.d_free_count;
  a.state = static_cast<int32_t*>(p->mem);
  a.pages = p->d.pages;
  a.slots = p->d.slots;
  a.stride = p->d.table_stride;
  a.page_shift = p->page_shift;
  return a;
}

// Every wavefront sums up to 64 slots up by itself, a workgroup 1,024, a slot a
// thread, or 4,096. Workgroups: two table entries or rows a thread, on every CU at
// most (extend and trim, 64 slots of 128 pages: 1 workgroup 6.6 + 4.0 us, 4 5.2 +
// 3.8, 64 4.9 + 3.9, 256 6.8 + 5.6; 4,096 slots of 512: 64 38.7 + 9.6, 128 25.3 +
// 8.6, 256 18.5 + 7.6, 512 24.8 + 9.3).
int launch(EosHipRuntime* rt, const EosHipKVPager* p, const char* op, long long rows, size_t lds,
           PagerArgs* a, char** err) {
  const std::string name = std::string("eos_pager_") + op +
                           (a->slots <= kPagerFew ? "_few" : a->slots <= kThreads ? "_some" : "_many");
  const long long work = std::max((long long)a->slots * a->stride, rows);
  const long long blocks = std::max(1LL, std::min<long long>(rt->compute_units, work / (2 * kThreads)));
  return rt->launch(name.c_str(), dim3((unsigned)blocks), dim3(kThreads), lds, a, err);
}

}  // namespace

extern "C" {

int eoship_kv_pager_bind(EosHipRuntime* rt, const EosHipKVPagerDesc* desc, EosHipKVPager** out,
                         char** err) {
  const char* what = "eoship_kv_pager_bind";
  return guarded(what, err, [&]() -> int {
    if (out != nullptr) *out = nullptr;
    if (check_desc(desc, what, err) != 0) return 1;
    if (rt == nullptr || out == nullptr) return set_err(err, "%s: NULL argument", what);
    const Arrays own(*desc);
    if (meet(own.table, own.free) || meet(own.table, own.lengths) || meet(own.table, own.count) ||
        meet(own.free, own.lengths) || meet(own.free, own.count) || meet(own.lengths, own.count))
      return set_err(err, "%s: arrays overlap", what);
    OnDevice on(rt->device);
    if (rt->load(eoship::Runtime::kStep, err) != 0) return 1;
    auto* p = new EosHipKVPager();
    p->rt = rt;
    p->d = *desc;
    while ((1 << p->page_shift) < desc->page_tokens) ++p->page_shift;
    if (rt->alloc(kPagerState * 4, &p->mem, err) != 0) {
      delete p;
      return 1;
    }
    const int32_t zero[kPagerState] = {};
    const hipError_t e = rt->copy_sync(p->mem, zero, sizeof(zero), hipMemcpyHostToDevice);
    if (e != hipSuccess) {
      delete p;
      return hip_err(err, "hipMemcpy(pager state)", e);
    }
    *out = p;
    return 0;
  });
}

int eoship_kv_pager_release(EosHipRuntime* rt, EosHipKVPager* pager, char** err) {
  if (pager == nullptr) return 0;
  if (rt == nullptr || pager->rt != rt)
    return set_err(err, "eoship_kv_pager_release: wrong runtime");
  OnDevice on(rt->device);
  if (rt->sync(err) != 0) return 1;
  delete pager;
  return 0;
}

int eoship_kv_pager_reset_device(EosHipRuntime* rt, EosHipKVPager* pager, char** err) {
  const char* what = "eoship_kv_pager_reset_device";
  return guarded(what, err, [&]() -> int {
    if (check(rt, pager, what, err) != 0) return 1;
    OnDevice on(rt->device);
    PagerArgs a = args(pager);
    const long long most = std::max((long long)a.slots * a.stride, a.pages);
    const unsigned n = (unsigned)std::max<long long>(
        (a.slots + 255) / 256, std::min<long long>((most + 255) / 256, 8LL * rt->compute_units));
    return rt->launch("eos_pager_reset", dim3(n), dim3(256), 0, &a, err);
  });
}

int eoship_kv_pager_extend_device(EosHipRuntime* rt, EosHipKVPager* pager, const int32_t* d_new,
                                  const EosHipKVPlan* plan, char** err) {
  const char* what = "eoship_kv_pager_extend_device";
  return guarded(what, err, [&]() -> int {
    if (check(rt, pager, what, err) != 0) return 1;
    if (d_new == nullptr || plan == nullptr) return set_err(err, "%s: NULL argument", what);
    if (plan->d_slots == nullptr || plan->d_lengths == nullptr || plan->d_offsets == nullptr)
      return set_err(err, "%s: NULL slots, lengths or offsets", what);
    if (plan->rows < 0 || plan->rows > INT32_MAX)
      return set_err(err, "%s: rows must be in 0..2^31-1, got %lld", what, (long long)plan->rows);
    if (!aligned(d_new, 4) || !aligned(plan->d_slots, 4) || !aligned(plan->d_lengths, 4) ||
        !aligned(plan->d_offsets, 4) || !aligned(plan->d_page_table, 4) ||
        !aligned(plan->d_positions, 4) || !aligned(plan->d_slot_map, 8))
      return set_err(err, "%s: arrays must be aligned to their elements", what);
    const EosHipKVPagerDesc& d = pager->d;
    const Arrays own(d);
    const int64_t slots = 4LL * d.slots;
    const Span put[] = {{plan->d_slots, slots},
                        {plan->d_page_table, slots * d.table_stride},
                        {plan->d_lengths, slots},
                        {plan->d_offsets, slots + 4},
                        {plan->d_positions, 4 * plan->rows},
                        {plan->d_slot_map, 8 * plan->rows}};
    const Span ask(d_new, slots);
    bool one = false, asked = false;
    for (int i = 0; i < 6; ++i) {
      for (int j = 0; j < i; ++j) one |= meet(put[i], put[j]);
      one |= meet(put[i], own.table) | meet(put[i], own.free) | meet(put[i], own.lengths) |
             meet(put[i], own.count);
      asked |= meet(put[i], ask);
    }
    if (one) return set_err(err, "%s: a plan's arrays overlap each other or the pager's", what);
    if (asked) return set_err(err, "%s: new overlaps a plan's arrays", what);
    // (lengths and the count are written when all workgroups have read theirs)
    if (meet(ask, own.table)) return set_err(err, "%s: new overlaps the page table", what);
    OnDevice on(rt->device);
    PagerArgs a = args(pager);
    a.ask = d_new;
    a.b_slots = plan->d_slots;
    a.b_table = plan->d_page_table;
    a.b_lengths = plan->d_lengths;
    a.b_offsets = plan->d_offsets;
    a.positions = plan->d_positions;
    a.slot_map = plan->d_slot_map;
    a.rows = plan->rows;
    const bool listed = a.positions != nullptr || a.slot_map != nullptr;
    return launch(rt, pager, "extend", listed ? a.rows : 0, (4 * (size_t)a.slots + 1) * 4, &a, err);
  });
}

int eoship_kv_pager_trim_device(EosHipRuntime* rt, EosHipKVPager* pager, const int32_t* d_keep,
                                char** err) {
  const char* what = "eoship_kv_pager_trim_device";
  return guarded(what, err, [&]() -> int {
    if (check(rt, pager, what, err) != 0) return 1;
    if (d_keep == nullptr) return set_err(err, "%s: NULL argument", what);
    if (!aligned(d_keep, 4))
      return set_err(err, "%s: arrays must be aligned to their elements", what);
    const Arrays own(pager->d);
    const Span ask(d_keep, 4LL * pager->d.slots);
    if (meet(ask, own.table) || meet(ask, own.free))
      return set_err(err, "%s: keep overlaps the page table or the free pages", what);
    OnDevice on(rt->device);
    PagerArgs a = args(pager);
    a.ask = d_keep;
    return launch(rt, pager, "trim", 0, 3 * (size_t)a.slots * 4, &a, err);
  });
}

int eoship_kv_pager_status(EosHipRuntime* rt, EosHipKVPager* pager, int32_t* status, char** err) {
  const char* what = "eoship_kv_pager_status";
  return guarded(what, err, [&]() -> int {
    if (check(rt, pager, what, err) != 0) return 1;
    if (status == nullptr) return set_err(err, "%s: NULL argument", what);
    OnDevice on(rt->device);
    hipError_t e = rt->copy_async(status, pager->mem, 4, hipMemcpyDeviceToHost);
    if (e != hipSuccess) return hip_err(err, what, e);
    if (rt->sync(err) != 0) return 1;
    if (*status == 0) return 0;
    const int32_t zero = 0;
    e = rt->copy_async(pager->mem, &zero, 4, hipMemcpyHostToDevice);
    if (e != hipSuccess) return hip_err(err, what, e);
    return rt->sync(err);
  });
}

}  // extern "C"
