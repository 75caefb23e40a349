// What the kernels over the paged KV cache share: the device's view of a call's
// pool and table, where a row of the call lives, and the checks of both.
#ifndef RPG_AMD_PAGED_KV_H_
#define RPG_AMD_PAGED_KV_H_

#include <hip/hip_runtime.h>

#include <cstdint>

#include "kernels_gpu.h"

namespace rpg {

// Throws unless kv and table describe a cache that a kernel can address.
void CheckPagedKv(const char* what, const GpuPagedKv& kv, const GpuPageTable& table);

// Whether [a, a + na) and [b, b + nb) share a byte.
inline bool Overlap(const void* a, int64_t na, const void* b, int64_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + static_cast<uint64_t>(nb) && y < x + static_cast<uint64_t>(na);
}

namespace dev {

// Passed to kernels by value.
struct PagedView {
  const int32_t* pages;
  int64_t n_seqs;
  int64_t max_pages;
  int32_t n_pages;
  int32_t n_kv;
  int32_t page_shift;  // log2(page_size)
  const void* k;
  const void* v;
  const float* k_scale;
  const float* v_scale;
};

inline PagedView ViewOf(const GpuPagedKv& kv, const GpuPageTable& table) {
  int32_t shift = 0;
  while ((1 << shift) < kv.page_size) ++shift;
  return PagedView{table.pages, table.n_seqs, table.max_pages, static_cast<int32_t>(kv.n_pages), kv.n_kv_heads,
                   shift,       kv.k,         kv.v,            kv.k_scale,                        kv.v_scale};
}

// A row's slot: the index of its kv head 0 among the pool's rows (row index =
// (page * n_kv + head) * page_size + slot), so head h is at first + h * page_size.
enum class SlotState : int32_t { kOk, kPadding, kBad };
struct Slot {
  SlotState state;
  int64_t first;
};

__device__ __forceinline__ Slot FindSlot(const PagedView& view, int64_t seq, int32_t pos) {
  Slot s{SlotState::kOk, 0};
  if (seq < 0) {
    s.state = SlotState::kPadding;
    return s;
  }
  const int64_t n = static_cast<int64_t>(pos) >> view.page_shift;
  s.state = SlotState::kBad;
  if (seq >= view.n_seqs || pos < 0 || n >= view.max_pages) return s;
  const int32_t page = view.pages[seq * view.max_pages + n];
  if (page < 0 || page >= view.n_pages) return s;
  s.state = SlotState::kOk;
  s.first = ((static_cast<int64_t>(page) * view.n_kv) << view.page_shift) + (pos & ((1 << view.page_shift) - 1));
  return s;
}

}  // namespace dev
}  // namespace rpg

#endif  // RPG_AMD_PAGED_KV_H_
