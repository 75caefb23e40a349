// What the kernels over the paged KV cache share: the device's view of a call's
// pool and table, where a row of the call lives, and the checks of both.
#ifndef RPG_AMD_PAGED_KV_H_
#define RPG_AMD_PAGED_KV_H_

#include <hip/hip_runtime.h>

#include <cstdint>

#include "attention_dev.h"
#include "kernels_gpu.h"

namespace rpg {

// Throws unless kv and table describe a cache that a kernel can address.
void CheckPagedKv(const char* what, const GpuPagedKv& kv, const GpuPageTable& table);

// Whether [a, a + na) and [b, b + nb) share a byte.
inline bool Overlap(const void* a, int64_t na, const void* b, int64_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + static_cast<uint64_t>(nb) && y < x + static_cast<uint64_t>(na);
}

// Attention of a batch whose rows share their beginnings: AttendPaged, given one of these, attends to what is each
// row's own and leaves for row r and head h, besides the output, ml[r][h] = (m, l), the maximum of its scores (as powers
// of two) and the sum of weights that the output is divided by; AttendPrefix (k_attention_prefix.hip) then attends to the
// shared positions and joins both in the output.
struct PagedPrefix {
  const int32_t* group_rows;
  const int32_t* group_pages;
  int32_t n_groups;
  int64_t least = 0;  // pages times rows that sharing has to save, at most kMostSaving
  char* workspace = nullptr;
  float* ml = nullptr;
};
constexpr int64_t kMostSaving = int64_t(1) << 50;  // of a group: what exceeds it counts as this

// GpuAttentionPaged, of what is behind the shared positions if there is a prefix (and then of the rest).
void AttendPaged(const GpuPagedKv& kv, const GpuPageTable& table, const int32_t* seq_ids, const int32_t* lens,
                 const float* q_dev, int32_t n_heads, int64_t n_rows, float* out_dev, void* workspace,
                 size_t workspace_bytes, PagedPrefix* prefix);

// Refuses what AttendPrefix cannot serve, and places prefix's part in the workspace.
void CheckPrefix(const GpuPagedKv& kv, const GpuPageTable& table, int32_t n_heads, int64_t n_rows, char* workspace,
                 PagedPrefix* prefix);
void AttendPrefix(const GpuPagedKv& kv, const GpuPageTable& table, const int32_t* seq_ids, const int32_t* lens,
                  const float* q_dev, int32_t n_heads, int64_t n_rows, float* out_dev, const PagedPrefix& prefix);

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

constexpr int kMaxSharedGroups = 64;

// A call's groups, one to a lane. Rows [first, last) of a group begin with the same `pages` pages; a row that several
// groups name is of the first of them. What is out of range is cut off. Groups that together save less than `least` pages
// times rows share nothing: their rows are attended to by themselves, in one kernel's work instead of three's.
struct SharedGroups {
  int32_t n;
  int32_t first = 0, last = 0, pages = 0;

  __device__ __forceinline__ SharedGroups(const int32_t* group_rows, const int32_t* group_pages, int32_t n_groups,
                                          int64_t least, int32_t n_rows, int64_t max_pages, int lane)
      : n(n_groups) {
    if (lane < n_groups) {
      first = min(max(group_rows[lane], 0), n_rows);
      last = min(max(group_rows[lane + 1], first), n_rows);
      const int32_t p = group_pages[lane];
      pages = p > 0 && p <= max_pages ? p : 0;
    }
    const int64_t rows_less_one = last > first ? last - first - 1 : 0, saving = min(rows_less_one * pages, kMostSaving);
    const uint32_t high = attn::ScanAdd(static_cast<uint32_t>(saving >> 25));  // in two parts, of 25 bits each
    const uint32_t low = attn::ScanAdd(static_cast<uint32_t>(saving) & ((1u << 25) - 1));
    const uint32_t high_all = __builtin_amdgcn_readlane(high, 63), low_all = __builtin_amdgcn_readlane(low, 63);
    if ((static_cast<int64_t>(high_all) << 25) + low_all < least) pages = 0;
  }
  // The group of row r, the lane's; -1 if there is none. Every lane has to be active, here and at PagesOfLane: what a lane
  // holds is read by all, and a lane that is not at work may hold anything.
  __device__ __forceinline__ int32_t OfLane(int32_t r) const {
    int32_t found = -1;
#pragma unroll 1
    for (int32_t g = n - 1; g >= 0; --g) {
      const int32_t from = __builtin_amdgcn_readlane(first, g), to = __builtin_amdgcn_readlane(last, g);
      found = (r >= from) & (r < to) ? g : found;
    }
    return found;
  }
  __device__ __forceinline__ int32_t PagesOfLane(int32_t r) const {
    int32_t found = 0;
#pragma unroll 1
    for (int32_t g = n - 1; g >= 0; --g) {
      const int32_t from = __builtin_amdgcn_readlane(first, g), to = __builtin_amdgcn_readlane(last, g);
      const int32_t shared = __builtin_amdgcn_readlane(pages, g);
      found = (r >= from) & (r < to) ? shared : found;
    }
    return found;
  }
  // r the same in every lane.
  __device__ __forceinline__ int32_t PagesOf(int32_t r) const {
    const uint64_t in = __ballot(r >= first && r < last);
    return in == 0 ? 0 : __builtin_amdgcn_readlane(pages, __builtin_ctzll(in));
  }
};

// Whether a row of len positions begins with all of these pages: one that does not is attended to by itself.
__device__ __forceinline__ bool TakesPart(int32_t pages, int32_t page_shift, int32_t len) {
  return pages > 0 && pages <= (len >> page_shift);
}

}  // namespace dev
}  // namespace rpg

#endif  // RPG_AMD_PAGED_KV_H_
