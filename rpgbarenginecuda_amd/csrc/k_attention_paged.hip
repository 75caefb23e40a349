// Attention of one new token per row over the paged KV cache.
//
// For row r, query head h of kv head h / G, over the positions j < lens[r]:
//   s_j = (q . k_j) / sqrt(D),  out = sum_j exp(s_j - max s) v_j / sum_j exp(s_j - max s)
// in one pass over the cache, with the running maximum m and sum l: on a new
// maximum the sum and the accumulated output are scaled by exp(m_old - m_new).
#include <hip/hip_runtime.h>

#include <cmath>

#include "dev_util.h"
#include "kernels_gpu.h"
#include "launch.h"
#include "paged_kv.h"

namespace rpg {
namespace {

using dev::PagedView;
using dev::Slot;
using dev::SlotState;

constexpr int kWaves = 4;

template <bool kQ8>
__device__ __forceinline__ float Cached(const void* pool, const float* scale, int64_t row, int64_t at) {
  if constexpr (kQ8) return static_cast<float>(static_cast<const int8_t*>(pool)[at]) * scale[row];
  return static_cast<float>(static_cast<const _Float16*>(pool)[at]);
}

// One workgroup per (row, query head); its waves take every fourth position, a
// lane holds D / 64 elements.
template <int D, bool kQ8>
__global__ __launch_bounds__(64 * kWaves) void PagedAttentionKernel(PagedView view,
                                                                    const int32_t* __restrict__ seq_ids,
                                                                    const int32_t* __restrict__ lens,
                                                                    const float* __restrict__ q, int32_t n_heads,
                                                                    float scale, float* __restrict__ out) {
  constexpr int kE = D / 64;
  __shared__ float part[kWaves][D + 2];
  const int64_t unit = blockIdx.x;
  const int64_t r = unit / n_heads;
  const int32_t h = static_cast<int32_t>(unit - r * n_heads);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t seq = seq_ids != nullptr ? seq_ids[r] : r;
  if (seq < 0) return;
  const int32_t len = lens[r];
  const bool bad = seq >= view.n_seqs || len < 0 || len > (view.max_pages << view.page_shift);
  const int32_t kh = h / (n_heads / view.n_kv);
  float x[kE], o[kE] = {};
#pragma unroll
  for (int e = 0; e < kE; ++e) x[e] = q[(r * n_heads + h) * D + lane * kE + e];
  float m = -INFINITY, l = bad ? NAN : 0.0f;
  for (int32_t j = wave; j < len && !bad; j += kWaves) {
    const Slot slot = dev::FindSlot(view, seq, j);
    const int64_t row = slot.first + (static_cast<int64_t>(kh) << view.page_shift);
    const bool ok = slot.state == SlotState::kOk;
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      s = fmaf(x[e], ok ? Cached<kQ8>(view.k, view.k_scale, row, row * D + lane * kE + e) : NAN, s);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
    s *= scale;
    const float top = fmaxf(m, s);
    const float safe = top == -INFINITY ? 0.0f : top;
    const float f = expf(m - safe), p = expf(s - safe);
    l = fmaf(l, f, p);
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      o[e] = fmaf(o[e], f, ok ? p * Cached<kQ8>(view.v, view.v_scale, row, row * D + lane * kE + e) : NAN);
    }
    m = top;
  }
#pragma unroll
  for (int e = 0; e < kE; ++e) part[wave][lane * kE + e] = o[e];
  if (lane == 0) {
    part[wave][D] = m;
    part[wave][D + 1] = l;
  }
  __syncthreads();
  if (threadIdx.x >= D) return;
  float top = -INFINITY, sum = 0.0f, total = 0.0f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) top = fmaxf(top, part[w][D]);
  const float safe = top == -INFINITY ? 0.0f : top;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const float f = expf(part[w][D] - safe);
    total = fmaf(part[w][D + 1], part[w][D] == -INFINITY && part[w][D + 1] == 0.0f ? 0.0f : f, total);
    sum = fmaf(part[w][threadIdx.x], f, sum);
  }
  if (bad) sum = total = NAN;
  out[(r * n_heads + h) * D + threadIdx.x] = len == 0 ? 0.0f : sum / total;
}

void CheckHeads(const char* what, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim) {
  RPG_CHECK(head_dim == 64 || head_dim == 128, "%s: head_dim %d is neither 64 nor 128", what, head_dim);
  RPG_CHECK(n_kv_heads > 0 && n_heads > 0 && n_heads <= (1 << 20) && n_heads % n_kv_heads == 0,
            "%s: %d query heads do not divide among %d kv heads", what, n_heads, n_kv_heads);
}

}  // namespace

size_t GpuAttentionPagedWorkspaceBytes(int32_t n_heads, int32_t n_kv_heads, int32_t head_dim) {
  CheckHeads("AttentionPagedWorkspace", n_heads, n_kv_heads, head_dim);
  return 256;
}

void GpuAttentionPagedWorkspaceInit(void* workspace, size_t bytes) {
  RPG_CHECK(workspace != nullptr && bytes > 0 && bytes % 16 == 0 && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0,
            "AttentionPagedWorkspaceInit: a workspace is 256-byte aligned and a multiple of 16 bytes");
  GpuStreamFill(workspace, static_cast<int64_t>(bytes), 0);
}

void GpuAttentionPaged(const GpuPagedKv& kv, const GpuPageTable& table, const int32_t* seq_ids, const int32_t* lens,
                       const float* q_dev, int32_t n_heads, int64_t n_rows, float* out_dev, void* workspace,
                       size_t workspace_bytes) {
  CheckPagedKv("AttentionPaged", kv, table);
  CheckHeads("AttentionPaged", n_heads, kv.n_kv_heads, kv.head_dim);
  RPG_CHECK(n_rows >= 0 && n_rows <= 0x7FFFFFFF, "AttentionPaged: %lld rows", static_cast<long long>(n_rows));
  if (n_rows == 0) return;
  RPG_CHECK(lens != nullptr && q_dev != nullptr && out_dev != nullptr && workspace != nullptr,
            "AttentionPaged got a null pointer");
  RPG_CHECK(seq_ids != nullptr || n_rows <= table.n_seqs, "AttentionPaged: %lld rows without seq_ids, but %lld sequences",
            static_cast<long long>(n_rows), static_cast<long long>(table.n_seqs));
  RPG_CHECK(((reinterpret_cast<uintptr_t>(q_dev) | reinterpret_cast<uintptr_t>(out_dev)) & 15) == 0,
            "AttentionPaged: q and out have to be 16-byte aligned");
  const int64_t q_bytes = n_rows * n_heads * kv.head_dim * 4;
  RPG_CHECK(!Overlap(q_dev, q_bytes, out_dev, q_bytes), "AttentionPaged: out must not overlap q");
  const size_t need = GpuAttentionPagedWorkspaceBytes(n_heads, kv.n_kv_heads, kv.head_dim);
  RPG_CHECK((reinterpret_cast<uintptr_t>(workspace) & 255) == 0 && workspace_bytes >= need,
            "AttentionPaged: a workspace of %zu bytes, 256-byte aligned, is needed (%zu given)", need, workspace_bytes);
  const float scale = static_cast<float>(1.0 / std::sqrt(static_cast<double>(kv.head_dim)));
  const bool q8 = kv.type == kKvQ8;
  auto* kern = kv.head_dim == 128 ? (q8 ? PagedAttentionKernel<128, true> : PagedAttentionKernel<128, false>)
                                  : (q8 ? PagedAttentionKernel<64, true> : PagedAttentionKernel<64, false>);
  Launch("PagedAttentionKernel", kern, dim3(GridFor(n_rows * n_heads, 1)), dim3(64 * kWaves), dev::ViewOf(kv, table),
         seq_ids, lens, q_dev, n_heads, scale, out_dev);
}

}  // namespace rpg
