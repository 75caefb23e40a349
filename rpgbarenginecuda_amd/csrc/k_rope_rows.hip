// Rotation of queries and keys at any positions: pairs (i, i + rot / 2) or (2i, 2i + 1)
// of the first `rot` elements of each head,
//   a <- a cos - b sin,  b <- b cos + a sin,
// each product rounded by itself, as the other rotations here; the rest of a head is
// copied. cos and sin come from a table of rows of positions, so that scaled
// frequencies (BuildRopeTableScaled) cost nothing here.
//
// What bounds it: every element is read and written once, a row of the table once a
// token. A thread has two chunks of four elements, the same of kHeads heads of one
// token, for which it reads the table once; of a rotated part the chunks lie half of
// that part apart in either layout, so that a lane has both members of its pairs and
// the lanes of a head read and write whole lines. 2811 tokens of 24 heads of 128 take 12.5 us (5.6 TB/s), 9001
// of 40, half of each rotated, 62 (6.0 TB/s), a single one 2.2, the launch.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "dev_util.h"
#include "kernels_gpu.h"
#include "launch.h"
#include "paged_kv.h"

namespace rpg {
namespace {

constexpr int kThreads = 256;
constexpr int32_t kMaxHeadDim = 1024;

struct RopeArgs {
  const float* q;
  const float* k;
  float* q_out;
  float* k_out;
  const float* tab;
  const int32_t* positions;
  int64_t tab_rows;
  int32_t n_heads;
  int32_t n_kv;
  int32_t head_dim;
  int32_t rot;
  uint32_t groups;  // groups of heads of a token
  uint32_t units;   // of all tokens
};

// Head h of token t (queries first, then keys), in `q`, `k`.
template <class T>
__device__ __forceinline__ T* HeadAt(T* q, T* k, const RopeArgs& a, uint32_t t, int32_t h) {
  return h < a.n_heads ? q + (static_cast<int64_t>(t) * a.n_heads + h) * a.head_dim
                       : k + (static_cast<int64_t>(t) * a.n_kv + (h - a.n_heads)) * a.head_dim;
}

// blockDim: x a head's pairs of chunks (head_dim / 8), y groups of heads.
template <int kHeads, bool kInterleaved>
__global__ __launch_bounds__(kThreads) void RopeRowsKernel(const RopeArgs a) {
  const uint32_t unit = blockIdx.x * blockDim.y + threadIdx.y;
  if (unit >= a.units) return;
  const uint32_t t = unit / a.groups;
  const int32_t h0 = static_cast<int32_t>(unit - t * a.groups) * kHeads;
  const int32_t j = threadIdx.x;
  const bool turns = j < a.rot / 8;
  const int32_t first = turns ? 4 * j : 4 * j + a.rot / 2;  // the copied part's chunk j - rot / 8, behind rot
  const int32_t second = first + (turns ? a.rot : a.head_dim - a.rot) / 2;
  const int32_t heads = min(kHeads, a.n_heads + a.n_kv - h0);
  float4 x[kHeads], y[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    if (i < heads) {
      const float* from = HeadAt(a.q, a.k, a, t, h0 + i);
      x[i] = dev::LoadStream4(from + first);
      y[i] = dev::LoadStream4(from + second);
    }
  }
  if (turns) {
    const int32_t pos = a.positions[t];
    const bool fine = pos >= 0 && pos < a.tab_rows;
    const float* row = a.tab + (fine ? static_cast<int64_t>(pos) * a.rot : 0);
    float4 co, si, co2, si2;  // of the first chunk's elements, and the second's
    if constexpr (kInterleaved) {
      const auto both = [](float2 p) { return make_float4(p.x, p.x, p.y, p.y); };
      const auto at = [row](int32_t i) { return *reinterpret_cast<const float2*>(row + i); };
      co = both(at(2 * j));
      si = both(at(a.rot / 2 + 2 * j));
      co2 = both(at(a.rot / 4 + 2 * j));
      si2 = both(at(3 * (a.rot / 4) + 2 * j));
    } else {
      co = co2 = dev::Load4(row + 4 * j);
      si = si2 = dev::Load4(row + a.rot / 2 + 4 * j);
    }
    const float bad = fine ? 0.0f : NAN;
    co = make_float4(co.x + bad, co.y + bad, co.z + bad, co.w + bad);
    co2 = make_float4(co2.x + bad, co2.y + bad, co2.z + bad, co2.w + bad);
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      const float4 p = x[i], r = y[i];
      if constexpr (kInterleaved) {
        x[i] = make_float4(p.x * co.x - p.y * si.x, p.y * co.y + p.x * si.y, p.z * co.z - p.w * si.z,
                           p.w * co.w + p.z * si.w);
        y[i] = make_float4(r.x * co2.x - r.y * si2.x, r.y * co2.y + r.x * si2.y, r.z * co2.z - r.w * si2.z,
                           r.w * co2.w + r.z * si2.w);
      } else {
        x[i] = make_float4(p.x * co.x - r.x * si.x, p.y * co.y - r.y * si.y, p.z * co.z - r.z * si.z,
                           p.w * co.w - r.w * si.w);
        y[i] = make_float4(r.x * co.x + p.x * si.x, r.y * co.y + p.y * si.y, r.z * co.z + p.z * si.z,
                           r.w * co.w + p.w * si.w);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    if (i < heads) {
      float* to = HeadAt(a.q_out, a.k_out, a, t, h0 + i);
      dev::StoreStream4(to + first, x[i]);
      dev::StoreStream4(to + second, y[i]);
    }
  }
}

// Any even rot and any head: a thread per pair, and per copied element. blockDim: x a wave of them, y heads.
template <bool kInterleaved>
__global__ __launch_bounds__(kThreads) void RopeRowsPairKernel(const RopeArgs a) {
  const uint32_t unit = blockIdx.x * blockDim.y + threadIdx.y;
  if (unit >= a.units) return;
  const uint32_t t = unit / a.groups;
  const int32_t h = static_cast<int32_t>(unit - t * a.groups);
  const float* from = HeadAt(a.q, a.k, a, t, h);
  float* to = HeadAt(a.q_out, a.k_out, a, t, h);
  const int32_t half = a.rot / 2;
  const int32_t pos = a.positions[t];
  const bool fine = pos >= 0 && pos < a.tab_rows;
  const float* row = a.tab + (fine ? static_cast<int64_t>(pos) * a.rot : 0);
  for (int32_t e = threadIdx.x; e < a.head_dim - half; e += blockDim.x) {
    if (e < half) {
      const int32_t i = kInterleaved ? 2 * e : e, k = kInterleaved ? 2 * e + 1 : e + half;
      const float co = fine ? row[e] : NAN, si = row[half + e];
      const float p = from[i], r = from[k];
      to[i] = p * co - r * si;
      to[k] = r * co + p * si;
    } else {
      to[half + e] = from[half + e];
    }
  }
}

}  // namespace

void GpuRopeRows(const float* q, const float* k, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim,
                 int32_t rot_dim, bool interleaved, const float* rope_tab, int64_t rope_rows,
                 const int32_t* positions, int64_t n_rows, float* q_out, float* k_out) {
  RPG_CHECK(n_heads > 0 && n_kv_heads >= 0 && n_heads <= (1 << 20) && n_kv_heads <= (1 << 20),
            "RopeRows: %d query heads and %d kv heads", n_heads, n_kv_heads);
  RPG_CHECK(head_dim > 0 && head_dim <= kMaxHeadDim, "RopeRows: head_dim %d is not 1 to %d", head_dim, kMaxHeadDim);
  RPG_CHECK(rot_dim > 0 && rot_dim % 2 == 0 && rot_dim <= head_dim,
            "RopeRows: rot_dim %d is not an even number of a head's %d elements", rot_dim, head_dim);
  RPG_CHECK(rope_rows > 0 && rope_rows <= (int64_t(1) << 40), "RopeRows: a RoPE table of %lld rows",
            static_cast<long long>(rope_rows));
  const int32_t per_token = n_heads + n_kv_heads;
  RPG_CHECK(n_rows >= 0 && n_rows <= 0x7FFFFFFF / per_token, "RopeRows: %lld rows of %d heads are out of range",
            static_cast<long long>(n_rows), per_token);
  if (n_rows == 0) return;
  RPG_CHECK(q != nullptr && q_out != nullptr && rope_tab != nullptr && positions != nullptr &&
                (n_kv_heads == 0 || (k != nullptr && k_out != nullptr)),
            "RopeRows got a null pointer");
  const auto at = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
  uintptr_t all = at(q) | at(q_out) | at(rope_tab);
  if (n_kv_heads > 0) all |= at(k) | at(k_out);
  RPG_CHECK(((all | at(positions)) & 3) == 0, "RopeRows: a pointer is not 4-byte aligned");
  const int64_t q_bytes = n_rows * n_heads * head_dim * 4, k_bytes = n_rows * n_kv_heads * head_dim * 4;
  RPG_CHECK(q == q_out || !Overlap(q, q_bytes, q_out, q_bytes), "RopeRows: q_out has to be q itself or apart from it");
  if (n_kv_heads > 0) {
    RPG_CHECK(k == k_out || !Overlap(k, k_bytes, k_out, k_bytes), "RopeRows: k_out has to be k itself or apart from it");
    RPG_CHECK(!Overlap(q_out, q_bytes, k, k_bytes) && !Overlap(k_out, k_bytes, q, q_bytes) &&
                  !Overlap(q_out, q_bytes, k_out, k_bytes),
              "RopeRows: queries must not overlap keys");
  }
  const int64_t tab_bytes = rope_rows * rot_dim * 4;
  RPG_CHECK(!Overlap(q_out, q_bytes, rope_tab, tab_bytes) && !Overlap(q_out, q_bytes, positions, 4 * n_rows) &&
                (n_kv_heads == 0 ||
                 (!Overlap(k_out, k_bytes, rope_tab, tab_bytes) && !Overlap(k_out, k_bytes, positions, 4 * n_rows))),
            "RopeRows: outputs must not overlap the table or the positions");
  RopeArgs a{q,         k,       q_out,      k_out,    rope_tab, positions,
             rope_rows, n_heads, n_kv_heads, head_dim, rot_dim,  static_cast<uint32_t>(per_token), 0};
  // whole chunks of four elements, aligned; else a pair to a thread (2811 rows of 24 heads of 128: 12.5 us against 21, one row
  // the same)
  if (head_dim % 8 == 0 && rot_dim % 8 == 0 && (all & 15) == 0) {
    constexpr int kHeads = 4;
    const dim3 block(head_dim / 8, std::max(1, kThreads / (head_dim / 8)));
    // one head to a thread up to six workgroups to a compute unit, so that more of the card works; then four, which read the
    // table's row once (24 heads of 128, us, one against four: 1 row 2.4 / 3.0, 341 3.5 / 4.3, 1024 5.5 / 5.6, 2811 13.9 / 12.5)
    const bool few = n_rows * per_token * (head_dim / 8) <= 6 * 256 * kThreads;
    a.groups = few ? per_token : (per_token + kHeads - 1) / kHeads;
    a.units = static_cast<uint32_t>(n_rows) * a.groups;
    const int64_t blocks = (int64_t{a.units} + block.y - 1) / block.y;
    RPG_CHECK(FitsLaunch(blocks, block.x), "RopeRows: %lld rows of %d heads are too many for one call",
              static_cast<long long>(n_rows), per_token);
    auto* kern = few ? (interleaved ? RopeRowsKernel<1, true> : RopeRowsKernel<1, false>)
                     : (interleaved ? RopeRowsKernel<kHeads, true> : RopeRowsKernel<kHeads, false>);
    Launch("RopeRowsKernel", kern, dim3(static_cast<uint32_t>(blocks)), block, a);
    return;
  }
  const dim3 block(64, kThreads / 64);
  a.units = static_cast<uint32_t>(n_rows) * a.groups;
  const int64_t blocks = (int64_t{a.units} + block.y - 1) / block.y;
  RPG_CHECK(FitsLaunch(blocks, block.x), "RopeRows: %lld rows of %d heads, in single elements, are too many for one call",
            static_cast<long long>(n_rows), per_token);
  Launch("RopeRowsPairKernel", interleaved ? RopeRowsPairKernel<true> : RopeRowsPairKernel<false>,
         dim3(static_cast<uint32_t>(blocks)), block, a);
}

}  // namespace rpg
