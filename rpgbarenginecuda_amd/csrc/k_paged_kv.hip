// The paged KV cache's writers and its reader: rows put into pages as fp16 or as
// 8-bit codes with a scale, with or without the q / k norm and rotation in front,
// and rows read back out of pages. The cache's layout and its 8-bit form are
// described in kernels_gpu.h.
//
// Every kernel here moves each byte once and computes a few operations on it, so
// memory bounds it (launch latency for a few tokens: 2.4 us for one). A head row of D elements is
// spread over D / 16 lanes, 16 elements each, arranged as head_row.h arranges 128
// of them over 8 lanes: both members of every rotated pair (i, i + D/2) sit in one
// lane, and the sums and maxima over a row are butterflies over its lanes.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>

#include "dev_util.h"
#include "kernels_gpu.h"
#include "launch.h"
#include "paged_kv.h"

namespace rpg {

void CheckPagedKv(const char* what, const GpuPagedKv& kv, const GpuPageTable& table) {
  RPG_CHECK(kv.type == kKvF16 || kv.type == kKvQ8, "%s: cache type %u is neither F16 nor Q8", what, kv.type);
  RPG_CHECK(kv.head_dim == 64 || kv.head_dim == 128, "%s: head_dim %d is neither 64 nor 128", what, kv.head_dim);
  RPG_CHECK(kv.n_kv_heads > 0 && kv.n_kv_heads <= 65536, "%s: n_kv_heads %d out of range", what, kv.n_kv_heads);
  RPG_CHECK(kv.page_size >= 16 && kv.page_size <= 256 && (kv.page_size & (kv.page_size - 1)) == 0,
            "%s: page_size %d is not a power of two from 16 to 256", what, kv.page_size);
  RPG_CHECK(kv.n_pages > 0 && kv.n_pages <= 0x7FFFFFFF, "%s: a pool of %lld pages is out of range", what,
            static_cast<long long>(kv.n_pages));
  RPG_CHECK(table.n_seqs > 0 && table.max_pages > 0 && table.n_seqs <= 0x7FFFFFFF && table.max_pages <= 0x7FFFFFFF,
            "%s: a page table of %lld x %lld entries is out of range", what, static_cast<long long>(table.n_seqs),
            static_cast<long long>(table.max_pages));
  RPG_CHECK(kv.k != nullptr && kv.v != nullptr && table.pages != nullptr, "%s got a null cache or table", what);
  const uintptr_t scales = kv.type == kKvQ8 ? reinterpret_cast<uintptr_t>(kv.k_scale) |
                                                  reinterpret_cast<uintptr_t>(kv.v_scale)
                                            : 0;
  RPG_CHECK(kv.type != kKvQ8 || (kv.k_scale != nullptr && kv.v_scale != nullptr), "%s: a Q8 cache needs its scales",
            what);
  RPG_CHECK(((reinterpret_cast<uintptr_t>(kv.k) | reinterpret_cast<uintptr_t>(kv.v) | scales) & 15) == 0 &&
                (reinterpret_cast<uintptr_t>(table.pages) & 3) == 0,
            "%s: the cache has to be 16-byte aligned, the table 4-byte aligned", what);
}

namespace {

using dev::PagedView;
using dev::Slot;
using dev::SlotState;

constexpr int kBlock = 256;

bool Aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Workgroups go to the eight XCDs in turn. Each XCD takes one stretch of the tokens
// instead of every eighth workgroup, so that neighbouring slots, and the 32 scales in
// a line of them, meet in one L2: 16.0 -> 15.1 us for 8 x 1024 tokens written as 8 bits.
__device__ __forceinline__ uint32_t WorkgroupInStretch() {
  const uint32_t x = blockIdx.x & 7, each = gridDim.x >> 3, rest = gridDim.x & 7;
  return x * each + (x < rest ? x : rest) + (blockIdx.x >> 3);
}

// A lane's 16 elements of a head row: a[c] is elements 4l + (D/4)c of the first
// half, b[c] the same of the second. At D = 128 this is dev::HeadRow.
struct Row {
  float4 a[2];
  float4 b[2];
};

template <int D>
struct RowOf {
  static constexpr int kLanes = D / 16;

  static __device__ __forceinline__ int Offset(int l, int c) { return 4 * l + (D / 4) * c; }

  static __device__ __forceinline__ Row Load(const float* p, int l) {
    Row r;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      r.a[c] = dev::Load4(p + Offset(l, c));
      r.b[c] = dev::Load4(p + D / 2 + Offset(l, c));
    }
    return r;
  }

  static __device__ __forceinline__ void StoreStream(float* p, int l, const Row& r) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      dev::StoreStream4(p + Offset(l, c), r.a[c]);
      dev::StoreStream4(p + D / 2 + Offset(l, c), r.b[c]);
    }
  }

  // (x * scale) * w with scale = float(1 / sqrt(sum of squares / D + eps)), the sum
  // in double and in head_row.h's order: the same bits at D = 128. ss / D is exact.
  static __device__ __forceinline__ void Norm(Row& r, const Row& w, float eps) {
    double ss = 0.0;
#pragma unroll
    for (int c = 0; c < 2; ++c) ss = dev::AddSquares(dev::AddSquares(ss, r.a[c]), r.b[c]);
    ss = dev::GroupSum<kLanes>(ss);
    const float scale = dev::HeadRmsScale(ss * (128.0 / D), eps);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      r.a[c] = dev::ScaleMul(r.a[c], scale, w.a[c]);
      r.b[c] = dev::ScaleMul(r.b[c], scale, w.b[c]);
    }
  }

  // x_i <- a cos - b sin, x_{i + D/2} <- b cos + a sin, each product rounded.
  static __device__ __forceinline__ void Rotate(Row& r, const Row& t) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const float4 co = t.a[c], si = t.b[c], a = r.a[c], b = r.b[c];
      r.a[c] = make_float4(a.x * co.x - b.x * si.x, a.y * co.y - b.y * si.y, a.z * co.z - b.z * si.z,
                           a.w * co.w - b.w * si.w);
      r.b[c] = make_float4(b.x * co.x + a.x * si.x, b.y * co.y + a.y * si.y, b.z * co.z + a.z * si.z,
                           b.w * co.w + a.w * si.w);
    }
  }

  // As fp16, 16 bytes a store: the lanes of a pair swap one of their two chunks of each half (as head_row.h does), so
  // that a store instruction writes whole lines.
  static __device__ __forceinline__ void StoreHalf(uint16_t* p, int l, const Row& r) {
    const bool odd = (l & 1) != 0;
    const int at = odd ? D / 4 + 4 * (l - 1) : 4 * l;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const uint2 c0 = dev::PackHalf4(s == 0 ? r.a[0] : r.b[0]);
      const uint2 c1 = dev::PackHalf4(s == 0 ? r.a[1] : r.b[1]);
      const uint2 send = odd ? c0 : c1;
      const uint2 recv = make_uint2(Quad<0xB1>(send.x), Quad<0xB1>(send.y));
      *reinterpret_cast<uint4*>(p + D / 2 * s + at) =
          odd ? make_uint4(recv.x, recv.y, c1.x, c1.y) : make_uint4(c0.x, c0.y, recv.x, recv.y);
    }
  }

  // The row's 8-bit form. Every lane of the row takes part.
  static __device__ __forceinline__ void StoreQ8(int8_t* p, float* scale, int l, const Row& r) {
    float top = 0.0f;
#pragma unroll
    for (int c = 0; c < 2; ++c) top = fmaxf(top, fmaxf(Top4(r.a[c]), Top4(r.b[c])));
#pragma unroll
    for (int off = kLanes / 2; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, kLanes));
    const bool finite = top <= FLT_MAX;
    float s = top * (1.0f / 127.0f);
    if (s < FLT_MIN) s = 0.0f;
    const float inv = finite && s > 0.0f ? 1.0f / s : 0.0f;
    if (l == 0) *scale = finite ? s : __builtin_nanf("");
    // word b of a lane is its four codes of quarter b of the row. The four lanes of a quad trade them, so that lane i has
    // the quad's words of quarter i, 16 bytes in a row.
    uint32_t w[4] = {Codes4(r.a[0], inv, finite), Codes4(r.a[1], inv, finite), Codes4(r.b[0], inv, finite),
                     Codes4(r.b[1], inv, finite)};
    const int i = l & 3;
    // lanes 1 apart trade the words of odd against even quarters, then lanes 2 apart those of 2 and 3 against 0 and 1
    Trade<0xB1>((i & 1) != 0, &w[0], &w[1]);
    Trade<0xB1>((i & 1) != 0, &w[2], &w[3]);
    Trade<0x4E>((i & 2) != 0, &w[0], &w[2]);
    Trade<0x4E>((i & 2) != 0, &w[1], &w[3]);
    *reinterpret_cast<uint4*>(p + D / 4 * i + 16 * (l >> 2)) = make_uint4(w[0], w[1], w[2], w[3]);
  }

 private:
  // x of the lane that kPerm (a quad_perm) names: 0xB1 the neighbour, 0x4E the one 2 apart.
  template <int kPerm>
  static __device__ __forceinline__ uint32_t Quad(uint32_t x) {
    return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(x), kPerm, 0xF, 0xF, false));
  }

  // A lower lane's b against the upper lane's a.
  template <int kPerm>
  static __device__ __forceinline__ void Trade(bool upper, uint32_t* a, uint32_t* b) {
    const uint32_t got = Quad<kPerm>(upper ? *a : *b);
    *a = upper ? got : *a;
    *b = upper ? *b : got;
  }

  // Largest magnitude of four, infinity if one of them is not a finite number.
  static __device__ __forceinline__ float Top4(float4 v) {
    const auto mag = [](float x) { return fabsf(x) <= FLT_MAX ? fabsf(x) : INFINITY; };
    return fmaxf(fmaxf(mag(v.x), mag(v.y)), fmaxf(mag(v.z), mag(v.w)));
  }

  static __device__ __forceinline__ uint32_t Codes4(float4 v, float inv, bool finite) {
    const auto code = [inv, finite](float x) {
      const float y = finite ? fminf(fmaxf(__builtin_rintf(x * inv), -127.0f), 127.0f) : 0.0f;
      return static_cast<uint32_t>(static_cast<int32_t>(y)) & 0xFFu;
    };
    return code(v.x) | (code(v.y) << 8) | (code(v.z) << 16) | (code(v.w) << 24);
  }
};

// Work units of a token: with kNorm its n_heads query rows, then the n_kv key rows,
// then the n_kv value rows; D / 16 lanes each.
//
// Plain loads, since the projections before this kernel have just written q, k and v;
// nontemporal stores of the queries; plain stores of the cache's rows, whole lines with
// 16 bytes a lane. Measured at 2811 tokens of 16 + 8 + 8 heads into 8 bits, 75 MB:
// 14.2 us = 5.3 TB/s; with nontemporal loads 17.2, with plain stores of the queries
// 16.0, with write-through ones a tenth more; held to 64 registers (spills) twice as long.
// (Times in this file: the kernel between events that its dispatch carries.)
// One argument: a launch takes longer for every pointer among its arguments (nine of them, 0.5 us of host time).
struct WriteArgs {
  PagedView view;
  const int32_t* seq_ids;
  const int32_t* positions;
  const float* q;
  const float* k;
  const float* v;
  const float* q_norm;
  const float* k_norm;
  const float* tab;
  float* q_out;
  int64_t rope_rows;
  int32_t n_heads;
  float eps;
  uint32_t n_units;
};

template <int D, bool kQ8, bool kNorm>
__global__ __launch_bounds__(kBlock) void PagedWriteKernel(const WriteArgs args) {
  const PagedView view = args.view;
  const int32_t* __restrict__ seq_ids = args.seq_ids;
  const int32_t* __restrict__ positions = args.positions;
  const float* q = args.q;
  const float* __restrict__ k = args.k;
  const float* __restrict__ v = args.v;
  const float* __restrict__ qw = args.q_norm;
  const float* __restrict__ kw = args.k_norm;
  const float* __restrict__ tab = args.tab;
  float* q_out = args.q_out;
  const int64_t rope_rows = args.rope_rows;
  const int32_t n_heads = args.n_heads;
  const float eps = args.eps;
  const uint32_t n_units = args.n_units;
  // the arguments in one batch of scalar loads at entry (the empty asm takes them as scalar inputs), not each before its
  // first use
  asm volatile("" ::"s"(seq_ids), "s"(positions), "s"(q), "s"(k), "s"(v), "s"(qw), "s"(kw), "s"(n_heads), "s"(tab),
               "s"(rope_rows), "s"(eps), "s"(q_out), "s"(n_units), "s"(view.pages), "s"(view.n_seqs), "s"(view.max_pages),
               "s"(view.n_pages), "s"(view.n_kv), "s"(view.page_shift));
  using R = RowOf<D>;
  const int l = threadIdx.x % R::kLanes;
  const uint32_t unit = WorkgroupInStretch() * (kBlock / R::kLanes) + threadIdx.x / R::kLanes;
  if (unit >= n_units) return;
  const uint32_t nq = kNorm ? n_heads : 0;
  const uint32_t per_tok = nq + 2 * view.n_kv;
  const uint32_t token = unit / per_tok;
  const uint32_t j = unit - token * per_tok;
  const int64_t t = token;
  const bool is_q = j < nq;
  const bool is_v = j >= nq + view.n_kv;
  const uint32_t h = is_q ? j : is_v ? j - nq - view.n_kv : j - nq;
  const float* src = is_q ? q + (t * n_heads + h) * D : (is_v ? v : k) + (t * view.n_kv + h) * D;
  const int32_t pos = positions[t];
  const int64_t seq = seq_ids != nullptr ? seq_ids[t] : t;
  Row r = R::Load(src, l);
  Row w{}, trig{};
  if (kNorm && !is_v) {  // a row of the table is read by this token alone: its load starts before the slot is known
    w = R::Load(is_q ? qw : kw, l);
    trig = R::Load(tab + (pos >= 0 && pos < rope_rows ? static_cast<int64_t>(pos) : 0) * D, l);
  }
  Slot slot = dev::FindSlot(view, seq, pos);
  if (slot.state == SlotState::kPadding) return;
  if (kNorm && pos >= rope_rows) slot.state = SlotState::kBad;
  const bool ok = slot.state == SlotState::kOk;
  if (kNorm && !is_v) {
    R::Norm(r, w, eps);
    R::Rotate(r, trig);
  }
  if (is_q) {
    if (!ok) {
      const float nan = __builtin_nanf("");
#pragma unroll
      for (int c = 0; c < 2; ++c) r.a[c] = r.b[c] = make_float4(nan, nan, nan, nan);
    }
    R::StoreStream(q_out + (t * n_heads + h) * D, l, r);
    return;
  }
  if (!ok) return;
  const int64_t row = slot.first + (static_cast<int64_t>(h) << view.page_shift);
  void* pool = const_cast<void*>(is_v ? view.v : view.k);
  if constexpr (kQ8) {
    R::StoreQ8(static_cast<int8_t*>(pool) + row * D, const_cast<float*>(is_v ? view.v_scale : view.k_scale) + row, l,
               r);
  } else {
    R::StoreHalf(static_cast<uint16_t*>(pool) + row * D, l, r);
  }
}

// kN (4 or 8) elements of a cached row as fp32: codes times the scale, or the halves.
template <bool kQ8, int kN>
__device__ __forceinline__ void LoadCached(const void* pool, const float* scale, int64_t row, int64_t at, float (&x)[kN]) {
  if constexpr (kQ8) {
    const float s = scale[row];
    uint32_t w[kN / 4];
    const int8_t* p = static_cast<const int8_t*>(pool) + at;
    if constexpr (kN == 8) {
      const dev::U32x2 d = *reinterpret_cast<const dev::U32x2*>(p);
      w[0] = d.x, w[1] = d.y;
    } else {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
#pragma unroll
    for (int i = 0; i < kN; ++i) x[i] = static_cast<float>(static_cast<int8_t>(w[i / 4] >> (8 * (i & 3)))) * s;
  } else {
    uint32_t w[kN / 2];
    const uint16_t* p = static_cast<const uint16_t*>(pool) + at;
    if constexpr (kN == 8) {
      const dev::U32x4 d = *reinterpret_cast<const dev::U32x4*>(p);
      w[0] = d.x, w[1] = d.y, w[2] = d.z, w[3] = d.w;
    } else {
      const dev::U32x2 d = *reinterpret_cast<const dev::U32x2*>(p);
      w[0] = d.x, w[1] = d.y;
    }
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      x[i] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[i / 2] >> (16 * (i & 1)))));
    }
  }
}

// One 16-byte store: 4 floats, or 8 halves.
template <int kN>
__device__ __forceinline__ void StoreRead(void* out, int64_t at, const float (&x)[kN]) {
  if constexpr (kN == 4) {
    dev::StoreStream4(static_cast<float*>(out) + at, make_float4(x[0], x[1], x[2], x[3]));
  } else {
    const uint2 a = dev::PackHalf4(make_float4(x[0], x[1], x[2], x[3]));
    const uint2 b = dev::PackHalf4(make_float4(x[4], x[5], x[6], x[7]));
    const dev::U32x4 w = {a.x, a.y, b.x, b.y};
    __builtin_nontemporal_store(w, reinterpret_cast<dev::U32x4*>(static_cast<uint16_t*>(out) + at));
  }
}

// One work unit per (token, kv head): a lane moves 16 bytes of output of its key and
// of its value row. Plain loads and nontemporal stores: 10.4 us for 6 x 700 tokens of
// 8 fp16 heads (52 MB, 5.0 TB/s); with nontemporal loads 12.7, with plain stores 11.0.
struct ReadArgs {
  PagedView view;
  const int32_t* seq_ids;
  const int32_t* positions;
  void* k_out;
  void* v_out;
  int64_t token_stride;
  int64_t head_stride;
  uint32_t n_units;
};

template <int D, bool kQ8, bool kF32>
__global__ __launch_bounds__(kBlock) void PagedReadKernel(const ReadArgs args) {
  const PagedView view = args.view;
  const int32_t* __restrict__ seq_ids = args.seq_ids;
  const int32_t* __restrict__ positions = args.positions;
  void* k_out = args.k_out;
  void* v_out = args.v_out;
  const int64_t token_stride = args.token_stride, head_stride = args.head_stride;
  const uint32_t n_units = args.n_units;
  asm volatile("" ::"s"(seq_ids), "s"(positions), "s"(k_out), "s"(v_out), "s"(token_stride), "s"(head_stride),
               "s"(n_units), "s"(view.pages), "s"(view.n_seqs), "s"(view.max_pages), "s"(view.n_pages), "s"(view.n_kv),
               "s"(view.page_shift), "s"(view.k), "s"(view.v), "s"(view.k_scale), "s"(view.v_scale));
  constexpr int kN = kF32 ? 4 : 8;
  constexpr int kLanes = D / kN;
  const int l = threadIdx.x % kLanes;
  const uint32_t unit = WorkgroupInStretch() * (kBlock / kLanes) + threadIdx.x / kLanes;
  if (unit >= n_units) return;
  const uint32_t token = unit / static_cast<uint32_t>(view.n_kv);
  const uint32_t h = unit - token * static_cast<uint32_t>(view.n_kv);
  const int64_t t = token;
  const Slot slot = dev::FindSlot(view, seq_ids != nullptr ? seq_ids[t] : t, positions[t]);
  if (slot.state == SlotState::kPadding) return;
  float kx[kN], vx[kN];
  if (slot.state == SlotState::kOk) {
    const int64_t row = slot.first + (static_cast<int64_t>(h) << view.page_shift);
    LoadCached<kQ8>(view.k, view.k_scale, row, row * D + kN * l, kx);
    LoadCached<kQ8>(view.v, view.v_scale, row, row * D + kN * l, vx);
  } else {
#pragma unroll
    for (int i = 0; i < kN; ++i) kx[i] = vx[i] = __builtin_nanf("");
  }
  const int64_t at = t * token_stride + h * head_stride + kN * l;
  StoreRead(k_out, at, kx);
  StoreRead(v_out, at, vx);
}

void CheckRows(const char* what, const GpuPageTable& table, const int32_t* seq_ids, const int32_t* positions,
               int64_t n_tokens) {
  RPG_CHECK(positions != nullptr, "%s got null positions", what);
  RPG_CHECK(((reinterpret_cast<uintptr_t>(seq_ids) | reinterpret_cast<uintptr_t>(positions)) & 3) == 0,
            "%s: seq_ids and positions have to be 4-byte aligned", what);
  RPG_CHECK(seq_ids != nullptr || n_tokens <= table.n_seqs, "%s: %lld tokens without seq_ids, but %lld sequences",
            what, static_cast<long long>(n_tokens), static_cast<long long>(table.n_seqs));
}

template <bool kNorm>
void LaunchWrite(const char* name, const GpuPagedKv& kv, WriteArgs args, int64_t n_tokens) {
  const int64_t units = n_tokens * ((kNorm ? args.n_heads : 0) + 2 * static_cast<int64_t>(kv.n_kv_heads));
  args.n_units = static_cast<uint32_t>(units);
  const bool q8 = kv.type == kKvQ8;
  auto* kern = kv.head_dim == 128 ? (q8 ? PagedWriteKernel<128, true, kNorm> : PagedWriteKernel<128, false, kNorm>)
                                  : (q8 ? PagedWriteKernel<64, true, kNorm> : PagedWriteKernel<64, false, kNorm>);
  Launch(name, kern, dim3(GridFor(units, kBlock / (kv.head_dim / 16))), dim3(kBlock), args);
}

// Whether a row of `bytes` at t * token_stride + h * head_stride (t < n_tokens, h < n_heads) and another `apart` behind such
// a place share a byte; strides and distances in bytes. For each difference of heads, the difference of tokens that brings
// the two nearest.
bool RowsMeet(int64_t apart, int64_t bytes, int64_t n_tokens, int64_t token_stride, int64_t n_heads, int64_t head_stride) {
  for (int64_t dh = 1 - n_heads; dh < n_heads; ++dh) {
    const int64_t x = apart + dh * head_stride;
    const int64_t whole = -x / token_stride;
    for (int64_t dt = whole - 1; dt <= whole + 1; ++dt) {
      const int64_t at = x + std::clamp(dt, 1 - n_tokens, n_tokens - 1) * token_stride;
      if (at > -bytes && at < bytes) return true;
    }
  }
  return false;
}

// Head rows of a call are counted in 32 bits.
void CheckUnits(const char* what, int64_t n_tokens, int64_t rows_per_token) {
  RPG_CHECK(n_tokens <= 0x7FFFFFFF / rows_per_token, "%s: %lld tokens of %lld rows are too many for one call", what,
            static_cast<long long>(n_tokens), static_cast<long long>(rows_per_token));
}

}  // namespace

void GpuKvWritePaged(const GpuPagedKv& kv, const GpuPageTable& table, const int32_t* seq_ids,
                     const int32_t* positions, const float* k_dev, const float* v_dev, int64_t n_tokens) {
  CheckPagedKv("KvWritePaged", kv, table);
  RPG_CHECK(n_tokens >= 0, "KvWritePaged: %lld tokens", static_cast<long long>(n_tokens));
  if (n_tokens == 0) return;
  CheckRows("KvWritePaged", table, seq_ids, positions, n_tokens);
  RPG_CHECK(k_dev != nullptr && v_dev != nullptr, "KvWritePaged got a null pointer");
  RPG_CHECK(Aligned16(k_dev) && Aligned16(v_dev), "KvWritePaged: k and v have to be 16-byte aligned");
  CheckUnits("KvWritePaged", n_tokens, 2 * static_cast<int64_t>(kv.n_kv_heads));
  LaunchWrite<false>("PagedWriteKernel", kv,
                     WriteArgs{dev::ViewOf(kv, table), seq_ids, positions, nullptr, k_dev, v_dev, nullptr, nullptr, nullptr,
                               nullptr, 0, 0, 0.0f, 0},
                     n_tokens);
}

void GpuQkNormRopeKvPaged(const GpuPagedKv& kv, const GpuPageTable& table, const int32_t* seq_ids,
                          const int32_t* positions, const float* q_dev, const float* k_dev, const float* v_dev,
                          const float* q_norm, const float* k_norm, int32_t n_heads, const float* rope_tab,
                          int64_t rope_rows, int64_t n_tokens, float eps, float* q_out) {
  CheckPagedKv("QkNormRopeKvPaged", kv, table);
  RPG_CHECK(n_tokens >= 0, "QkNormRopeKvPaged: %lld tokens", static_cast<long long>(n_tokens));
  RPG_CHECK(n_heads > 0 && n_heads <= (1 << 20), "QkNormRopeKvPaged: n_heads %d out of range", n_heads);
  RPG_CHECK(rope_rows > 0 && rope_rows <= 0x7FFFFFFF, "QkNormRopeKvPaged: a RoPE table of %lld rows", static_cast<long long>(rope_rows));
  if (n_tokens == 0) return;
  CheckRows("QkNormRopeKvPaged", table, seq_ids, positions, n_tokens);
  RPG_CHECK(q_dev && k_dev && v_dev && q_norm && k_norm && rope_tab && q_out, "QkNormRopeKvPaged got a null pointer");
  RPG_CHECK(Aligned16(q_dev) && Aligned16(k_dev) && Aligned16(v_dev) && Aligned16(q_norm) && Aligned16(k_norm) &&
                Aligned16(rope_tab) && Aligned16(q_out),
            "QkNormRopeKvPaged: every buffer has to be 16-byte aligned");
  CheckUnits("QkNormRopeKvPaged", n_tokens, n_heads + 2 * static_cast<int64_t>(kv.n_kv_heads));
  const int64_t row = kv.head_dim * 4;
  const int64_t q_bytes = n_tokens * n_heads * row, kv_bytes = n_tokens * kv.n_kv_heads * row;
  RPG_CHECK(q_out == q_dev || !Overlap(q_dev, q_bytes, q_out, q_bytes),
            "QkNormRopeKvPaged: q_out has to be q itself or apart from it");
  RPG_CHECK(!Overlap(k_dev, kv_bytes, q_out, q_bytes) && !Overlap(v_dev, kv_bytes, q_out, q_bytes) &&
                !Overlap(q_norm, row, q_out, q_bytes) && !Overlap(k_norm, row, q_out, q_bytes) &&
                !Overlap(rope_tab, rope_rows * row, q_out, q_bytes),
            "QkNormRopeKvPaged: q_out must not overlap k, v, the norms or the RoPE table");
  LaunchWrite<true>("PagedQkNormRopeWriteKernel", kv,
                    WriteArgs{dev::ViewOf(kv, table), seq_ids, positions, q_dev, k_dev, v_dev, q_norm, k_norm, rope_tab,
                              q_out, rope_rows, n_heads, eps, 0},
                    n_tokens);
}

void GpuKvReadPaged(const GpuPagedKv& kv, const GpuPageTable& table, const int32_t* seq_ids,
                    const int32_t* positions, int64_t n_tokens, bool out_f32, void* k_out, void* v_out,
                    int64_t token_stride, int64_t head_stride) {
  CheckPagedKv("KvReadPaged", kv, table);
  RPG_CHECK(n_tokens >= 0, "KvReadPaged: %lld tokens", static_cast<long long>(n_tokens));
  if (n_tokens == 0) return;
  CheckRows("KvReadPaged", table, seq_ids, positions, n_tokens);
  RPG_CHECK(k_out != nullptr && v_out != nullptr, "KvReadPaged got a null pointer");
  RPG_CHECK(Aligned16(k_out) && Aligned16(v_out), "KvReadPaged: k_out and v_out have to be 16-byte aligned");
  const int64_t far = int64_t{1} << 56;
  RPG_CHECK(token_stride >= kv.head_dim && head_stride >= kv.head_dim && token_stride % 8 == 0 &&
                head_stride % 8 == 0 && token_stride < far / n_tokens && head_stride < far / kv.n_kv_heads,
            "KvReadPaged: strides %lld and %lld have to be multiples of 8, at least head_dim",
            static_cast<long long>(token_stride), static_cast<long long>(head_stride));
  RPG_CHECK(token_stride >= (kv.n_kv_heads - 1) * head_stride + kv.head_dim ||
                head_stride >= (n_tokens - 1) * token_stride + kv.head_dim,
            "KvReadPaged: rows of strides %lld and %lld overlap", static_cast<long long>(token_stride),
            static_cast<long long>(head_stride));
  RPG_CHECK(k_out != v_out, "KvReadPaged: k_out and v_out are the same");
  CheckUnits("KvReadPaged", n_tokens, kv.n_kv_heads);
  const int64_t size = out_f32 ? 4 : 2, row = size * kv.head_dim;
  const int64_t span = size * ((n_tokens - 1) * token_stride + (kv.n_kv_heads - 1) * head_stride) + row;
  RPG_CHECK(!Overlap(k_out, span, v_out, span) ||
                !RowsMeet(static_cast<const char*>(v_out) - static_cast<const char*>(k_out), row, n_tokens,
                          size * token_stride, kv.n_kv_heads, size * head_stride),
            "KvReadPaged: rows of k_out and v_out overlap");
  const int64_t units = n_tokens * kv.n_kv_heads;
  const bool q8 = kv.type == kKvQ8;
  auto* kern = kv.head_dim == 128
                   ? (q8 ? (out_f32 ? PagedReadKernel<128, true, true> : PagedReadKernel<128, true, false>)
                         : (out_f32 ? PagedReadKernel<128, false, true> : PagedReadKernel<128, false, false>))
                   : (q8 ? (out_f32 ? PagedReadKernel<64, true, true> : PagedReadKernel<64, true, false>)
                         : (out_f32 ? PagedReadKernel<64, false, true> : PagedReadKernel<64, false, false>));
  Launch("PagedReadKernel", kern, dim3(GridFor(units, kBlock / (kv.head_dim / (out_f32 ? 4 : 8)))), dim3(kBlock),
         ReadArgs{dev::ViewOf(kv, table), seq_ids, positions, k_out, v_out, token_stride, head_stride,
                  static_cast<uint32_t>(units)});
}

}  // namespace rpg
