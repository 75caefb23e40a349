// The paged KV cache's writers and its reader: rows put into pages as fp16 or as
// 8-bit codes with a scale, with or without the q / k norm and rotation in front,
// and rows read back out of pages. The cache's layout and its 8-bit form are
// described in kernels_gpu.h.
//
// Every kernel here moves each byte once and computes a few operations on it, so
// memory bounds it (launch latency for a few tokens). A head row of D elements is
// spread over D / 16 lanes, 16 elements each, arranged as head_row.h arranges 128
// of them over 8 lanes: both members of every rotated pair (i, i + D/2) sit in one
// lane, and the sums and maxima over a row are butterflies over its lanes.
#include <hip/hip_runtime.h>

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

  static __device__ __forceinline__ Row LoadStream(const float* p, int l) {
    Row r;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      r.a[c] = dev::LoadStream4(p + Offset(l, c));
      r.b[c] = dev::LoadStream4(p + D / 2 + Offset(l, c));
    }
    return r;
  }

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

  static __device__ __forceinline__ void StoreHalf(uint16_t* p, int l, const Row& r) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      *reinterpret_cast<uint2*>(p + Offset(l, c)) = dev::PackHalf4(r.a[c]);
      *reinterpret_cast<uint2*>(p + D / 2 + Offset(l, c)) = dev::PackHalf4(r.b[c]);
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
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      *reinterpret_cast<uint32_t*>(p + Offset(l, c)) = Codes4(r.a[c], inv, finite);
      *reinterpret_cast<uint32_t*>(p + D / 2 + Offset(l, c)) = Codes4(r.b[c], inv, finite);
    }
  }

 private:
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
template <int D, bool kQ8, bool kNorm>
__global__ __launch_bounds__(kBlock) void PagedWriteKernel(
    PagedView view, const int32_t* __restrict__ seq_ids, const int32_t* __restrict__ positions, const float* q,
    const float* __restrict__ k, const float* __restrict__ v, const float* __restrict__ qw,
    const float* __restrict__ kw, int32_t n_heads, const float* __restrict__ tab, int64_t rope_rows, float eps,
    float* q_out, int64_t n_units) {
  using R = RowOf<D>;
  const int l = threadIdx.x % R::kLanes;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * (kBlock / R::kLanes) + threadIdx.x / R::kLanes;
  if (unit >= n_units) return;
  const int32_t nq = kNorm ? n_heads : 0;
  const int32_t per_tok = nq + 2 * view.n_kv;
  const int64_t t = unit / per_tok;
  const int32_t j = static_cast<int32_t>(unit - t * per_tok);
  const bool is_q = j < nq;
  const bool is_v = j >= nq + view.n_kv;
  const int32_t h = is_q ? j : is_v ? j - nq - view.n_kv : j - nq;
  const float* src = is_q ? q + (t * n_heads + h) * D : (is_v ? v : k) + (t * view.n_kv + h) * D;
  Row r = R::LoadStream(src, l);
  const int32_t pos = positions[t];
  Slot slot = dev::FindSlot(view, seq_ids != nullptr ? seq_ids[t] : t, pos);
  if (slot.state == SlotState::kPadding) return;
  if (kNorm && pos >= rope_rows) slot.state = SlotState::kBad;
  const bool ok = slot.state == SlotState::kOk;
  if (kNorm && !is_v && ok) {
    const Row trig = R::Load(tab + static_cast<int64_t>(pos) * D, l);
    R::Norm(r, R::Load(is_q ? qw : kw, l), eps);
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

// Eight elements of a cached row as fp32: codes times the scale, or the halves.
template <bool kQ8>
__device__ __forceinline__ void LoadCached8(const void* pool, const float* scale, int64_t row, int64_t at, float (&x)[8]) {
  if constexpr (kQ8) {
    const float s = scale[row];
    const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const int8_t*>(pool) + at);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = static_cast<float>(static_cast<int8_t>((i < 4 ? w.x : w.y) >> (8 * (i & 3)))) * s;
    }
  } else {
    const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(pool) + at);
    const uint32_t d[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(d[i / 2] >> (16 * (i & 1)))));
    }
  }
}

template <bool kF32>
__device__ __forceinline__ void StoreRead8(void* out, int64_t at, const float (&x)[8]) {
  if constexpr (kF32) {
    float* p = static_cast<float*>(out) + at;
    dev::StoreStream4(p, make_float4(x[0], x[1], x[2], x[3]));
    dev::StoreStream4(p + 4, make_float4(x[4], x[5], x[6], x[7]));
  } else {
    const uint2 a = dev::PackHalf4(make_float4(x[0], x[1], x[2], x[3]));
    const uint2 b = dev::PackHalf4(make_float4(x[4], x[5], x[6], x[7]));
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + at) = make_uint4(a.x, a.y, b.x, b.y);
  }
}

// One work unit per (token, kv head): D / 8 lanes move 8 elements each of its key
// and of its value row.
template <int D, bool kQ8, bool kF32>
__global__ __launch_bounds__(kBlock) void PagedReadKernel(PagedView view, const int32_t* __restrict__ seq_ids,
                                                          const int32_t* __restrict__ positions, void* k_out,
                                                          void* v_out, int64_t token_stride, int64_t head_stride,
                                                          int64_t n_units) {
  constexpr int kLanes = D / 8;
  const int l = threadIdx.x % kLanes;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * (kBlock / kLanes) + threadIdx.x / kLanes;
  if (unit >= n_units) return;
  const int64_t t = unit / view.n_kv;
  const int32_t h = static_cast<int32_t>(unit - t * view.n_kv);
  const Slot slot = dev::FindSlot(view, seq_ids != nullptr ? seq_ids[t] : t, positions[t]);
  if (slot.state == SlotState::kPadding) return;
  float kx[8], vx[8];
  if (slot.state == SlotState::kOk) {
    const int64_t row = slot.first + (static_cast<int64_t>(h) << view.page_shift);
    LoadCached8<kQ8>(view.k, view.k_scale, row, row * D + 8 * l, kx);
    LoadCached8<kQ8>(view.v, view.v_scale, row, row * D + 8 * l, vx);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) kx[i] = vx[i] = __builtin_nanf("");
  }
  const int64_t at = t * token_stride + h * head_stride + 8 * l;
  StoreRead8<kF32>(k_out, at, kx);
  StoreRead8<kF32>(v_out, at, vx);
}

void CheckRows(const char* what, const GpuPageTable& table, const int32_t* seq_ids, const int32_t* positions,
               int64_t n_tokens) {
  RPG_CHECK(positions != nullptr, "%s got null positions", what);
  RPG_CHECK(seq_ids != nullptr || n_tokens <= table.n_seqs, "%s: %lld tokens without seq_ids, but %lld sequences",
            what, static_cast<long long>(n_tokens), static_cast<long long>(table.n_seqs));
}

template <bool kNorm>
void LaunchWrite(const char* name, const GpuPagedKv& kv, const GpuPageTable& table, const int32_t* seq_ids,
                 const int32_t* positions, const float* q, const float* k, const float* v, const float* qw,
                 const float* kw, int32_t n_heads, const float* tab, int64_t rope_rows, float eps, float* q_out,
                 int64_t n_tokens) {
  const int64_t units = n_tokens * ((kNorm ? n_heads : 0) + 2 * static_cast<int64_t>(kv.n_kv_heads));
  const bool q8 = kv.type == kKvQ8;
  auto* kern = kv.head_dim == 128 ? (q8 ? PagedWriteKernel<128, true, kNorm> : PagedWriteKernel<128, false, kNorm>)
                                  : (q8 ? PagedWriteKernel<64, true, kNorm> : PagedWriteKernel<64, false, kNorm>);
  Launch(name, kern, dim3(GridFor(units, kBlock / (kv.head_dim / 16))), dim3(kBlock), dev::ViewOf(kv, table), seq_ids,
         positions, q, k, v, qw, kw, n_heads, tab, rope_rows, eps, q_out, units);
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
  LaunchWrite<false>("PagedWriteKernel", kv, table, seq_ids, positions, nullptr, k_dev, v_dev, nullptr, nullptr, 0,
                     nullptr, 0, 0.0f, nullptr, n_tokens);
}

void GpuQkNormRopeKvPaged(const GpuPagedKv& kv, const GpuPageTable& table, const int32_t* seq_ids,
                          const int32_t* positions, const float* q_dev, const float* k_dev, const float* v_dev,
                          const float* q_norm, const float* k_norm, int32_t n_heads, const float* rope_tab,
                          int64_t rope_rows, int64_t n_tokens, float eps, float* q_out) {
  CheckPagedKv("QkNormRopeKvPaged", kv, table);
  RPG_CHECK(n_tokens >= 0, "QkNormRopeKvPaged: %lld tokens", static_cast<long long>(n_tokens));
  RPG_CHECK(n_heads > 0 && n_heads <= (1 << 20), "QkNormRopeKvPaged: n_heads %d out of range", n_heads);
  RPG_CHECK(rope_rows > 0, "QkNormRopeKvPaged: a RoPE table of %lld rows", static_cast<long long>(rope_rows));
  if (n_tokens == 0) return;
  CheckRows("QkNormRopeKvPaged", table, seq_ids, positions, n_tokens);
  RPG_CHECK(q_dev && k_dev && v_dev && q_norm && k_norm && rope_tab && q_out, "QkNormRopeKvPaged got a null pointer");
  RPG_CHECK(Aligned16(q_dev) && Aligned16(k_dev) && Aligned16(v_dev) && Aligned16(q_norm) && Aligned16(k_norm) &&
                Aligned16(rope_tab) && Aligned16(q_out),
            "QkNormRopeKvPaged: every buffer has to be 16-byte aligned");
  const int64_t q_bytes = n_tokens * n_heads * kv.head_dim * 4;
  RPG_CHECK(q_out == q_dev || !Overlap(q_dev, q_bytes, q_out, q_bytes),
            "QkNormRopeKvPaged: q_out has to be q itself or apart from it");
  LaunchWrite<true>("PagedQkNormRopeWriteKernel", kv, table, seq_ids, positions, q_dev, k_dev, v_dev, q_norm, k_norm,
                    n_heads, rope_tab, rope_rows, eps, q_out, n_tokens);
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
  const int64_t units = n_tokens * kv.n_kv_heads;
  const bool q8 = kv.type == kKvQ8;
  auto* kern = kv.head_dim == 128
                   ? (q8 ? (out_f32 ? PagedReadKernel<128, true, true> : PagedReadKernel<128, true, false>)
                         : (out_f32 ? PagedReadKernel<128, false, true> : PagedReadKernel<128, false, false>))
                   : (q8 ? (out_f32 ? PagedReadKernel<64, true, true> : PagedReadKernel<64, true, false>)
                         : (out_f32 ? PagedReadKernel<64, false, true> : PagedReadKernel<64, false, false>));
  Launch("PagedReadKernel", kern, dim3(GridFor(units, kBlock / (kv.head_dim / 8))), dim3(kBlock),
         dev::ViewOf(kv, table), seq_ids, positions, k_out, v_out, token_stride, head_stride, units);
}

}  // namespace rpg
