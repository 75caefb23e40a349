// The next tokens of a batch of conversations, from given random numbers (the semantics
// are listed in sampler_gpu.h).
//
// Three launches, the first of which reads the logits once, in slices of 4096:
//   SampleSlices   each workgroup keeps a slice in registers: its largest value m_s, and of what its weights
//                  2^((x - m_s) log2(e) / T) come to, sums by value: bins an eighth of an octave wide (a twelfth of a nat,
//                  for T above 1), whose borders are the same in all slices, counted and weighed upwards from the top. The
//                  row's last workgroup to arrive joins the slices, each by 2^((m_s - m) log2(e) / T), and finds between
//                  which bins each filter cuts: what lies above these bins is kept, what lies below is not;
//   SampleCollect  what lies in them (some dozen to a few thousand values) is collected, in index order, from the slices that
//                  have any;
//   SampleChoose   a workgroup for each row cuts there exactly, by radix selection, adds up the slices' kept weights, finds
//                  u's place among them and walks that one slice.
// Weights are formed in double, which on this card costs what fp32 does, and summed as integers wherever atomics or a
// border depend on it, so that results are the same from run to run.
//
// What bounds it: reading the logits once and forming their weights; one row is the chain of round trips.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "attention_dev.h"
#include "block_dev.h"
#include "dev_util.h"
#include "kernels_gpu.h"
#include "launch.h"
#include "paged_kv.h"
#include "sampler_gpu.h"

namespace rpg {
namespace {

using namespace block;

constexpr int kSlice = 4096;
constexpr int kEach = kSlice / kThreads;
constexpr int kMaxSlices = static_cast<int>(kSamplerMaxVocab / kSlice);
constexpr int kSlicesEach = kMaxSlices / kThreads;
constexpr int kBins = 256;         // of a slice; the last has all that is further down
constexpr int kInLds = 8192;       // candidates that are kept there
constexpr int kRowsAtOnce = 2048;  // rows of a launch: their counters have a place of their own in the workspace
constexpr int kCounterBytes = 128;
// A slice's sums, in one number: count in the upper 13 bits, weight in units of 2^-38 of its largest in the lower 51.
constexpr int kWeightBits = 51;
constexpr int kSliceUnits = 38;
static_assert((int64_t(kSlice) << kSliceUnits) < (int64_t(1) << kWeightBits) && kSlice < (1 << (64 - kWeightBits)), "");
constexpr int kDevicePolicy = 16;  // of stores that the last workgroup to arrive reads

// ---------------------------------------------------------------- order and weights

// What a logit counts as: NaN as minus infinity, plus infinity as the largest number.
__device__ __forceinline__ float Clean(float x) { return x != x ? -INFINITY : fminf(x, FLT_MAX); }

// Order-preserving map onto uint32, both zeros alike, and its inverse.
__device__ __forceinline__ uint32_t KeyOf(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float ValueOf(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7FFFFFFFu) : ~key);
}

// 2^f for f in [-1/2, 1/2], 1 + f g(f) with g the polynomial of degree 7 through 2^f's own at the Chebyshev nodes: within
// 2^-38 of the value, and exactly 1 at 0.
__device__ __forceinline__ double Exp2Near(double f) {
  double p = fma(0x1.63b2d797a3663p-20, f, 0x1.00c0e4e151fbep-16);
  p = fma(p, f, 0x1.4308c7183cd99p-13);
  p = fma(p, f, 0x1.5d877598350dap-10);
  p = fma(p, f, 0x1.3b2ab70ad256bp-7);
  p = fma(p, f, 0x1.c6b08da70cce3p-5);
  p = fma(p, f, 0x1.ebfbdff82a734p-3);
  p = fma(p, f, 0x1.62e42fef9cc69p-1);
  return fma(p, f, 1.0);
}
// 2^(v + bits) for v <= 0; below 2^-1000, and for a NaN, next to nothing.
__device__ __forceinline__ double Exp2Down(double v, int bits) {
  v = fmax(v, -1000.0);
  const double k = rint(v);
  return ldexp(Exp2Near(v - k), static_cast<int>(k) + bits);
}
// A slice's sum of one value of weight 2^v, v <= 0 (any that counts for nothing, down to minus infinity).
__device__ __forceinline__ uint64_t OneOf(double v) {
  v = fmax(v, -200.0);
  // 1.5 * 2^52 added rounds v to a whole number, the low word; 2^52 added to a weight leaves its whole units
  const double shifted = v + 0x1.8p52;
  const int k = static_cast<int>(__builtin_bit_cast(uint64_t, shifted));
  const uint64_t near = __builtin_bit_cast(uint64_t, Exp2Near(v - (shifted - 0x1.8p52)));
  const double scaled =
      __builtin_bit_cast(double, near + (static_cast<uint64_t>(static_cast<uint32_t>(k + kSliceUnits) << 20) << 32));
  const uint64_t bits = __builtin_bit_cast(uint64_t, scaled + 0x1p52);
  return bits - (uint64_t(0x43300000u - (1u << (kWeightBits - 32))) << 32);
}
__device__ __forceinline__ uint32_t CountOf(uint64_t sum) { return static_cast<uint32_t>(sum >> kWeightBits); }
__device__ __forceinline__ double WeightOf(uint64_t sum) {
  return static_cast<double>(sum & ((uint64_t(1) << kWeightBits) - 1)) * (1.0 / static_cast<double>(uint64_t(1) << kSliceUnits));
}

// A row's settings.
struct Setting {
  float t, p, m, u;
  int32_t k;
  bool greedy;
  double by;     // log2(e) / T
  float bin_by;  // bins to a logit

  __device__ __forceinline__ bool OnP() const { return p > 0.0f && p < 1.0f; }
  __device__ __forceinline__ bool Filters() const { return k > 0 || OnP() || m > 0.0f; }
  // The number of x's bin: falls with x, whatever the rounding. x is no NaN.
  __device__ __forceinline__ int32_t BinOf(float x) const {
    return static_cast<int32_t>(floorf(__builtin_amdgcn_fmed3f(x * bin_by, -2e9f, 2e9f)));
  }
  // That bin counted down from bin `top`, of which x's is not above.
  __device__ __forceinline__ int BinBelow(int32_t top, float x) const {
    return static_cast<int>(min(static_cast<uint32_t>(top) - static_cast<uint32_t>(BinOf(x)), static_cast<uint32_t>(kBins - 1)));
  }
};

struct SampleArgs {
  const float* logits;
  int64_t row_stride;
  int32_t n;
  int32_t slices;
  int32_t units;  // s: in the last step weights are whole numbers of 2^-s
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  const float* u;
  int32_t* tokens;
  float* probs;
  char* workspace;
  int32_t first_row;
};

__device__ __forceinline__ Setting SettingOf(const SampleArgs& a, int64_t r) {
  Setting s;
  s.t = a.temperature != nullptr ? a.temperature[r] : 1.0f;
  s.k = a.top_k != nullptr ? a.top_k[r] : 0;
  s.p = a.top_p != nullptr ? a.top_p[r] : 1.0f;
  s.m = a.min_p != nullptr && a.min_p[r] > 0.0f ? fminf(a.min_p[r], 1.0f) : 0.0f;
  s.u = a.u[r];
  s.greedy = !(s.t > 0.0f);
  s.by = 1.4426950408889634 / static_cast<double>(s.t);
  s.bin_by = s.greedy ? 0.0f : fminf(11.541560f * fmaxf(1.0f, 1.0f / s.t), 1e30f);
  return s;
}

// ---------------------------------------------------------------- a row's place in the workspace

struct SliceSums {  // of one slice
  float top;
  int32_t top_index;  // where that is looked for: the first of it
  uint64_t sum;
};

enum class Kind : int32_t { kDone, kAll, kCut };
struct Plan {  // what the first launch finds out for the others
  Kind kind;
  float top;
  int32_t top_bin;
  int32_t hi, lo;                // the bins below the row's top one that are collected
  uint32_t cut_k, cut_p, cut_m;  // filters that may cut there; cut_p 2: of what top_k leaves
  uint32_t base_count;           // values above these bins
  uint32_t candidates;
  double base;                   // their weight
  double all;                    // the weight of all
};

__host__ __device__ constexpr int64_t RoundUp(int64_t x) { return (x + 127) / 128 * 128; }
struct RowPlace {
  int64_t sums, above, offsets, bins, keys, bytes;  // the plan is in front
  __host__ __device__ explicit RowPlace(int32_t slices) {
    sums = RoundUp(sizeof(Plan));
    above = sums + RoundUp(slices * sizeof(SliceSums));
    offsets = above + RoundUp(slices * 8);
    bins = offsets + RoundUp((slices + 1) * 4);
    keys = bins + RoundUp(static_cast<int64_t>(slices) * kBins * 8);
    bytes = keys + static_cast<int64_t>(slices) * kSlice * 4;
  }
};
constexpr int64_t kCounters = static_cast<int64_t>(kRowsAtOnce) * kCounterBytes;

struct Row {  // of the logits and the workspace
  int64_t r;
  RowPlace place;
  char* at;
  __amdgpu_buffer_rsrc_t logits;
  int32_t n;

  __device__ __forceinline__ Row(const SampleArgs& a, uint32_t in_launch)
      : r(a.first_row + static_cast<int64_t>(in_launch)),
        place(a.slices),
        at(a.workspace + kCounters + in_launch * place.bytes),
        logits(dev::OutResource(const_cast<float*>(a.logits) + r * a.row_stride, 4u * static_cast<uint32_t>(a.n))),
        n(a.n) {}
  __device__ __forceinline__ Plan* ThePlan() const { return reinterpret_cast<Plan*>(at); }
  __device__ __forceinline__ SliceSums* Sums() const { return reinterpret_cast<SliceSums*>(at + place.sums); }
  __device__ __forceinline__ double* Above() const { return reinterpret_cast<double*>(at + place.above); }
  __device__ __forceinline__ int32_t* Offsets() const { return reinterpret_cast<int32_t*>(at + place.offsets); }
  // Of slice s, the sums of its bins down to each.
  __device__ __forceinline__ uint64_t* Bins(int s) const {
    return reinterpret_cast<uint64_t*>(at + place.bins) + static_cast<int64_t>(s) * kBins;
  }
  __device__ __forceinline__ uint32_t* Keys() const { return reinterpret_cast<uint32_t*>(at + place.keys); }
  // Four logits from i on; what lies behind the row's end is minus infinity.
  __device__ __forceinline__ float4 Load(int32_t i) const {
    const float4 x = dev::LoadBuf4<0>(logits, 4u * static_cast<uint32_t>(i));
    return make_float4(i < n ? Clean(x.x) : -INFINITY, i + 1 < n ? Clean(x.y) : -INFINITY,
                       i + 2 < n ? Clean(x.z) : -INFINITY, i + 3 < n ? Clean(x.w) : -INFINITY);
  }
};

// ---------------------------------------------------------------- a workgroup's sums

__device__ __forceinline__ uint64_t BlockSum(uint64_t x, uint64_t* sh) {
  uint64_t total;
  BlockExclScan(x, sh, &total);
  return total;
}
__device__ __forceinline__ uint64_t BlockMaxU64(uint64_t x, uint64_t* sh) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const uint64_t o = __shfl_xor(x, off, 64);
    x = o > x ? o : x;
  }
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = x;
  __syncthreads();
  uint64_t r = sh[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) r = sh[w] > r ? sh[w] : r;
  __syncthreads();
  return r;
}
// The sum of doubles over the threads before this one, in one order; *total that over all.
__device__ __forceinline__ double BlockBeforeD(double x, double* sh, double* total) {
  double upto = x;
  upto += DppDbl<0x111>(upto, 0.0);
  upto += DppDbl<0x112>(upto, 0.0);
  upto += DppDbl<0x114>(upto, 0.0);
  upto += DppDbl<0x118>(upto, 0.0);
  upto += DppDbl<0x142, 0xA>(upto, 0.0);
  upto += DppDbl<0x143, 0xC>(upto, 0.0);
  const double mine = __shfl_up(upto, 1, 64);
  if ((threadIdx.x & 63) == 63) sh[threadIdx.x >> 6] = upto;
  __syncthreads();
  double base = 0.0, all = 0.0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w == static_cast<int>(threadIdx.x >> 6)) base = all;
    all += sh[w];
  }
  __syncthreads();
  *total = all;
  return (threadIdx.x & 63) == 0 ? base : base + mine;
}

// ---------------------------------------------------------------- the slices

struct JoinShared {
  double scale[kMaxSlices];  // of a slice's weights
  int32_t off[kMaxSlices];   // bins that a slice's top one lies below the row's, at most all
  double weight[kBins];      // of all bins down to one
  uint32_t count[kBins];
  uint32_t found[4];
};

// The row's last workgroup: where its filters cut.
__device__ __forceinline__ void JoinSlices(const SampleArgs& a, const Setting& set, const Row& row, JoinShared& sh,
                                           uint64_t* parts, double* dparts, float* fparts) {
  const int tid = threadIdx.x;
  SliceSums mine[kSlicesEach];
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kSlicesEach; ++i) {
    const int s = tid + i * kThreads;
    mine[i] = s < a.slices ? row.Sums()[s] : SliceSums{-INFINITY, 0, 0};
    top = fmaxf(top, mine[i].top);
  }
  top = BlockMax(top, fparts);
  if (top == -INFINITY || set.greedy) {
    uint64_t first = 0;
#pragma unroll
    for (int i = 0; i < kSlicesEach; ++i) {
      if (mine[i].top == top) first = max(first, static_cast<uint64_t>(0x7FFFFFFF - mine[i].top_index));
    }
    first = BlockMaxU64(first, parts);
    if (tid == 0) {
      const bool none = top == -INFINITY;
      a.tokens[row.r] = none ? -1 : 0x7FFFFFFF - static_cast<int32_t>(first);
      if (a.probs != nullptr) a.probs[row.r] = none ? 0.0f : 1.0f;
      row.ThePlan()->kind = Kind::kDone;
    }
    return;
  }
  const int32_t top_bin = set.BinOf(top);
  double all = 0.0;
  uint64_t live = 0;
#pragma unroll
  for (int i = 0; i < kSlicesEach; ++i) {
    const int s = tid + i * kThreads;
    if (s < a.slices) {
      const bool any = mine[i].top > -INFINITY;
      const double scale =
          any ? Exp2Down((static_cast<double>(mine[i].top) - static_cast<double>(top)) * set.by, 0) : 0.0;
      sh.scale[s] = scale;
      sh.off[s] = any ? set.BinBelow(top_bin, mine[i].top) : kBins - 1;
      all += scale * WeightOf(mine[i].sum);
      live += CountOf(mine[i].sum);
    }
  }
  if (tid < 4) sh.found[tid] = kBins - 1;
  all = BlockSumD(all, dparts);
  live = BlockSum(live, parts);

  // a slice's sum over the row's bins down to j
  const auto sum_at = [&](int s, int j) -> uint64_t {
    const int in_slice = j == kBins - 1 ? j : j - sh.off[s];
    return in_slice >= 0 ? row.Bins(s)[in_slice] : 0;
  };
  const bool on_k = set.k > 0 && static_cast<uint64_t>(set.k) < live, on_p = set.OnP(), on_m = set.m > 0.0f;
  if (!on_k && !on_p && !on_m) {
#pragma unroll
    for (int i = 0; i < kSlicesEach; ++i) {
      const int s = tid + i * kThreads;
      if (s < a.slices) row.Above()[s] = sh.scale[s] * WeightOf(mine[i].sum);
    }
    if (tid == 0) *row.ThePlan() = Plan{Kind::kAll, top, top_bin, kBins, kBins, 0, 0, 0, 0, 0, 0.0, all};
    return;
  }
  double weight = 0.0;
  uint32_t count = 0;
  static_assert(kThreads == kBins, "a bin to a thread");
  constexpr int kBatch = 16;
#pragma unroll 1
  for (int s0 = 0; s0 < a.slices; s0 += kBatch) {
    uint64_t sums[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) sums[i] = s0 + i < a.slices ? sum_at(s0 + i, tid) : 0;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (s0 + i < a.slices) weight += sh.scale[s0 + i] * WeightOf(sums[i]);
      count += CountOf(sums[i]);
    }
  }
  sh.weight[tid] = weight;
  sh.count[tid] = count;
  __syncthreads();
  const uint32_t before_count = tid == 0 ? 0 : sh.count[tid - 1];
  const double before_weight = tid == 0 ? 0.0 : sh.weight[tid - 1];
  // top_k's bin
  const uint32_t k = static_cast<uint32_t>(set.k);
  if (on_k && before_count < k && k <= count) sh.found[0] = static_cast<uint32_t>(tid);
  __syncthreads();
  const int bin_k = on_k ? static_cast<int>(sh.found[0]) : kBins - 1;
  // top_p's: between those of the least and the most that what top_k leaves may weigh, and a rounding more
  const double most = sh.weight[bin_k], least = !on_k ? most : bin_k == 0 ? 0.0 : sh.weight[bin_k - 1];
  const double p = static_cast<double>(set.p);
  const double goal_hi = p * least * (1.0 - 0x1p-40), goal_lo = fmin(p * most * (1.0 + 0x1p-40), most);
  if (on_p && weight >= goal_hi && (tid == 0 || before_weight < goal_hi)) sh.found[1] = static_cast<uint32_t>(tid);
  if (on_p && weight >= goal_lo && (tid == 0 || before_weight < goal_lo)) sh.found[2] = static_cast<uint32_t>(tid);
  __syncthreads();
  const int p_hi = static_cast<int>(sh.found[1]), p_lo = static_cast<int>(sh.found[2]);
  // min_p's: from the next number above its border to the next below
  int m_hi = kBins - 1, m_lo = kBins - 1;
  if (on_m) {
    const double border = static_cast<double>(top) + log(static_cast<double>(set.m)) * static_cast<double>(set.t);
    const float near = static_cast<float>(fmax(border, -static_cast<double>(FLT_MAX)));
    m_hi = set.BinBelow(top_bin, fminf(nextafterf(near, INFINITY), top));
    m_lo = set.BinBelow(top_bin, nextafterf(near, -INFINITY));
  }

  // The cut that counts is the highest: filters that start below where another has cut for sure do not matter. top_p's
  // place needs what top_k leaves, and so the bins down to its.
  const int sure = min(on_k ? bin_k : kBins - 1, min(on_p ? p_lo : kBins - 1, m_lo));
  const bool cut_k = on_k && bin_k <= sure, cut_p = on_p && p_hi <= sure, cut_m = on_m && m_hi <= sure;
  int hi = kBins - 1, lo = 0;
  if (cut_k) hi = min(hi, bin_k), lo = max(lo, bin_k);
  if (cut_p) hi = min(hi, p_hi), lo = max(lo, on_k ? bin_k : p_lo);
  if (cut_m) hi = min(hi, m_hi), lo = max(lo, m_lo);

  // of each slice: the weight above these bins, and where its values in them go
  uint32_t placed = 0;
#pragma unroll 1
  for (int s0 = 0; s0 < a.slices; s0 += kThreads) {
    const int s = s0 + tid;
    uint64_t in = 0;
    if (s < a.slices) {
      const uint64_t above = hi > 0 ? sum_at(s, hi - 1) : 0, upto = sum_at(s, lo);
      row.Above()[s] = sh.scale[s] * WeightOf(above);
      in = CountOf(upto) - CountOf(above);
    }
    uint64_t sum;
    const uint64_t before = BlockExclScan(in, parts, &sum);
    if (s < a.slices) row.Offsets()[s] = static_cast<int32_t>(placed + before);
    placed += static_cast<uint32_t>(sum);
  }
  if (tid == 0) {
    row.Offsets()[a.slices] = static_cast<int32_t>(placed);
    *row.ThePlan() = Plan{Kind::kCut, top, top_bin, hi, lo, cut_k ? 1u : 0u, cut_p ? (on_k ? 2u : 1u) : 0u,
                          cut_m ? 1u : 0u, hi > 0 ? sh.count[hi - 1] : 0u, placed, hi > 0 ? sh.weight[hi - 1] : 0.0,
                          sh.weight[kBins - 1]};
  }
}

// Grid: slices times rows.
__global__ __launch_bounds__(kThreads) void SampleSlicesKernel(const SampleArgs a) {
  struct SliceShared {
    uint64_t bins[kWaves][kBins];
  };
  __shared__ union {
    SliceShared slice;
    JoinShared join;
  } sh;
  __shared__ uint64_t parts[kWaves];
  __shared__ double dparts[kWaves];
  __shared__ float fparts[kWaves];
  __shared__ int first;
  const int tid = threadIdx.x;
  const uint32_t in_launch = blockIdx.x / static_cast<uint32_t>(a.slices);
  const int slice = static_cast<int>(blockIdx.x - in_launch * static_cast<uint32_t>(a.slices));
  const Row row(a, in_launch);
  float x[kEach];
#pragma unroll
  for (int i = 0; i < kEach; i += 4) {
    const float4 v = row.Load(slice * kSlice + i * kThreads + 4 * tid);
    x[i] = v.x, x[i + 1] = v.y, x[i + 2] = v.z, x[i + 3] = v.w;
  }
  const Setting set = SettingOf(a, row.r);
  const bool filters = !set.greedy && set.Filters();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) sh.slice.bins[w][tid] = 0;
  if (tid == 0) first = 0x7FFFFFFF;
  float top = x[0];
#pragma unroll
  for (int i = 1; i < kEach; ++i) top = fmaxf(top, x[i]);
  top = BlockMax(top, fparts);
  uint64_t sum = 0;
  if (set.greedy) {
#pragma unroll
    for (int i = kEach - 1; i >= 0; --i) {
      if (x[i] == top) atomicMin(&first, slice * kSlice + (i & ~3) * kThreads + 4 * tid + (i & 3));
    }
    __syncthreads();
  } else {
    const int32_t top_bin = set.BinOf(top);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (x[i] == -INFINITY) continue;
      const uint64_t add = OneOf((static_cast<double>(x[i]) - static_cast<double>(top)) * set.by);
      if (filters) {
        atomicAdd(reinterpret_cast<unsigned long long*>(&sh.slice.bins[tid >> 6][set.BinBelow(top_bin, x[i])]),
                  static_cast<unsigned long long>(add));
      } else {
        sum += add;
      }
    }
    if (filters) {
      __syncthreads();
      uint64_t mine = 0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) mine += sh.slice.bins[w][tid];
      const uint64_t before = BlockExclScan(mine, parts, &sum);
      __hip_atomic_store(row.Bins(slice) + tid, before + mine, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    } else {
      sum = BlockSum(sum, parts);
    }
  }
  if (tid == 0) {
    const __amdgpu_buffer_rsrc_t rs = dev::OutResource(row.Sums() + slice, sizeof(SliceSums));
    dev::StoreBufU4<kDevicePolicy>(rs, 0, make_uint4(__float_as_uint(top), static_cast<uint32_t>(first),
                                                     static_cast<uint32_t>(sum), static_cast<uint32_t>(sum >> 32)));
  }
  // stored at device scope, acknowledged, counted: the last one sees all of it behind its fence
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) first = attn::Count(a.workspace, in_launch * (kCounterBytes / 4), static_cast<uint32_t>(a.slices));
  __syncthreads();
  if (__builtin_amdgcn_readfirstlane(first) == 0) return;
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
  JoinSlices(a, set, row, sh.join, parts, dparts, fparts);
}

// ---------------------------------------------------------------- the candidates

// Grid: slices times rows. In index order: four rounds of four neighbours to a thread, whose counts are summed as one number.
__global__ __launch_bounds__(kThreads) void SampleCollectKernel(const SampleArgs a) {
  __shared__ uint64_t parts[kWaves];
  const int tid = threadIdx.x;
  const uint32_t in_launch = blockIdx.x / static_cast<uint32_t>(a.slices);
  const int slice = static_cast<int>(blockIdx.x - in_launch * static_cast<uint32_t>(a.slices));
  const Row row(a, in_launch);
  const Plan plan = *row.ThePlan();
  const int32_t to = row.Offsets()[slice], end = row.Offsets()[slice + 1];
  if (plan.kind != Kind::kCut || to == end) return;
  const Setting set = SettingOf(a, row.r);
  float x[kEach];
#pragma unroll
  for (int i = 0; i < kEach; i += 4) {
    const float4 v = row.Load(slice * kSlice + i * kThreads + 4 * tid);
    x[i] = v.x, x[i + 1] = v.y, x[i + 2] = v.z, x[i + 3] = v.w;
  }
  uint32_t in = 0;
  uint64_t counts = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int j = set.BinBelow(plan.top_bin, x[i]);
    const bool takes = x[i] > -INFINITY && j >= plan.hi && j <= plan.lo;
    in |= takes ? 1u << i : 0u;
    counts += takes ? uint64_t(1) << (16 * (i / 4)) : 0;
  }
  uint64_t total;
  const uint64_t before = BlockExclScan(counts, parts, &total);
  uint32_t* const keys = row.Keys() + to;
  uint32_t round = 0;
#pragma unroll
  for (int i = 0; i < kEach; i += 4) {
    uint32_t next = round + static_cast<uint32_t>(before >> (4 * i) & 0xFFFF);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if (in >> (i + c) & 1) keys[next++] = KeyOf(x[i + c]);
    }
    round += static_cast<uint32_t>(total >> (4 * i) & 0xFFFF);
  }
}

// ---------------------------------------------------------------- the choice

struct ChooseShared {
  uint32_t keys[kInLds];
  uint64_t bins[256];
  double kept[kMaxSlices];       // weight of a slice
  uint64_t kept_in[kMaxSlices];  // of its candidates, in whole units
  uint32_t ties[kMaxSlices];     // candidates of the cut's key
  uint32_t first[kMaxSlices];    // of these those that are kept
  int32_t offsets[kMaxSlices + 1];
  uint64_t found[2];
  uint64_t parts[kWaves];
  double dparts[kWaves];
  int32_t slice;
  double before;
};

// Kept are the keys above `key`, and of those equal to it the first `ties` in index order.
struct Cut {
  uint32_t key = 0;
  uint64_t ties = 0;
};

// A row's weights, in units of 2^-bits.
struct Units {
  float top;
  double by;
  int32_t bits;
  __device__ __forceinline__ double Of(float x) const {
    return Exp2Down((static_cast<double>(x) - static_cast<double>(top)) * by, bits);
  }
  static __device__ __forceinline__ uint64_t Whole(double of) { return static_cast<uint64_t>(of + 0.5); }
  __device__ __forceinline__ uint64_t OfKey(uint32_t key) const { return Whole(Of(ValueOf(key))); }
};

// The cut after the fewest first candidates, in order, whose amounts (1, or their weight) reach `goal`, among those that
// `cut` keeps: radix selection from the upper of the `width` bits down in which keys, less the least, differ. The amounts
// of all ties of cut.key enter, which decides nothing: it is the last key.
template <class Keys>
__device__ __forceinline__ Cut Select(const Keys& key_at, uint32_t n, uint32_t least, int width, const Units& units,
                                      bool by_weight, const Cut& cut, uint64_t goal, ChooseShared& sh) {
  uint32_t prefix = 0;
  uint64_t above = 0;
#pragma unroll 1
  while (width > 0) {
    const int bits = min(width, 8), shift = width - bits;
    sh.bins[threadIdx.x] = 0;
    __syncthreads();
#pragma unroll 1
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
      const uint32_t key = key_at(i), part = key - least;
      if (key < cut.key || (width < 32 && (part >> width) != prefix)) continue;
      atomicAdd(reinterpret_cast<unsigned long long*>(&sh.bins[(part >> shift) & 255]),
                static_cast<unsigned long long>(by_weight ? units.OfKey(key) : 1));
    }
    __syncthreads();
    const int digit = 255 - static_cast<int>(threadIdx.x);
    const uint64_t mine = sh.bins[digit];
    uint64_t unused;
    const uint64_t before = above + BlockExclScan(mine, sh.parts, &unused);
    if (before < goal && goal <= before + mine) {
      sh.found[0] = static_cast<uint64_t>(digit);
      sh.found[1] = before;
    }
    __syncthreads();
    prefix = prefix << bits | static_cast<uint32_t>(sh.found[0]);
    above = sh.found[1];
    width = shift;
    __syncthreads();
  }
  const uint32_t key = least + prefix;
  const uint64_t each = by_weight ? units.OfKey(key) : 1;
  return Cut{key, (goal - above + each - 1) / each};
}

// Grid: rows.
__global__ __launch_bounds__(kThreads) void SampleChooseKernel(const SampleArgs a) {
  __shared__ ChooseShared sh;
  const int tid = threadIdx.x;
  const Row row(a, blockIdx.x);
  const Plan plan = *row.ThePlan();
  if (plan.kind == Kind::kDone) return;
  const Setting set = SettingOf(a, row.r);
  const Units units{plan.top, set.by, a.units};
  const double unit = ldexp(1.0, -a.units);
  const uint32_t n = plan.candidates;
  const bool in_lds = n <= kInLds;
  const uint32_t* const keys = row.Keys();
  if (in_lds) {
#pragma unroll 4
    for (uint32_t i = tid; i < n; i += kThreads) sh.keys[i] = keys[i];
  }
  for (int s = tid; s < a.slices; s += kThreads) {
    sh.kept[s] = row.Above()[s];
    sh.kept_in[s] = 0;
    sh.ties[s] = 0;
    sh.first[s] = 0;
    if (n > 0) sh.offsets[s] = row.Offsets()[s];
  }
  __syncthreads();
  const auto key_at = [&](uint32_t i) { return in_lds ? sh.keys[i] : keys[i]; };

  // ---- the cut
  const double least = plan.cut_m ? static_cast<double>(set.m) / unit : 0.0;  // in units
  Cut cut;
  bool ties_count = false;
  if (n > 0) {
    if (plan.cut_k || plan.cut_p) {
      uint32_t low = 0xFFFFFFFFu, high = 0;
#pragma unroll 1
      for (uint32_t i = tid; i < n; i += kThreads) {
        const uint32_t key = key_at(i);
        low = min(low, key);
        high = max(high, key);
      }
      high = static_cast<uint32_t>(BlockMaxU64(high, sh.parts));
      low = ~static_cast<uint32_t>(BlockMaxU64(~low, sh.parts));
      const int width = 32 - __builtin_clz((high - low) | 1);
      // first top_k's among its candidates, then top_p's among what that keeps
#pragma unroll 1
      for (int filter = plan.cut_k || plan.cut_p == 2 ? 0 : 1; filter < (plan.cut_p ? 2 : 1); ++filter) {
        uint64_t goal;
        if (filter == 0) {
          goal = static_cast<uint64_t>(set.k) - plan.base_count;
        } else {
          uint64_t whole = 0;
#pragma unroll 1
          for (uint32_t i = tid; i < n; i += kThreads) {
            const uint32_t key = key_at(i);
            if (key > cut.key) whole += units.OfKey(key);
          }
          whole = BlockSum(whole, sh.parts);
          if (cut.ties > 0) whole += cut.ties * units.OfKey(cut.key);
          if (whole == 0) break;
          const double all = plan.cut_p == 2 ? plan.base + static_cast<double>(whole) * unit : plan.all;
          const double of = ceil((static_cast<double>(set.p) * all - plan.base) / unit);
          goal = of < 1.0 ? 1 : of < static_cast<double>(whole) ? static_cast<uint64_t>(of) : whole;
        }
        cut = Select(key_at, n, low, width, units, filter == 1, cut, goal, sh);
      }
    }
    ties_count = cut.ties > 0 && units.Of(ValueOf(cut.key)) >= least;

    // ---- what it keeps of each slice's candidates
    sh.offsets[a.slices] = static_cast<int32_t>(n);
    __syncthreads();
#pragma unroll 1
    for (uint32_t i = tid; i < n; i += kThreads) {
      const uint32_t key = key_at(i);
      if (key < cut.key) continue;
      int s = 0;  // the last slice that begins at or before i, of those that have any
      for (int step = kMaxSlices / 2; step > 0; step >>= 1) {
        if (s + step < a.slices && sh.offsets[s + step] <= static_cast<int32_t>(i)) s += step;
      }
      if (key == cut.key) {
        atomicAdd(&sh.ties[s], 1u);
      } else {
        const double w = units.Of(ValueOf(key));
        if (w >= least) {
          atomicAdd(reinterpret_cast<unsigned long long*>(&sh.kept_in[s]), static_cast<unsigned long long>(Units::Whole(w)));
        }
      }
    }
    __syncthreads();
    const uint64_t tie = ties_count ? units.OfKey(cut.key) : 0;
    uint64_t ties_before = 0;
#pragma unroll 1
    for (int s0 = 0; s0 < a.slices; s0 += kThreads) {
      const int s = s0 + tid;
      const uint64_t mine = s < a.slices && ties_count ? sh.ties[s] : 0;
      uint64_t all;
      const uint64_t before = ties_before + BlockExclScan(mine, sh.parts, &all);
      ties_before += all;
      if (s < a.slices) {
        const uint64_t left = before < cut.ties ? cut.ties - before : 0;
        const uint64_t kept = mine < left ? mine : left;
        sh.first[s] = static_cast<uint32_t>(kept);
        sh.kept[s] += static_cast<double>(sh.kept_in[s] + kept * tie) * unit;
      }
    }
    __syncthreads();
  }

  // ---- u's slice, by sums in index order: the first whose end passes it, or the last that has any weight
  double weight = 0.0;
  for (int s = tid; s < a.slices; s += kThreads) weight += sh.kept[s];
  if (tid == 0) sh.slice = 0x7FFFFFFF;
  weight = BlockSumD(weight, sh.dparts);
  const double goal = (set.u > 0.0f ? fmin(static_cast<double>(set.u), 1.0) : 0.0) * weight;
  double upto = 0.0;
#pragma unroll 1
  for (int s0 = 0; s0 < a.slices; s0 += kThreads) {
    const int s = s0 + tid;
    const double mine = s < a.slices ? sh.kept[s] : 0.0;
    double all;
    const double before = upto + BlockBeforeD(mine, sh.dparts, &all);
    if (mine > 0.0 && goal < before + mine) atomicMin(&sh.slice, s);
    __syncthreads();
    const bool found = sh.slice != 0x7FFFFFFF;
    if (sh.slice == s) sh.before = before;
    __syncthreads();
    if (found) break;
    upto += all;
  }
  if (sh.slice == 0x7FFFFFFF) {  // u of 1, or rounding: the last
    int last = 0;
    for (int s = tid; s < a.slices; s += kThreads) last = sh.kept[s] > 0.0 ? s : last;
    const uint64_t of_all = BlockMaxU64(static_cast<uint64_t>(last), sh.parts);
    if (tid == 0) {
      sh.slice = static_cast<int32_t>(of_all);
      sh.before = -1.0;  // the last of it
    }
    __syncthreads();
  }
  const int slice = __builtin_amdgcn_readfirstlane(sh.slice);
  const double inside = sh.before < 0.0 ? 0x1p63 : floor(fmax(goal - sh.before, 0.0) / unit);
  const uint64_t place = inside < 0x1p63 ? static_cast<uint64_t>(inside) : ~uint64_t(0);

  // ---- the walk: four rounds of four neighbours to a thread
  const uint64_t ties_kept = sh.first[slice];
  const bool some_ties = ties_kept > 0 && ties_kept < sh.ties[slice];  // and not all: their order counts
  uint64_t seen = 0, ties_seen = 0;
  uint64_t last = 0;  // the last kept one, before all those of a weight above 0
#pragma unroll 1
  for (int round = 0; round < kEach / 4; ++round) {
    const int at = slice * kSlice + round * 4 * kThreads + 4 * tid;
    const float4 v = row.Load(at);
    const float x[4] = {v.x, v.y, v.z, v.w};
    uint64_t tie_at = 0;
    if (some_ties) {
      uint64_t mine = 0, all;
#pragma unroll
      for (int c = 0; c < 4; ++c) mine += x[c] > -INFINITY && KeyOf(x[c]) == cut.key ? 1 : 0;
      tie_at = ties_seen + BlockExclScan(mine, sh.parts, &all);
      ties_seen += all;
    }
    uint64_t w[4], sum = 0;
    double of[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint32_t key = KeyOf(x[c]);
      const int j = set.BinBelow(plan.top_bin, x[c]);
      of[c] = units.Of(x[c]);
      bool keep = plan.kind == Kind::kAll || j < plan.hi;
      if (!keep && j <= plan.lo && of[c] >= least) {
        keep = key > cut.key;
        if (key == cut.key) {
          keep = some_ties ? tie_at < ties_kept : ties_kept > 0;
          ++tie_at;
        }
      }
      keep = keep && x[c] > -INFINITY;
      w[c] = keep ? Units::Whole(of[c]) : 0;
      sum += w[c];
      if (keep) last = max(last, (w[c] > 0 ? uint64_t(1) << 32 : 0) + static_cast<uint64_t>(at + c + 1));
    }
    uint64_t all;
    uint64_t before = seen + BlockExclScan(sum, sh.parts, &all);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if (before <= place && place < before + w[c]) {
        a.tokens[row.r] = at + c;
        if (a.probs != nullptr) a.probs[row.r] = static_cast<float>(of[c] * unit / weight);
      }
      before += w[c];
    }
    seen += all;
    if (seen > place) return;
  }
  // rounding, u of 1, or weights of less than half a unit each, of which one is as near as another
  last = BlockMaxU64(last, sh.parts);
  if (tid == 0) {
    const int32_t token = static_cast<int32_t>(last & 0xFFFFFFFFu) - 1;
    a.tokens[row.r] = token;
    if (a.probs != nullptr) {
      a.probs[row.r] = static_cast<float>(units.Of(Clean(a.logits[row.r * a.row_stride + token])) * unit / weight);
    }
  }
}

// ---------------------------------------------------------------- host side

int32_t UnitsFor(int64_t n) {
  int32_t bits = 0;
  while ((int64_t(1) << bits) < n) ++bits;
  return 62 - bits;
}

int32_t SlicesOf(int64_t n) { return static_cast<int32_t>((n + kSlice - 1) / kSlice); }

void CheckSizes(const char* what, int64_t n_rows, int64_t n) {
  RPG_CHECK(n > 0 && n <= kSamplerMaxVocab, "%s: %lld logits a row, the limit is %lld", what,
            static_cast<long long>(n), static_cast<long long>(kSamplerMaxVocab));
  RPG_CHECK(n_rows >= 0 && n_rows <= (1 << 20), "%s: %lld rows", what, static_cast<long long>(n_rows));
}

}  // namespace

size_t GpuSampleBatchWorkspaceBytes(int64_t n_rows, int64_t n) {
  CheckSizes("SampleBatchWorkspace", n_rows, n);
  return static_cast<size_t>(kCounters + std::min<int64_t>(n_rows, kRowsAtOnce) * RowPlace(SlicesOf(n)).bytes);
}

void GpuSampleBatchWorkspaceInit(void* workspace, size_t bytes) {
  RPG_CHECK(workspace != nullptr && bytes > 0 && bytes % 16 == 0 && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0,
            "SampleBatchWorkspaceInit: a workspace is 256-byte aligned and a multiple of 16 bytes");
  GpuStreamFill(workspace, static_cast<int64_t>(bytes), 0);
}

void GpuSampleBatch(const float* logits_dev, int64_t n_rows, int64_t n, int64_t row_stride,
                    const SampleBatchOptions& opt, const float* u_dev, int32_t* tokens_dev, float* probs_dev,
                    void* workspace, size_t workspace_bytes) {
  CheckSizes("SampleBatch", n_rows, n);
  RPG_CHECK(row_stride >= n && row_stride <= (int64_t(1) << 40), "SampleBatch: rows of %lld logits, %lld apart",
            static_cast<long long>(n), static_cast<long long>(row_stride));
  if (n_rows == 0) return;
  RPG_CHECK(logits_dev != nullptr && u_dev != nullptr && tokens_dev != nullptr && workspace != nullptr,
            "SampleBatch got a null pointer");
  const auto at = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
  RPG_CHECK(((at(logits_dev) | at(opt.temperature) | at(opt.top_k) | at(opt.top_p) | at(opt.min_p) | at(u_dev) |
              at(tokens_dev) | at(probs_dev)) & 3) == 0,
            "SampleBatch: a pointer is not 4-byte aligned");
  const size_t need = GpuSampleBatchWorkspaceBytes(n_rows, n);
  RPG_CHECK((at(workspace) & 255) == 0 && workspace_bytes >= need,
            "SampleBatch: a workspace of %zu bytes, 256-byte aligned, is needed (%zu given)", need, workspace_bytes);
  const int64_t bytes = 4 * n_rows, x_bytes = 4 * ((n_rows - 1) * row_stride + n);
  for (const void* in : {static_cast<const void*>(opt.temperature), static_cast<const void*>(opt.top_k),
                         static_cast<const void*>(opt.top_p), static_cast<const void*>(opt.min_p),
                         static_cast<const void*>(u_dev)}) {
    RPG_CHECK(in == nullptr || (!Overlap(tokens_dev, bytes, in, bytes) &&
                                (probs_dev == nullptr || !Overlap(probs_dev, bytes, in, bytes)) &&
                                !Overlap(workspace, static_cast<int64_t>(need), in, bytes)),
              "SampleBatch: outputs and the workspace must not overlap the settings or u");
  }
  RPG_CHECK(!Overlap(tokens_dev, bytes, logits_dev, x_bytes) &&
                !Overlap(workspace, static_cast<int64_t>(need), logits_dev, x_bytes) &&
                !Overlap(workspace, static_cast<int64_t>(need), tokens_dev, bytes) &&
                (probs_dev == nullptr ||
                 (!Overlap(probs_dev, bytes, logits_dev, x_bytes) && !Overlap(probs_dev, bytes, tokens_dev, bytes) &&
                  !Overlap(workspace, static_cast<int64_t>(need), probs_dev, bytes))),
            "SampleBatch: logits, outputs and the workspace must not overlap");
  const int32_t slices = SlicesOf(n);
  for (int64_t first = 0; first < n_rows; first += kRowsAtOnce) {
    const unsigned rows = static_cast<unsigned>(std::min<int64_t>(n_rows - first, kRowsAtOnce));
    const SampleArgs a{logits_dev,     row_stride, static_cast<int32_t>(n), slices,   UnitsFor(n), opt.temperature,
                       opt.top_k,      opt.top_p,  opt.min_p,               u_dev,    tokens_dev,  probs_dev,
                       static_cast<char*>(workspace), static_cast<int32_t>(first)};
    Launch("SampleSlicesKernel", SampleSlicesKernel, dim3(rows * slices), dim3(kThreads), a);
    Launch("SampleCollectKernel", SampleCollectKernel, dim3(rows * slices), dim3(kThreads), a);
    Launch("SampleChooseKernel", SampleChooseKernel, dim3(rows), dim3(kThreads), a);
  }
}

}  // namespace rpg
