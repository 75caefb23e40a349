// The next tokens of a batch of conversations, from given random numbers (the semantics
// are listed in sampler_gpu.h).
//
// Two launches, the first of which reads the logits once, in slices of 4096:
//   SampleSlices  each workgroup keeps a slice in registers: its largest value m_s, and of what its weights
//                 2^((x - m_s) log2(e) / T) come to, sums by value: bins an eighth of an octave wide (of 1/8 nat, for T
//                 above 1), whose borders are the same in all slices, counted and weighed upwards from the top. The row's
//                 last workgroup to arrive joins the slices, each by 2^((m_s - m) log2(e) / T), and finds between which
//                 bins each filter cuts: what lies above these bins is kept, what lies below is not;
//   SampleChoose  what lies in them (some hundred to a few thousand values) is collected in index order from the slices
//                 that have any, and the last workgroup to arrive cuts there exactly, by radix selection; it adds up
//                 the slices' kept weights, finds u's place among them, and walks that one slice.
// Weights are formed in double, which on this card costs what fp32 does, and summed as integers wherever atomics or a
// border depend on it, so that results are the same from run to run.
//
// What bounds it: reading the logits once; one row is the chain of round trips.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "attention_dev.h"
#include "dev_util.h"
#include "kernels_gpu.h"
#include "launch.h"
#include "paged_kv.h"
#include "sampler_gpu.h"

namespace rpg {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kSlice = 4096;
constexpr int kEach = kSlice / kThreads;
constexpr int kMaxSlices = static_cast<int>(kSamplerMaxVocab / kSlice);
constexpr int kBins = 256;       // of a slice; the last has all that is further down
constexpr int kInLds = 8192;     // candidates that are kept there
constexpr int kRowsAtOnce = 2048;  // rows of a launch: their counters have a place of their own in the workspace
constexpr int kCounterBytes = 128;
// A slice's sums: 13 bits of count, 51 of weight in units of 2^-38 of its largest
constexpr int kCountBits = 13;
constexpr int kSliceBits = 38;
static_assert(kSlice < (1 << kCountBits) && (int64_t(kSlice) << kSliceBits) < (int64_t(1) << (64 - kCountBits)), "");
constexpr int kDevice = 16;  // the cache policy of device-scope stores and loads

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

// ln(2)^n / n!
constexpr double SeriesOf2(int n) { return n == 0 ? 1.0 : SeriesOf2(n - 1) * 0.69314718055994530942 / n; }

// 2^(v + bits) for v <= 0: the Taylor series of 2^f, f = v - round(v), whose first term left out, (f ln 2)^10 / 10!, is
// below 2^-37. Below 2^-1000, and for a NaN, it is next to nothing.
__device__ __forceinline__ double Exp2Down(double v, int bits) {
  v = fmax(v, -1000.0);
  const double k = rint(v);
  const double f = v - k;
  double p = SeriesOf2(9);
#pragma unroll
  for (int i = 8; i >= 0; --i) p = fma(p, f, SeriesOf2(i));
  return ldexp(p, static_cast<int>(k) + bits);
}
// x as a whole number, 0 <= x < 2^51
__device__ __forceinline__ uint64_t Whole(double x) {
  return __builtin_bit_cast(uint64_t, x + 0x1p52) & 0xFFFFFFFFFFFFFull;
}

// A row's settings.
struct Setting {
  float t, p, m, u;
  int32_t k;
  bool greedy;
  double by;        // log2(e) / T
  float bin_by;     // bins to a logit

  __device__ __forceinline__ bool Filters() const { return k > 0 || OnP() || OnM(); }
  __device__ __forceinline__ bool OnP() const { return p > 0.0f && p < 1.0f; }
  __device__ __forceinline__ bool OnM() const { return m > 0.0f; }
  // The number of x's bin: falls with x, whatever the rounding; x is no NaN.
  __device__ __forceinline__ int32_t BinOf(float x) const {
    return static_cast<int32_t>(floorf(fminf(fmaxf(x * bin_by, -1e9f), 1e9f)));
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
  int32_t choosers;  // workgroups of SampleChoose for a row
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
  int32_t top_index;  // the first of that value
  uint64_t sum;
};

enum class Kind : int32_t { kDone, kWalk, kCut };
struct Plan {  // what the first launch finds out for the second
  Kind kind;
  float top;
  int32_t top_bin;
  int32_t hi, lo;  // the bins below the row's top one that are collected
  uint32_t cut_k, cut_p, cut_m;  // filters that may cut there
  uint32_t base_count;  // values above these bins
  uint32_t candidates;
  double base;  // their weight
  double all;   // the weight of all
};

__host__ __device__ constexpr int64_t RoundUp(int64_t x) { return (x + 127) / 128 * 128; }
struct RowPlace {
  int64_t sums, plan, above, offsets, bins, keys, bytes;
  __host__ __device__ explicit RowPlace(int32_t slices) {
    plan = 0;
    sums = RoundUp(sizeof(Plan));
    above = sums + RoundUp(slices * sizeof(SliceSums));
    offsets = above + RoundUp(slices * 8);
    bins = offsets + RoundUp((slices + 1) * 4);
    keys = bins + RoundUp(static_cast<int64_t>(slices) * kBins * 8);
    bytes = keys + static_cast<int64_t>(slices) * kSlice * 4;
  }
};
constexpr int64_t kCounters = static_cast<int64_t>(kRowsAtOnce) * kCounterBytes;

__device__ __forceinline__ char* RowAt(const SampleArgs& a, uint32_t row_of_launch, const RowPlace& place) {
  return a.workspace + kCounters + row_of_launch * place.bytes;
}

// ---------------------------------------------------------------- a workgroup's sums

__device__ __forceinline__ uint64_t ShflXor(uint64_t x, int by) { return __shfl_xor(x, by, 64); }
__device__ __forceinline__ double ShflXor(double x, int by) { return __shfl_xor(x, by, 64); }

template <class T>
__device__ __forceinline__ T BlockSum(T x, T* parts) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) x += ShflXor(x, off);
  if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = x;
  __syncthreads();
  T r = parts[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) r += parts[w];
  __syncthreads();
  return r;
}
// The larger of (value, and of equal ones the lower index), as one number.
__device__ __forceinline__ uint64_t Ranked(float x, uint32_t index) {
  return static_cast<uint64_t>(KeyOf(x)) << 32 | (0xFFFFFFFFu - index);
}
__device__ __forceinline__ uint64_t BlockMax(uint64_t x, uint64_t* parts) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const uint64_t o = ShflXor(x, off);
    x = o > x ? o : x;
  }
  if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = x;
  __syncthreads();
  uint64_t r = parts[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) r = parts[w] > r ? parts[w] : r;
  __syncthreads();
  return r;
}
// The sum over the threads before this one; *total that over all.
template <class T>
__device__ __forceinline__ T BlockBefore(T x, T* parts, T* total) {
  T upto = x;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const T o = __shfl_up(upto, off, 64);
    if ((threadIdx.x & 63) >= off) upto += o;
  }
  T before = __shfl_up(upto, 1, 64);
  if ((threadIdx.x & 63) == 0) before = T(0);
  if ((threadIdx.x & 63) == 63) parts[threadIdx.x >> 6] = upto;
  __syncthreads();
  T base = T(0), all = T(0);
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w == static_cast<int>(threadIdx.x >> 6)) base = all;
    all += parts[w];
  }
  __syncthreads();
  *total = all;
  return base + before;
}

__device__ __forceinline__ double CountOf(uint64_t sum) { return static_cast<double>(sum & ((1u << kCountBits) - 1)); }
__device__ __forceinline__ double WeightOf(uint64_t sum) {
  return static_cast<double>(sum >> kCountBits) * (1.0 / static_cast<double>(uint64_t(1) << kSliceBits));
}

__device__ __forceinline__ uint64_t LoadDevice8(__amdgpu_buffer_rsrc_t rs, uint32_t at) {
  const uint2 v = dev::LoadBufU2<kDevice>(rs, at);
  return static_cast<uint64_t>(v.y) << 32 | v.x;
}
__device__ __forceinline__ void StoreDevice8(__amdgpu_buffer_rsrc_t rs, uint32_t at, uint64_t v) {
  dev::StoreBufU2<kDevice>(rs, at, make_uint2(static_cast<uint32_t>(v), static_cast<uint32_t>(v >> 32)));
}

// Counts in at the row's counter: whether this is the last of `all` workgroups. What they stored for it is there.
__device__ __forceinline__ bool LastOf(const SampleArgs& a, uint32_t row_of_launch, int which, uint32_t all, int* flag) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    *flag = attn::Count(a.workspace, row_of_launch * (kCounterBytes / 4) + which, all);
  }
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(*flag) != 0;
}

// Four elements of a row from `i` on; what lies behind its end is minus infinity.
__device__ __forceinline__ float4 LoadLogits(__amdgpu_buffer_rsrc_t row, int32_t i, int32_t n) {
  const float4 x = dev::LoadBuf4<0>(row, 4u * static_cast<uint32_t>(i));
  return make_float4(i < n ? Clean(x.x) : -INFINITY, i + 1 < n ? Clean(x.y) : -INFINITY,
                     i + 2 < n ? Clean(x.z) : -INFINITY, i + 3 < n ? Clean(x.w) : -INFINITY);
}

// ---------------------------------------------------------------- the slices

struct JoinShared {
  double scale[kMaxSlices];  // of a slice's weights
  int32_t off[kMaxSlices];   // bins that a slice's top one lies below the row's
  double weight[kBins];      // of all bins up to one
  uint32_t count[kBins];
  uint32_t found[4];
};

// The row's last workgroup: where its filters cut.
__device__ void JoinSlices(const SampleArgs& a, const Setting& set, int64_t r, char* at, const RowPlace& place,
                           JoinShared& sh, uint64_t* parts, double* dparts) {
  const int tid = threadIdx.x;
  const __amdgpu_buffer_rsrc_t rs = dev::OutResource(at, static_cast<uint32_t>(place.keys));
  uint64_t best = 0;
  for (int s = tid; s < a.slices; s += kThreads) {
    const uint64_t head = LoadDevice8(rs, static_cast<uint32_t>(place.sums + s * sizeof(SliceSums)));
    const uint64_t mine = Ranked(__uint_as_float(static_cast<uint32_t>(head)), static_cast<uint32_t>(head >> 32));
    best = mine > best ? mine : best;
  }
  best = BlockMax(best, parts);
  const float top = ValueOf(static_cast<uint32_t>(best >> 32));
  Plan* const plan = reinterpret_cast<Plan*>(at + place.plan);
  if (top == -INFINITY || set.greedy) {
    if (tid == 0) {
      a.tokens[r] = top == -INFINITY ? -1 : static_cast<int32_t>(0xFFFFFFFFu - static_cast<uint32_t>(best));
      if (a.probs != nullptr) a.probs[r] = top == -INFINITY ? 0.0f : 1.0f;
      plan->kind = Kind::kDone;
    }
    return;
  }
  const int32_t top_bin = set.BinOf(top);
  double all = 0.0;
  uint64_t live = 0;
  for (int s = tid; s < a.slices; s += kThreads) {
    const uint32_t from = static_cast<uint32_t>(place.sums + s * sizeof(SliceSums));
    const float slice_top = __uint_as_float(static_cast<uint32_t>(LoadDevice8(rs, from)));
    const uint64_t sum = LoadDevice8(rs, from + 8);
    const double scale =
        slice_top == -INFINITY ? 0.0 : Exp2Down((static_cast<double>(slice_top) - static_cast<double>(top)) * set.by, 0);
    sh.scale[s] = scale;
    sh.off[s] = top_bin - set.BinOf(slice_top);
    all += scale * WeightOf(sum);
    live += static_cast<uint64_t>(CountOf(sum));
  }
  all = BlockSum(all, dparts);
  live = BlockSum(live, parts);
  if (tid < 4) sh.found[tid] = kBins - 1;
  __syncthreads();

  // a slice's sum over the row's bins up to j
  const auto sum_at = [&](int s, int j) -> uint64_t {
    const int in_slice = j == kBins - 1 ? j : j - sh.off[s];
    if (in_slice < 0) return 0;
    return LoadDevice8(rs, static_cast<uint32_t>(place.bins + (static_cast<int64_t>(s) * kBins + in_slice) * 8));
  };
  const bool on_k = set.k > 0 && static_cast<uint64_t>(set.k) < live, on_p = set.OnP(), on_m = set.OnM();
  if (!on_k && !on_p && !on_m) {
    for (int s = tid; s < a.slices; s += kThreads) {
      const uint64_t sum = LoadDevice8(rs, static_cast<uint32_t>(place.sums + s * sizeof(SliceSums)) + 8);
      reinterpret_cast<double*>(at + place.above)[s] = sh.scale[s] * WeightOf(sum);
    }
    if (tid == 0) *plan = Plan{Kind::kWalk, top, top_bin, kBins, kBins, 0, 0, 0, 0, 0, 0.0, all};
    return;
  }
  double weight = 0.0, count = 0.0;
#pragma unroll 8
  for (int s = 0; s < a.slices; ++s) {
    const uint64_t sum = sum_at(s, tid);
    weight += sh.scale[s] * WeightOf(sum);
    count += CountOf(sum);
  }
  static_assert(kThreads == kBins, "a bin to a thread");
  sh.weight[tid] = weight;
  sh.count[tid] = static_cast<uint32_t>(count);
  __syncthreads();
  const uint32_t before_count = tid == 0 ? 0 : sh.count[tid - 1];
  const double before_weight = tid == 0 ? 0.0 : sh.weight[tid - 1];
  const uint32_t my_count = sh.count[tid];
  // top_k's bin
  const uint32_t k = static_cast<uint32_t>(set.k);
  if (on_k && before_count < k && k <= my_count) sh.found[0] = tid;
  __syncthreads();
  const int bin_k = on_k ? static_cast<int>(sh.found[0]) : kBins - 1;
  // top_p's: between what all that top_k leaves may weigh, and a rounding more
  const double total = sh.weight[kBins - 1];
  const double least = on_k ? (bin_k == 0 ? 0.0 : sh.weight[bin_k - 1]) : total;
  const double most = on_k ? sh.weight[bin_k] : total;
  const double p = static_cast<double>(set.p);
  const double goal_hi = p * least * (1.0 - 0x1p-40), goal_lo = fmin(p * most * (1.0 + 0x1p-40), most);
  if (on_p && weight >= goal_hi && (tid == 0 || before_weight < goal_hi)) sh.found[1] = tid;
  if (on_p && weight >= goal_lo && (tid == 0 || before_weight < goal_lo)) sh.found[2] = tid;
  __syncthreads();
  const int p_hi = static_cast<int>(sh.found[1]), p_lo = static_cast<int>(sh.found[2]);
  // min_p's: from one number above its border to one below
  const double border = static_cast<double>(top) + log(static_cast<double>(set.m)) * static_cast<double>(set.t);
  const float near = static_cast<float>(fmax(border, -FLT_MAX));
  const auto bin_of = [&](float x) {
    return static_cast<int>(min(static_cast<int64_t>(top_bin) - set.BinOf(x), static_cast<int64_t>(kBins - 1)));
  };
  const int m_hi = on_m ? max(bin_of(nextafterf(near, INFINITY)), 0) : kBins - 1;
  const int m_lo = on_m ? max(bin_of(nextafterf(near, -INFINITY)), 0) : kBins - 1;

  // The cut that counts is the highest: filters that start below where another has cut for sure do not matter. top_p's
  // place needs what top_k leaves, and so the bins down to its.
  const int sure = min(on_k ? bin_k : kBins - 1, min(on_p ? p_lo : kBins - 1, on_m ? m_lo : kBins - 1));
  const bool cut_k = on_k && bin_k <= sure, cut_p = on_p && p_hi <= sure, cut_m = on_m && m_hi <= sure;
  int hi = kBins - 1, lo = 0;
  if (cut_k) hi = min(hi, bin_k), lo = max(lo, bin_k);
  if (cut_p) hi = min(hi, p_hi), lo = max(lo, on_k ? bin_k : p_lo);
  if (cut_m) hi = min(hi, m_hi), lo = max(lo, m_lo);

  // of each slice: the weight above these bins, and where its values in them go
  uint32_t placed = 0;
  int32_t* const offsets = reinterpret_cast<int32_t*>(at + place.offsets);
#pragma unroll 1
  for (int s0 = 0; s0 < a.slices; s0 += kThreads) {
    const int s = s0 + tid;
    uint64_t mine = 0;
    if (s < a.slices) {
      const uint64_t above = hi > 0 ? sum_at(s, hi - 1) : 0, upto = sum_at(s, lo);
      reinterpret_cast<double*>(at + place.above)[s] = sh.scale[s] * WeightOf(above);
      mine = static_cast<uint64_t>(CountOf(upto) - CountOf(above));
    }
    uint64_t sum;
    const uint64_t before = BlockBefore(mine, parts, &sum);
    if (s < a.slices) offsets[s] = static_cast<int32_t>(placed + before);
    placed += static_cast<uint32_t>(sum);
  }
  if (tid == 0) {
    offsets[a.slices] = static_cast<int32_t>(placed);
    *plan = Plan{Kind::kCut, top, top_bin, hi, lo, cut_k ? 1u : 0u, cut_p ? (on_k ? 2u : 1u) : 0u, cut_m ? 1u : 0u,
                 hi > 0 ? sh.count[hi - 1] : 0u, placed, hi > 0 ? sh.weight[hi - 1] : 0.0, total};
  }
}

__global__ __launch_bounds__(kThreads) void SampleSlicesKernel(const SampleArgs a) {
  __shared__ uint64_t bins[kWaves][kBins];
  __shared__ uint64_t parts[kWaves];
  __shared__ double dparts[kWaves];
  __shared__ int flag;
  __shared__ JoinShared join;
  const int tid = threadIdx.x;
  const uint32_t in_launch = blockIdx.x / static_cast<uint32_t>(a.slices);
  const int slice = static_cast<int>(blockIdx.x - in_launch * static_cast<uint32_t>(a.slices));
  const int64_t r = a.first_row + static_cast<int64_t>(in_launch);
  const RowPlace place(a.slices);
  char* const at = RowAt(a, in_launch, place);
  const __amdgpu_buffer_rsrc_t row =
      dev::OutResource(const_cast<float*>(a.logits) + r * a.row_stride, 4u * static_cast<uint32_t>(a.n));
  float x[kEach];
#pragma unroll
  for (int i = 0; i < kEach; i += 4) {
    const float4 v = LoadLogits(row, slice * kSlice + i * kThreads + 4 * tid, a.n);
    x[i] = v.x, x[i + 1] = v.y, x[i + 2] = v.z, x[i + 3] = v.w;
  }
  const Setting set = SettingOf(a, r);
  const bool filters = !set.greedy && set.Filters();
  if (filters) {
#pragma unroll
    for (int w = 0; w < kWaves; ++w) bins[w][tid] = 0;
  }
  uint64_t best = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const uint64_t mine = Ranked(x[i], static_cast<uint32_t>(slice * kSlice + (i & ~3) * kThreads + 4 * tid + (i & 3)));
    best = mine > best ? mine : best;
  }
  best = BlockMax(best, parts);
  const float top = ValueOf(static_cast<uint32_t>(best >> 32));
  uint64_t sum = 0;
  if (!set.greedy && top > -INFINITY) {
    const int32_t top_bin = set.BinOf(top);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (x[i] == -INFINITY) continue;
      const double w = Exp2Down((static_cast<double>(x[i]) - static_cast<double>(top)) * set.by, kSliceBits);
      const uint64_t add = Whole(w) << kCountBits | 1;
      if (filters) {
        const int j = min(top_bin - set.BinOf(x[i]), kBins - 1);
        atomicAdd(reinterpret_cast<unsigned long long*>(&bins[tid >> 6][j]), static_cast<unsigned long long>(add));
      } else {
        sum += add;
      }
    }
  }
  const __amdgpu_buffer_rsrc_t rs = dev::OutResource(at, static_cast<uint32_t>(place.keys));
  if (filters) {
    __syncthreads();
    uint64_t mine = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) mine += bins[w][tid];
    const uint64_t before = BlockBefore(mine, parts, &sum);
    StoreDevice8(rs, static_cast<uint32_t>(place.bins + (static_cast<int64_t>(slice) * kBins + tid) * 8), before + mine);
  } else if (!set.greedy) {
    sum = BlockSum(sum, parts);
  }
  if (tid == 0) {
    const uint32_t to = static_cast<uint32_t>(place.sums + slice * sizeof(SliceSums));
    dev::StoreBufU2<kDevice>(rs, to, make_uint2(__float_as_uint(top), 0xFFFFFFFFu - static_cast<uint32_t>(best)));
    StoreDevice8(rs, to + 8, sum);
  }
  if (!LastOf(a, in_launch, 0, static_cast<uint32_t>(a.slices), &flag)) return;
  JoinSlices(a, set, r, at, place, join, parts, dparts);
}

// ---------------------------------------------------------------- the choice

struct ChooseShared {
  uint32_t keys[kInLds];
  uint64_t bins[256];
  double kept[kMaxSlices];   // weight of a slice
  uint32_t ties[kMaxSlices];  // of a slice
  uint64_t found[2];
  int32_t slice;
  double before;
};

// Kept are the keys above `key`, and of those equal to it the first `ties` in index order.
struct Cut {
  uint32_t key = 0;
  uint64_t ties = 0;
};

// Whole units of a row's weights.
struct Units {
  float top;
  double by;
  int32_t bits;
  __device__ __forceinline__ double Of(float x) const {
    return Exp2Down((static_cast<double>(x) - static_cast<double>(top)) * by, bits);
  }
  __device__ __forceinline__ uint64_t OfKey(uint32_t key) const {
    return static_cast<uint64_t>(Of(ValueOf(key)) + 0.5);
  }
};

// The cut after the fewest first candidates, in order, whose amounts (1, or their weight) reach `goal`, among those that
// `cut` keeps: radix selection from the keys' upper digits down. The amounts of all ties of cut.key enter, which decides
// nothing: it is the last key.
template <bool kByWeight, class Keys>
__device__ Cut Select(const Keys& key_at, uint32_t n, const Units& units, const Cut& cut, uint64_t goal, ChooseShared& sh,
                      uint64_t* parts) {
  uint32_t prefix = 0;
  uint64_t above = 0;
#pragma unroll 1
  for (int shift = 24; shift >= 0; shift -= 8) {
    sh.bins[threadIdx.x] = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
      const uint32_t key = key_at(i);
      if (key < cut.key || (shift < 24 && (key >> (shift + 8)) != prefix)) continue;
      atomicAdd(reinterpret_cast<unsigned long long*>(&sh.bins[(key >> shift) & 255]),
                static_cast<unsigned long long>(kByWeight ? units.OfKey(key) : 1));
    }
    __syncthreads();
    const int digit = 255 - static_cast<int>(threadIdx.x);
    const uint64_t mine = sh.bins[digit];
    uint64_t unused;
    const uint64_t before = above + BlockBefore(mine, parts, &unused);
    if (before < goal && goal <= before + mine) {
      sh.found[0] = static_cast<uint64_t>(digit);
      sh.found[1] = before;
    }
    __syncthreads();
    prefix = prefix << 8 | static_cast<uint32_t>(sh.found[0]);
    above = sh.found[1];
    __syncthreads();
  }
  const uint64_t each = kByWeight ? units.OfKey(prefix) : 1;
  return Cut{prefix, (goal - above + each - 1) / each};
}

// Candidates' weight that a cut keeps.
template <class Keys>
__device__ uint64_t KeptWeight(const Keys& key_at, uint32_t n, const Units& units, const Cut& cut, uint64_t* parts) {
  uint64_t sum = 0;
  for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
    const uint32_t key = key_at(i);
    if (key > cut.key) sum += units.OfKey(key);
  }
  sum = BlockSum(sum, parts);
  return cut.ties > 0 ? sum + cut.ties * units.OfKey(cut.key) : sum;
}

template <class Keys>
__device__ void Choose(const SampleArgs& a, const Setting& set, const Plan& plan, int64_t r, const char* at,
                       const RowPlace& place, const Keys& key_at, ChooseShared& sh, uint64_t* parts, double* dparts) {
  const int tid = threadIdx.x;
  const Units units{plan.top, set.by, a.units};
  const double unit = ldexp(1.0, -a.units);
  const uint32_t n = plan.candidates;
  const int32_t* const offsets = reinterpret_cast<const int32_t*>(at + place.offsets);
  const double least = plan.cut_m ? static_cast<double>(set.m) / unit : 0.0;  // in units, as Units::Of's
  Cut cut;
  if (n > 0) {
    if (plan.cut_k || plan.cut_p == 2) {
      cut = Select<false>(key_at, n, units, cut, static_cast<uint64_t>(set.k) - plan.base_count, sh, parts);
    }
    if (plan.cut_p) {
      const uint64_t whole = KeptWeight(key_at, n, units, cut, parts);
      const double all = plan.cut_p == 2 ? plan.base + static_cast<double>(whole) * unit : plan.all;
      const double goal = ceil((static_cast<double>(set.p) * all - plan.base) / unit);
      const uint64_t in_units = goal < 1.0 ? 1 : static_cast<uint64_t>(goal);
      if (whole > 0) cut = Select<true>(key_at, n, units, cut, in_units < whole ? in_units : whole, sh, parts);
    }
  }
  const bool ties_count = cut.ties > 0 && units.Of(ValueOf(cut.key)) >= least;

  // the slices' kept weights: what is above, and of the candidates, a wave to a slice, what the cut keeps
  uint64_t ties_before = 0;
#pragma unroll 1
  for (int s0 = 0; s0 < a.slices; s0 += kThreads) {
    const int to = min(a.slices, s0 + kThreads);
#pragma unroll 1
    for (int s = s0 + (tid >> 6); s < to; s += kWaves) {
      uint64_t sum = 0, ties = 0;
      if (n > 0) {
        const int32_t from = offsets[s], end = offsets[s + 1];
        for (int32_t i = from + (tid & 63); i < end; i += 64) {
          const uint32_t key = key_at(static_cast<uint32_t>(i));
          if (key > cut.key) {
            const double w = units.Of(ValueOf(key));
            sum += w >= least ? static_cast<uint64_t>(w + 0.5) : 0;
          }
          ties += key == cut.key ? 1 : 0;
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
          sum += ShflXor(sum, off);
          ties += ShflXor(ties, off);
        }
      }
      if ((tid & 63) == 0) {
        sh.kept[s] = reinterpret_cast<const double*>(at + place.above)[s] + static_cast<double>(sum) * unit;
        sh.ties[s] = static_cast<uint32_t>(ties);
      }
    }
    __syncthreads();
    // of a slice's ties those that are still among the first
    const int s = s0 + tid;
    const uint64_t mine = s < to && ties_count ? sh.ties[s] : 0;
    uint64_t all;
    const uint64_t before = ties_before + BlockBefore(mine, parts, &all);
    ties_before += all;
    if (s < to) {
      const uint64_t left = before < cut.ties ? cut.ties - before : 0;
      const uint64_t kept = mine < left ? mine : left;
      sh.ties[s] = static_cast<uint32_t>(kept);
      if (kept > 0) sh.kept[s] += static_cast<double>(kept * units.OfKey(cut.key)) * unit;
    }
    __syncthreads();
  }
  double weight = 0.0;
  for (int s = tid; s < a.slices; s += kThreads) weight += sh.kept[s];
  weight = BlockSum(weight, dparts);
  const double u = set.u > 0.0f ? fmin(static_cast<double>(set.u), 1.0) : 0.0;
  const double goal = u * weight;

  // the slice, by sums in index order: the first whose end passes the goal, or the last that has any weight
  if (tid == 0) sh.slice = -1;
  __syncthreads();
  double upto = 0.0;
#pragma unroll 1
  for (int s0 = 0; s0 < a.slices; s0 += kThreads) {
    const int s = s0 + tid;
    const double mine = s < a.slices ? sh.kept[s] : 0.0;
    double all;
    const double before = upto + BlockBefore(mine, dparts, &all);
    if (mine > 0.0 && goal < before + mine) {
      atomicMin(reinterpret_cast<unsigned int*>(&sh.slice), static_cast<unsigned int>(s));
    }
    __syncthreads();
    const int32_t found = sh.slice;
    if (found == s) sh.before = before;
    __syncthreads();
    if (found >= 0) break;
    upto += all;
  }
  if (sh.slice < 0) {  // u of 1, or rounding: the last
    int32_t last = -1;
    for (int s = tid; s < a.slices; s += kThreads) last = sh.kept[s] > 0.0 ? s : last;
    const uint64_t top = BlockMax(static_cast<uint64_t>(last + 1), parts);
    if (tid == 0) {
      sh.slice = static_cast<int32_t>(top) - 1;
      sh.before = -1.0;  // the last of it
    }
    __syncthreads();
  }
  const int slice = __builtin_amdgcn_readfirstlane(sh.slice);
  const double inside = sh.before < 0.0 ? INFINITY : fmax(goal - sh.before, 0.0);

  // the walk, sixteen neighbours to a thread
  const __amdgpu_buffer_rsrc_t row =
      dev::OutResource(const_cast<float*>(a.logits) + r * a.row_stride, 4u * static_cast<uint32_t>(a.n));
  float x[kEach];
  uint64_t w[kEach];
  uint64_t sum = 0, ties = 0;
  uint32_t kept = 0;
#pragma unroll
  for (int i = 0; i < kEach; i += 4) {
    const float4 v = LoadLogits(row, slice * kSlice + kEach * tid + i, a.n);
    x[i] = v.x, x[i + 1] = v.y, x[i + 2] = v.z, x[i + 3] = v.w;
  }
  const auto bin_of = [&](float v) {
    return static_cast<int>(min(static_cast<int64_t>(plan.top_bin) - set.BinOf(v), static_cast<int64_t>(kBins - 1)));
  };
  const auto tied = [&](int i) {
    return cut.ties > 0 && x[i] > -INFINITY && KeyOf(x[i]) == cut.key && bin_of(x[i]) >= plan.hi;
  };
#pragma unroll
  for (int i = 0; i < kEach; ++i) ties += tied(i) ? 1 : 0;
  uint64_t unused;
  uint64_t ties_seen = BlockBefore(ties, parts, &unused);
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    w[i] = 0;
    const bool tie = tied(i);
    if (x[i] > -INFINITY) {
      const int j = bin_of(x[i]);
      const double of = units.Of(x[i]);
      bool keep = plan.kind == Kind::kWalk || j < plan.hi;
      if (!keep && j <= plan.lo) {
        keep = (tie ? ties_count && ties_seen < sh.ties[slice] : KeyOf(x[i]) > cut.key) && of >= least;
      }
      if (keep) {
        w[i] = static_cast<uint64_t>(of + 0.5);
        kept |= 1u << i;
      }
    }
    ties_seen += tie ? 1 : 0;
    sum += w[i];
  }
  uint64_t total;
  uint64_t before = BlockBefore(sum, parts, &total);
  if (total == 0) {  // weights of less than half a unit each: any of them is as near
#pragma unroll
    for (int i = 0; i < kEach; ++i) w[i] = kept >> i & 1;
    before = BlockBefore(static_cast<uint64_t>(__builtin_popcount(kept)), parts, &total);
  }
  const double in_units = floor(inside / unit);
  const uint64_t place_of = in_units < static_cast<double>(total) ? static_cast<uint64_t>(in_units) : total - 1;
  uint64_t seen = before;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    if (seen <= place_of && place_of < seen + w[i]) {
      a.tokens[r] = slice * kSlice + kEach * tid + i;
      if (a.probs != nullptr) a.probs[r] = static_cast<float>(units.Of(x[i]) * unit / weight);
    }
    seen += w[i];
  }
}

__global__ __launch_bounds__(kThreads) void SampleChooseKernel(const SampleArgs a) {
  __shared__ ChooseShared sh;
  __shared__ uint64_t parts[kWaves];
  __shared__ double dparts[kWaves];
  __shared__ int flag;
  const int tid = threadIdx.x;
  const uint32_t in_launch = blockIdx.x / static_cast<uint32_t>(a.choosers);
  const int me = static_cast<int>(blockIdx.x - in_launch * static_cast<uint32_t>(a.choosers));
  const int64_t r = a.first_row + static_cast<int64_t>(in_launch);
  const RowPlace place(a.slices);
  char* const at = RowAt(a, in_launch, place);
  const Plan plan = *reinterpret_cast<const Plan*>(at + place.plan);
  if (plan.kind == Kind::kDone) return;
  const Setting set = SettingOf(a, r);
  uint32_t* const list = reinterpret_cast<uint32_t*>(at + place.keys);
  const __amdgpu_buffer_rsrc_t keys = dev::OutResource(list, static_cast<uint32_t>(place.bytes - place.keys));
  if (plan.kind == Kind::kWalk || plan.candidates == 0) {
    if (me != 0) return;
    Choose(a, set, plan, r, at, place, [](uint32_t) { return 0u; }, sh, parts, dparts);
    return;
  }
  const int32_t* const offsets = reinterpret_cast<const int32_t*>(at + place.offsets);
  const __amdgpu_buffer_rsrc_t row =
      dev::OutResource(const_cast<float*>(a.logits) + r * a.row_stride, 4u * static_cast<uint32_t>(a.n));
#pragma unroll 1
  for (int s = me; s < a.slices; s += a.choosers) {
    const int32_t to = offsets[s];
    if (offsets[s + 1] == to) continue;
    // in index order: four rounds of four neighbours to a thread, whose counts are summed as one number
    float x[kEach];
    uint32_t in = 0;
    uint64_t counts = 0;
#pragma unroll
    for (int i = 0; i < kEach; i += 4) {
      const float4 v = LoadLogits(row, s * kSlice + i * kThreads + 4 * tid, a.n);
      x[i] = v.x, x[i + 1] = v.y, x[i + 2] = v.z, x[i + 3] = v.w;
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int64_t j = min(static_cast<int64_t>(plan.top_bin) - set.BinOf(x[i]), static_cast<int64_t>(kBins - 1));
      const bool takes = x[i] > -INFINITY && j >= plan.hi && j <= plan.lo;
      in |= takes ? 1u << i : 0u;
      counts += takes ? uint64_t(1) << (16 * (i / 4)) : 0;
    }
    uint64_t total;
    const uint64_t before = BlockBefore(counts, parts, &total);
    uint32_t round = 0;
#pragma unroll
    for (int i = 0; i < kEach; i += 4) {
      uint32_t next = static_cast<uint32_t>(to) + round + static_cast<uint32_t>(before >> (4 * i) & 0xFFFF);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (in >> (i + c) & 1) {
          __builtin_amdgcn_raw_buffer_store_b32(KeyOf(x[i + c]), keys, static_cast<int>(4 * next), 0, kDevice);
          ++next;
        }
      }
      round += static_cast<uint32_t>(total >> (4 * i) & 0xFFFF);
    }
  }
  if (!LastOf(a, in_launch, 1, static_cast<uint32_t>(a.choosers), &flag)) return;
  const auto load = [&](uint32_t i) { return __float_as_uint(dev::LoadBuf1<kDevice>(keys, 4 * i)); };
  if (plan.candidates <= kInLds) {
#pragma unroll 4
    for (uint32_t i = tid; i < plan.candidates; i += kThreads) sh.keys[i] = load(i);
    __syncthreads();
    Choose(a, set, plan, r, at, place, [&](uint32_t i) { return sh.keys[i]; }, sh, parts, dparts);
  } else {
    Choose(a, set, plan, r, at, place, load, sh, parts, dparts);
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
    const int64_t rows = std::min<int64_t>(n_rows - first, kRowsAtOnce);
    // enough workgroups to fill the card, each with some slices of a row
    const int32_t choosers = static_cast<int32_t>(std::min<int64_t>(slices, std::max<int64_t>(1, 1024 / rows)));
    const SampleArgs a{logits_dev,  row_stride, static_cast<int32_t>(n),      slices,
                       UnitsFor(n), opt.temperature, opt.top_k,               opt.top_p,
                       opt.min_p,   u_dev,      tokens_dev,                   probs_dev,
                       static_cast<char*>(workspace), static_cast<int32_t>(first), choosers};
    Launch("SampleSlicesKernel", SampleSlicesKernel, dim3(static_cast<unsigned>(rows * slices)), dim3(kThreads), a);
    Launch("SampleChooseKernel", SampleChooseKernel, dim3(static_cast<unsigned>(rows * choosers)), dim3(kThreads), a);
  }
}

}  // namespace rpg
