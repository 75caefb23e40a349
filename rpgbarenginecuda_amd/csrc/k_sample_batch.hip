// The next tokens of a batch of conversations, from given random numbers (the semantics
// are listed in sampler_gpu.h).
//
// Two launches, the first of which reads the logits once, in slices of 4096:
//   SampleSlices   a workgroup for each keeps it in registers: its largest value m_s, and of what its weights
//                  2^((x - m_s) log2(e) / T) come to, sums by value: bins an eighth of an octave wide (a twelfth of a nat,
//                  for T above 1), whose borders are the same in all slices, counted and weighed upwards from the top;
//                  and each value's bin, a byte;
//   SampleChoose   a workgroup for each row joins the slices, each by 2^((m_s - m) log2(e) / T), and finds between which
//                  bins each filter cuts: what lies above these bins is kept, what lies below is not. The values in them
//                  (some dozen to a few thousand) it collects by their bytes, and cuts there exactly, by radix selection;
//                  it adds up the slices' kept weights, finds u's place among them, and walks that one slice.
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
constexpr int kRowThreads = 1024;  // of a workgroup for a row
constexpr int kRowWaves = kRowThreads / 64;
static_assert(kMaxSlices <= kRowThreads, "a slice to a thread");
constexpr int kBins = 256;         // of a slice; the last has all that is further down
constexpr int kInLds = 8192;       // candidates that are kept there
// A slice's sums, in one number: count in the upper 13 bits, weight in units of 2^-38 of its largest in the lower 51.
constexpr int kWeightBits = 51;
constexpr int kSliceUnits = 38;
static_assert((int64_t(kSlice) << kSliceUnits) < (int64_t(1) << kWeightBits) && kSlice < (1 << (64 - kWeightBits)), "");

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
// 2^-38 of the value, and exactly 1 at 0. The coefficients, times 2^kBits, in scalar registers: written as constants, the
// compiler moves each to a vector register for every use.
template <int kBits>
struct Exp2Near {
  double c[9];
  __device__ __forceinline__ Exp2Near() {
    constexpr double kC[9] = {1.0,
                              0x1.62e42fef9cc69p-1,
                              0x1.ebfbdff82a734p-3,
                              0x1.c6b08da70cce3p-5,
                              0x1.3b2ab70ad256bp-7,
                              0x1.5d877598350dap-10,
                              0x1.4308c7183cd99p-13,
                              0x1.00c0e4e151fbep-16,
                              0x1.63b2d797a3663p-20};
#pragma unroll
    for (int i = 0; i < 9; ++i) {
      c[i] = kC[i] * static_cast<double>(uint64_t(1) << kBits);
      asm volatile("" : "+s"(c[i]));
    }
  }
  __device__ __forceinline__ double Of(double f) const {
    double p = fma(c[8], f, c[7]);
#pragma unroll
    for (int i = 6; i >= 0; --i) p = fma(p, f, c[i]);
    return p;
  }
};
// 2^(v + bits) for v <= 0; below 2^-1000, and for a NaN, next to nothing.
__device__ __forceinline__ double Exp2Down(const Exp2Near<0>& near, double v, int bits) {
  v = fmax(v, -1000.0);
  const double k = rint(v);
  return ldexp(near.Of(v - k), static_cast<int>(k) + bits);
}
// A slice's sum of one value of weight 2^v, v <= 0 (any that counts for nothing, down to minus infinity).
__device__ __forceinline__ uint64_t OneOf(const Exp2Near<kSliceUnits>& near, double v) {
  v = fmax(v, -200.0);
  // 1.5 * 2^52 added rounds v to a whole number, the low word; 2^52 added to a weight leaves its whole units
  const double shifted = v + 0x1.8p52;
  const uint64_t part = __builtin_bit_cast(uint64_t, near.Of(v - (shifted - 0x1.8p52)));
  const uint32_t exponent = static_cast<uint32_t>(__builtin_bit_cast(uint64_t, shifted)) << 20;
  const uint64_t scaled = (static_cast<uint64_t>(static_cast<uint32_t>(part >> 32) + exponent) << 32) |
                          static_cast<uint32_t>(part);
  const uint64_t bits = __builtin_bit_cast(uint64_t, __builtin_bit_cast(double, scaled) + 0x1p52);
  constexpr uint32_t kOne = 1u << (kWeightBits - 32);
  return (static_cast<uint64_t>(static_cast<uint32_t>(bits >> 32) - (0x43300000u - kOne)) << 32) |
         static_cast<uint32_t>(bits);
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

__host__ __device__ constexpr int64_t RoundUp(int64_t x) { return (x + 127) / 128 * 128; }
struct RowPlace {
  int64_t bins, bytes_of, keys, size;  // the slices' sums are in front
  __host__ __device__ explicit RowPlace(int32_t slices) {
    bins = RoundUp(slices * sizeof(SliceSums));
    bytes_of = bins + static_cast<int64_t>(slices) * kBins * 8;
    keys = bytes_of + static_cast<int64_t>(slices) * kSlice;
    size = keys + static_cast<int64_t>(slices) * kSlice * 4;
  }
};

struct Row {  // of the logits and the workspace
  int64_t r;
  RowPlace place;
  char* at;
  __amdgpu_buffer_rsrc_t logits;
  int32_t n;

  __device__ __forceinline__ Row(const SampleArgs& a, uint32_t row)
      : r(row),
        place(a.slices),
        at(a.workspace + row * place.size),
        logits(dev::OutResource(const_cast<float*>(a.logits) + r * a.row_stride, 4u * static_cast<uint32_t>(a.n))),
        n(a.n) {}
  __device__ __forceinline__ SliceSums* Sums() const { return reinterpret_cast<SliceSums*>(at); }
  // Of slice s, the sums of its bins down to each.
  __device__ __forceinline__ uint64_t* Bins(int s) const {
    return reinterpret_cast<uint64_t*>(at + place.bins) + static_cast<int64_t>(s) * kBins;
  }
  // Of slice s, each value's bin.
  __device__ __forceinline__ char* BytesOf(int s) const { return at + place.bytes_of + static_cast<int64_t>(s) * kSlice; }
  // Candidates that do not fit into LDS.
  __device__ __forceinline__ uint32_t* Keys() const { return reinterpret_cast<uint32_t*>(at + place.keys); }
  // Four logits from i on; what lies behind the row's end is minus infinity.
  __device__ __forceinline__ float4 Load(int32_t i) const {
    const float4 x = dev::LoadBuf4<0>(logits, 4u * static_cast<uint32_t>(i));
    return make_float4(i < n ? Clean(x.x) : -INFINITY, i + 1 < n ? Clean(x.y) : -INFINITY,
                       i + 2 < n ? Clean(x.z) : -INFINITY, i + 3 < n ? Clean(x.w) : -INFINITY);
  }
  __device__ __forceinline__ float LoadOne(int32_t i) const {
    return i < n ? Clean(dev::LoadBuf1<0>(logits, 4u * static_cast<uint32_t>(i))) : -INFINITY;
  }
};

// ---------------------------------------------------------------- the slices

// Grid: slices times rows.
__global__ __launch_bounds__(kThreads) void SampleSlicesKernel(const SampleArgs a) {
  __shared__ uint64_t bins[kWaves][kBins];
  __shared__ uint64_t parts[kWaves];
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
  for (int w = 0; w < kWaves; ++w) bins[w][tid] = 0;
  if (tid == 0) first = 0x7FFFFFFF;
  float top = x[0];
#pragma unroll
  for (int i = 1; i < kEach; ++i) top = fmaxf(top, x[i]);
  top = BlockMax(top, fparts);
  uint64_t sum = 0;
  const Exp2Near<kSliceUnits> near;
  const double dtop = static_cast<double>(top);
  if (set.greedy) {
#pragma unroll
    for (int i = kEach - 1; i >= 0; --i) {
      if (x[i] == top) atomicMin(&first, slice * kSlice + (i & ~3) * kThreads + 4 * tid + (i & 3));
    }
    __syncthreads();
  } else if (filters) {
    const int32_t top_bin = set.BinOf(top);
#pragma unroll
    for (int i = 0; i < kEach; i += 4) {
      uint32_t bytes = 0;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int j = x[i + c] > -INFINITY ? set.BinBelow(top_bin, x[i + c]) : kBins - 1;
        const uint64_t add = OneOf(near, (static_cast<double>(x[i + c]) - dtop) * set.by);
        if (x[i + c] > -INFINITY) {
          atomicAdd(reinterpret_cast<unsigned long long*>(&bins[tid >> 6][j]), static_cast<unsigned long long>(add));
        }
        bytes |= static_cast<uint32_t>(j) << (8 * c);
      }
      *reinterpret_cast<uint32_t*>(row.BytesOf(slice) + i * kThreads + 4 * tid) = bytes;
    }
    __syncthreads();
    uint64_t mine = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) mine += bins[w][tid];
    const uint64_t before = BlockExclScan(mine, parts, &sum);
    row.Bins(slice)[tid] = before + mine;
  } else {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const uint64_t add = OneOf(near, (static_cast<double>(x[i]) - dtop) * set.by);
      sum += x[i] > -INFINITY ? add : 0;
    }
    uint64_t total;
    BlockExclScan(sum, parts, &total);
    sum = total;
  }
  if (tid == 0) row.Sums()[slice] = SliceSums{top, first, sum};
}

// ---------------------------------------------------------------- a row's sums

// Over the workgroup of a row. `sh` has room for kRowWaves, and is not to be used again before a barrier: calls take turns
// with two of them.
template <int kCtrl, int kRowMask = 0xF>
__device__ __forceinline__ uint64_t MaxStep(uint64_t x) {
  const uint64_t o = DppU64<kCtrl, kRowMask>(x, 0);
  return o > x ? o : x;
}
__device__ __forceinline__ uint64_t RowMax(uint64_t x, uint64_t* sh) {
  x = MaxStep<0x111>(x);
  x = MaxStep<0x112>(x);
  x = MaxStep<0x114>(x);
  x = MaxStep<0x118>(x);
  x = MaxStep<0x142, 0xA>(x);
  x = MaxStep<0x143, 0xC>(x);
  if ((threadIdx.x & 63) == 63) sh[threadIdx.x >> 6] = x;
  __syncthreads();
  uint64_t r = sh[0];
#pragma unroll
  for (int w = 1; w < kRowWaves; ++w) r = sh[w] > r ? sh[w] : r;
  return r;
}
// The sum over the threads before this one; *total that over all.
__device__ __forceinline__ uint64_t RowBefore(uint64_t x, uint64_t* sh, uint64_t* total) {
  const uint64_t upto = WaveInclScanU64(x);
  if ((threadIdx.x & 63) == 63) sh[threadIdx.x >> 6] = upto;
  __syncthreads();
  uint64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kRowWaves; ++w) {
    before = w == static_cast<int>(threadIdx.x >> 6) ? all : before;
    all += sh[w];
  }
  *total = all;
  return before + upto - x;
}
// The same of doubles, in one order.
__device__ __forceinline__ double RowBeforeD(double x, double* sh, double* total) {
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
  for (int w = 0; w < kRowWaves; ++w) {
    base = w == static_cast<int>(threadIdx.x >> 6) ? all : base;
    all += sh[w];
  }
  *total = all;
  return (threadIdx.x & 63) == 0 ? base : base + mine;
}

// ---------------------------------------------------------------- the choice

constexpr int kJoiners = kRowThreads / kBins;  // threads to a bin, each for every kJoiners-th slice

struct ChooseShared {
  union {
    uint32_t keys[kInLds];
    struct {
      double weight[kJoiners][kBins];
      uint32_t count[kJoiners][kBins];
    } join;
  };
  double weight[kBins];  // of all bins down to one
  uint32_t count[kBins];
  uint64_t digits[kRowThreads];
  double scale[kMaxSlices];      // of a slice's weights
  int32_t off[kMaxSlices];       // bins that a slice's top one lies below the row's, at most all
  int32_t offsets[kMaxSlices + 1];  // of its candidates
  double kept[kMaxSlices];       // weight of a slice
  uint64_t kept_in[kMaxSlices];  // of its candidates, in whole units
  uint32_t ties[kMaxSlices];     // candidates of the cut's key
  uint32_t first[kMaxSlices];    // of these those that are kept
  uint64_t found[2];
  uint32_t bin[3];
  uint64_t parts[2][kRowWaves];
  double dparts[kRowWaves];
  int32_t slice;
  double before;
};

// Kept are the keys above `key`, and of those equal to it the first `ties` in index order.
struct Cut {
  uint32_t key = 0;
  uint64_t ties = 0;
};

// A row's weights, in units of 2^-s.
struct Units {
  Exp2Near<0> near;
  double top;
  double by;
  int32_t bits;
  __device__ __forceinline__ double Of(float x) const {
    return Exp2Down(near, (static_cast<double>(x) - top) * by, bits);
  }
  static __device__ __forceinline__ uint64_t Whole(double of) { return static_cast<uint64_t>(of + 0.5); }
  __device__ __forceinline__ uint64_t OfKey(uint32_t key) const { return Whole(Of(ValueOf(key))); }
};

// The cut after the fewest first candidates, in order, whose amounts (1, or their weight) reach `goal` (or all of them),
// among those that `cut` keeps: radix selection from the upper of the `width` bits down in which keys, less the least,
// differ. The amounts of all ties of cut.key enter, which decides nothing: it is the last key.
template <class Keys>
__device__ __forceinline__ Cut Select(const Keys& key_at, uint32_t n, uint32_t least, int width, const Units& units,
                                      bool by_weight, const Cut& cut, uint64_t goal, ChooseShared& sh) {
  constexpr int kDigit = 10;
  static_assert(1 << kDigit == kRowThreads, "a digit to a thread");
  uint32_t prefix = 0;
  uint64_t above = 0;
  sh.digits[threadIdx.x] = 0;
  __syncthreads();
#pragma unroll 1
  for (bool first = true; width > 0; first = false) {
    const int bits = min(width, kDigit), shift = width - bits;
#pragma unroll 1
    for (uint32_t i = threadIdx.x; i < n; i += kRowThreads) {
      const uint32_t key = key_at(i), part = key - least;
      if (key < cut.key || (!first && (part >> width) != prefix)) continue;
      atomicAdd(reinterpret_cast<unsigned long long*>(&sh.digits[(part >> shift) & (kRowThreads - 1)]),
                static_cast<unsigned long long>(by_weight ? units.OfKey(key) : 1));
    }
    __syncthreads();
    const int digit = kRowThreads - 1 - static_cast<int>(threadIdx.x);
    const uint64_t mine = sh.digits[digit];
    sh.digits[digit] = 0;
    uint64_t all;
    const uint64_t before = above + RowBefore(mine, sh.parts[first ? 0 : 1], &all);
    if (first) goal = goal < all ? goal : all;
    if (before < goal && goal <= before + mine) {
      sh.found[0] = static_cast<uint64_t>(digit);
      sh.found[1] = before;
    }
    __syncthreads();
    prefix = prefix << bits | static_cast<uint32_t>(sh.found[0]);
    above = sh.found[1];
    width = shift;
  }
  __syncthreads();
  const uint32_t key = least + prefix;
  const uint64_t each = by_weight ? units.OfKey(key) : 1;
  return Cut{key, each > 0 ? (goal - above + each - 1) / each : 0};
}

// Grid: rows.
__global__ __launch_bounds__(kRowThreads) void SampleChooseKernel(const SampleArgs a) {
  __shared__ ChooseShared sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Row row(a, blockIdx.x);
  const Setting set = SettingOf(a, row.r);

  // ---- the slices joined: a slice to a thread
  const SliceSums mine_of = tid < a.slices ? row.Sums()[tid] : SliceSums{-INFINITY, 0, 0};
  // the largest, and of those of it the one that is first
  const uint64_t best = RowMax(static_cast<uint64_t>(KeyOf(mine_of.top)) << 32 |
                                   (0xFFFFFFFFu - static_cast<uint32_t>(mine_of.top_index)), sh.parts[0]);
  const float top = ValueOf(static_cast<uint32_t>(best >> 32));
  if (top == -INFINITY || set.greedy) {
    if (tid == 0) {
      const bool none = top == -INFINITY;
      a.tokens[row.r] = none ? -1 : static_cast<int32_t>(0xFFFFFFFFu - static_cast<uint32_t>(best));
      if (a.probs != nullptr) a.probs[row.r] = none ? 0.0f : 1.0f;
    }
    return;
  }
  const int32_t top_bin = set.BinOf(top);
  const Units units{Exp2Near<0>(), static_cast<double>(top), set.by, a.units};
  const double unit = __builtin_bit_cast(double, static_cast<uint64_t>(1023 - a.units) << 52);
  double scale = 0.0;
  if (tid < a.slices) {
    const bool any = mine_of.top > -INFINITY;
    scale = any ? units.Of(mine_of.top) * unit : 0.0;
    sh.scale[tid] = scale;
    sh.off[tid] = any ? set.BinBelow(top_bin, mine_of.top) : kBins - 1;
    sh.kept_in[tid] = 0;
    sh.ties[tid] = 0;
    sh.first[tid] = 0;
  }
  if (tid < 3) sh.bin[tid] = kBins - 1;
  __syncthreads();
  // a slice's sum over the row's bins down to j
  const auto sum_at = [&](int s, int j) -> uint64_t {
    const int in_slice = j == kBins - 1 ? j : j - sh.off[s];
    return in_slice >= 0 ? row.Bins(s)[in_slice] : 0;
  };
  bool on_k = false;
  const bool on_p = set.OnP(), on_m = set.m > 0.0f, filters = set.Filters();

  // ---- between which bins the filters cut
  int hi = kBins, lo = -1;  // none: all that is live is above them
  bool cut_k = false, cut_p = false, cut_m = false;
  uint32_t base_count = 0, n = 0;
  double base = 0.0, all_weight = 0.0;
  if (filters) {
    const int j = tid % kBins, joiner = tid / kBins;
    double weight = 0.0;
    uint32_t count = 0;
    constexpr int kBatch = 10;
#pragma unroll 1
    for (int s0 = joiner; s0 < a.slices; s0 += kBatch * kJoiners) {
      uint64_t sums[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) sums[i] = s0 + i * kJoiners < a.slices ? sum_at(s0 + i * kJoiners, j) : 0;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (s0 + i * kJoiners < a.slices) weight += sh.scale[s0 + i * kJoiners] * WeightOf(sums[i]);
        count += CountOf(sums[i]);
      }
    }
    sh.join.weight[joiner][j] = weight;
    sh.join.count[joiner][j] = count;
    __syncthreads();
    if (tid < kBins) {
      weight = 0.0;
      count = 0;
#pragma unroll
      for (int i = 0; i < kJoiners; ++i) {
        weight += sh.join.weight[i][tid];
        count += sh.join.count[i][tid];
      }
      sh.weight[tid] = weight;
      sh.count[tid] = count;
    }
    __syncthreads();
    const bool first_bin = tid == 0, a_bin = tid < kBins;
    on_k = set.k > 0 && static_cast<uint32_t>(set.k) < sh.count[kBins - 1];  // else it keeps all that is live
    const uint32_t before_count = first_bin || !a_bin ? 0 : sh.count[tid - 1];
    const double before_weight = first_bin || !a_bin ? 0.0 : sh.weight[tid - 1];
    // top_k's bin
    const uint32_t k = static_cast<uint32_t>(set.k);
    if (a_bin && on_k && before_count < k && k <= count) sh.bin[0] = static_cast<uint32_t>(tid);
    __syncthreads();
    const int bin_k = on_k ? static_cast<int>(sh.bin[0]) : kBins - 1;
    // top_p's: between those of the least and the most that what top_k leaves may weigh, and a rounding more
    const double most = sh.weight[bin_k], least = !on_k ? most : bin_k == 0 ? 0.0 : sh.weight[bin_k - 1];
    const double p = static_cast<double>(set.p);
    const double goal_hi = p * least * (1.0 - 0x1p-40), goal_lo = fmin(p * most * (1.0 + 0x1p-40), most);
    if (a_bin && on_p) {
      if (weight >= goal_hi && (first_bin || before_weight < goal_hi)) sh.bin[1] = static_cast<uint32_t>(tid);
      if (weight >= goal_lo && (first_bin || before_weight < goal_lo)) sh.bin[2] = static_cast<uint32_t>(tid);
    }
    __syncthreads();
    const int p_hi = static_cast<int>(sh.bin[1]), p_lo = static_cast<int>(sh.bin[2]);
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
    cut_k = on_k && bin_k <= sure, cut_p = on_p && p_hi <= sure, cut_m = on_m && m_hi <= sure;
    if (on_k || on_p || on_m) hi = kBins - 1, lo = 0;
    if (cut_k) hi = min(hi, bin_k), lo = max(lo, bin_k);
    if (cut_p) hi = min(hi, p_hi), lo = max(lo, on_k ? bin_k : p_lo);
    if (cut_m) hi = min(hi, m_hi), lo = max(lo, m_lo);
    cut_k = cut_k || (cut_p && on_k);
    base_count = hi > 0 ? sh.count[min(hi, kBins) - 1] : 0;
    base = hi > 0 ? sh.weight[min(hi, kBins) - 1] : 0.0;
    all_weight = sh.weight[kBins - 1];
  }

  // ---- of each slice: the weight above these bins, and where its candidates go
  uint64_t in = 0;
  if (tid < a.slices) {
    uint64_t above = mine_of.sum;
    if (lo >= 0) {
      above = hi > 0 ? sum_at(tid, hi - 1) : 0;
      in = CountOf(sum_at(tid, lo)) - CountOf(above);
    }
    sh.kept[tid] = scale * WeightOf(above);
  }
  uint64_t placed;
  const uint64_t before_in = RowBefore(in, sh.parts[1], &placed);
  if (tid < a.slices) sh.offsets[tid] = static_cast<int32_t>(before_in);
  n = static_cast<uint32_t>(placed);
  if (tid == 0) sh.offsets[a.slices] = static_cast<int32_t>(n);
  __syncthreads();

  // ---- the candidates, in index order: first where they are, a wave to a slice, sixteen neighbours to a lane in each of
  // four rounds; then what they are, all at once
  const bool in_lds = n <= kInLds;
  uint32_t* const keys = in_lds ? sh.keys : row.Keys();
#pragma unroll 1
  for (int s = n > 0 ? wave : a.slices; s < a.slices; s += kRowWaves) {
    uint32_t to = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(sh.offsets[s]));
    if (to == static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(sh.offsets[s + 1]))) continue;
    const int off = __builtin_amdgcn_readfirstlane(sh.off[s]);
    // in the slice's own bins, whose last is the row's last
    const int from = max(0, hi - off), upto = lo == kBins - 1 ? lo : lo - off;
    uint4 b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = *reinterpret_cast<const uint4*>(row.BytesOf(s) + 1024 * i + 16 * lane);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t words[4] = {b[i].x, b[i].y, b[i].z, b[i].w};
      uint32_t takes = 0;
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        const uint32_t byte = words[c / 4] >> (8 * (c % 4)) & 255;
        takes |= (byte - static_cast<uint32_t>(from) <= static_cast<uint32_t>(upto - from) ? 1u : 0u) << c;
      }
      const int32_t at = s * kSlice + 1024 * i + 16 * lane;
      if (lo == kBins - 1) {  // minus infinity has the last bin's byte too
        for (uint32_t left = takes; left != 0; left &= left - 1) {
          const int c = __builtin_ctz(left);
          if (row.LoadOne(at + c) == -INFINITY) takes &= ~(1u << c);
        }
      }
      const uint32_t count = static_cast<uint32_t>(__builtin_popcount(takes));
      const uint32_t sum = attn::ScanAdd(count);
      uint32_t next = to + sum - count;
      to += __builtin_amdgcn_readlane(sum, 63);
      for (; takes != 0; takes &= takes - 1) keys[next++] = static_cast<uint32_t>(at + __builtin_ctz(takes));
    }
  }
  __syncthreads();
  uint32_t low = 0xFFFFFFFFu, high = 0;
#pragma unroll 1
  for (uint32_t i0 = tid; i0 < n; i0 += 4 * kRowThreads) {
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t at = i0 + i * kRowThreads;
      x[i] = row.LoadOne(static_cast<int32_t>(at < n ? keys[at] : 0));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t at = i0 + i * kRowThreads;
      if (at < n) {
        keys[at] = KeyOf(x[i]);
        low = min(low, KeyOf(x[i]));
        high = max(high, KeyOf(x[i]));
      }
    }
  }
  const auto key_at = [&](uint32_t i) { return keys[i]; };

  // ---- the cut
  const double least = cut_m ? static_cast<double>(set.m) / unit : 0.0;  // in units
  Cut cut;
  uint64_t tie = 0;  // weight of a tie, if it counts
  if (n > 0) {
    if (cut_k || cut_p) {
      high = static_cast<uint32_t>(RowMax(high, sh.parts[0]));
      low = ~static_cast<uint32_t>(RowMax(~low, sh.parts[1]));
      const int width = 32 - __builtin_clz((high - low) | 1);
      // first top_k's among its candidates, then top_p's among what that keeps
      if (cut_k) cut = Select(key_at, n, low, width, units, false, cut, static_cast<uint64_t>(set.k) - base_count, sh);
      if (cut_p) {
        double of_all = all_weight;
        if (on_k) {
          uint64_t whole = 0, total;
#pragma unroll 1
          for (uint32_t i = tid; i < n; i += kRowThreads) {
            const uint32_t key = key_at(i);
            if (key > cut.key) whole += units.OfKey(key);
          }
          RowBefore(whole, sh.parts[0], &total);
          of_all = base + static_cast<double>(total + cut.ties * units.OfKey(cut.key)) * unit;
        }
        const double of = ceil((static_cast<double>(set.p) * of_all - base) / unit);
        cut = Select(key_at, n, low, width, units, true, cut, of < 1.0 ? 1 : static_cast<uint64_t>(fmin(of, 0x1p62)), sh);
      }
    }
    if (cut.ties > 0) {
      const double of = units.Of(ValueOf(cut.key));
      tie = of >= least ? Units::Whole(of) : 0;
      if (of < least) cut.ties = 0;
    }

    // ---- what it keeps of each slice's candidates
#pragma unroll 1
    for (uint32_t i = tid; i < n; i += kRowThreads) {
      const uint32_t key = key_at(i);
      if (key < cut.key) continue;
      int s = 0;  // the last slice that begins at or before i
      for (int step = 1 << (31 - __builtin_clz(a.slices)); step > 0; step >>= 1) {
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
    const uint64_t ties = tid < a.slices ? sh.ties[tid] : 0;
    uint64_t unused;
    const uint64_t before = RowBefore(ties, sh.parts[0], &unused);
    if (tid < a.slices) {
      const uint64_t left = before < cut.ties ? cut.ties - before : 0;
      const uint64_t first = ties < left ? ties : left;
      sh.first[tid] = static_cast<uint32_t>(first);
      sh.kept[tid] += static_cast<double>(sh.kept_in[tid] + first * tie) * unit;
    }
  }

  // ---- u's slice, by sums in index order: the first whose end passes it, or the last that has any weight
  if (tid == 0) sh.slice = 0x7FFFFFFF;
  const double mine = tid < a.slices ? sh.kept[tid] : 0.0;
  double weight;
  const double before = RowBeforeD(mine, sh.dparts, &weight);
  const double goal = (set.u > 0.0f ? fmin(static_cast<double>(set.u), 1.0) : 0.0) * weight;
  if (mine > 0.0 && goal < before + mine) atomicMin(&sh.slice, tid);
  __syncthreads();
  if (sh.slice == tid) sh.before = before;
  if (sh.slice == 0x7FFFFFFF) {  // u of 1, or rounding: the last
    const uint64_t last = RowMax(mine > 0.0 ? static_cast<uint64_t>(tid) : 0, sh.parts[1]);
    if (tid == 0) {
      sh.slice = static_cast<int32_t>(last);
      sh.before = -1.0;  // the last of it
    }
  }
  __syncthreads();
  const int slice = __builtin_amdgcn_readfirstlane(sh.slice);
  const double inside = sh.before < 0.0 ? 0x1p63 : floor(fmax(goal - sh.before, 0.0) / unit);
  const uint64_t place = inside < 0x1p63 ? static_cast<uint64_t>(inside) : ~uint64_t(0);

  // ---- the walk: four neighbours to a thread
  static_assert(kSlice == 4 * kRowThreads, "");
  const uint64_t ties_kept = sh.first[slice];
  const bool some_ties = ties_kept > 0 && ties_kept < sh.ties[slice];  // and not all: their order counts
  const int at = slice * kSlice + 4 * tid;
  const float4 v = row.Load(at);
  const float x[4] = {v.x, v.y, v.z, v.w};
  uint64_t tie_at = 0;
  if (some_ties) {
    uint64_t ties = 0, unused;
#pragma unroll
    for (int c = 0; c < 4; ++c) ties += x[c] > -INFINITY && KeyOf(x[c]) == cut.key ? 1 : 0;
    tie_at = RowBefore(ties, sh.parts[1], &unused);
    __syncthreads();
  }
  uint64_t w[4], sum = 0;
  double of[4];
  uint64_t last = 0;  // the last kept one, before all those of a weight above 0
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const uint32_t key = KeyOf(x[c]);
    const int j = set.BinBelow(top_bin, x[c]);
    of[c] = units.Of(x[c]);
    bool keep = j < hi;
    if (!keep && j <= lo && of[c] >= least) {
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
  uint64_t total;
  uint64_t seen = RowBefore(sum, sh.parts[0], &total);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    if (seen <= place && place < seen + w[c]) {
      a.tokens[row.r] = at + c;
      if (a.probs != nullptr) a.probs[row.r] = static_cast<float>(of[c] * unit / weight);
    }
    seen += w[c];
  }
  if (total > place) return;
  // rounding, u of 1, or weights of less than half a unit each, of which one is as near as another
  last = RowMax(last, sh.parts[1]);
  if (tid == 0) {
    const int32_t token = static_cast<int32_t>(last & 0xFFFFFFFFu) - 1;
    a.tokens[row.r] = token;
    if (a.probs != nullptr) a.probs[row.r] = static_cast<float>(units.Of(row.LoadOne(token)) * unit / weight);
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
  return static_cast<size_t>(std::max<int64_t>(n_rows, 1) * RowPlace(SlicesOf(n)).size);
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
  RPG_CHECK(n_rows * slices <= 0x7FFFFFFF, "SampleBatch: %lld rows of %lld logits are too many for one call",
            static_cast<long long>(n_rows), static_cast<long long>(n));
  const SampleArgs a{logits_dev, row_stride, static_cast<int32_t>(n), slices, UnitsFor(n), opt.temperature, opt.top_k,
                     opt.top_p,  opt.min_p,  u_dev,                   tokens_dev, probs_dev, static_cast<char*>(workspace)};
  Launch("SampleSlicesKernel", SampleSlicesKernel, dim3(static_cast<unsigned>(n_rows * slices)), dim3(kThreads), a);
  Launch("SampleChooseKernel", SampleChooseKernel, dim3(static_cast<unsigned>(n_rows)), dim3(kRowThreads), a);
}

}  // namespace rpg
