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
// What bounds it: of the slices of many rows reading and weighing (128 rows of 151936: 28 us, 78 MB read and 30 written; the
// read alone would take 12), of the choice the chain of barriers and round trips of one workgroup (one row 12 to 14 us, of
// which the bins take 2.5, the candidates 2.7, the cut 1 to 3, the walk 2; its instructions already in the cache, one less), and
// for rows of some thousand candidates their logits, each a line of its own (128 rows of 2300: 24 us).
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
constexpr int kBins = 256;         // of a slice; the last has all that is further down
constexpr int kInLds = 8192;       // candidates that are kept there
// A slice's sums, in one number: count in the upper 13 bits, weight in units of 2^-38 of its largest in the lower 51.
constexpr int kWeightBits = 51;
constexpr int kSliceUnits = 38;
static_assert((int64_t(kSlice) << kSliceUnits) < (int64_t(1) << kWeightBits) && kSlice < (1 << (64 - kWeightBits)), "");

// ---------------------------------------------------------------- order and weights

// What a logit counts as: NaN as minus infinity, plus infinity as the largest number.
__device__ __forceinline__ float Clean(float x) { return fminf(fmaxf(x, -INFINITY), FLT_MAX); }

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
      if (i == 7) {  // c[8] f + c[7] has room for one scalar
        asm volatile("" : "+v"(c[i]));
      } else {
        asm volatile("" : "+s"(c[i]));
      }
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
  dev::U32x2 part = __builtin_bit_cast(dev::U32x2, near.Of(v - (shifted - 0x1.8p52)));
  part[1] += __builtin_bit_cast(dev::U32x2, shifted)[0] << 20;
  dev::U32x2 bits = __builtin_bit_cast(dev::U32x2, __builtin_bit_cast(double, part) + 0x1p52);
  constexpr uint32_t kOne = 1u << (kWeightBits - 32);
  bits[1] -= 0x43300000u - kOne;
  return __builtin_bit_cast(uint64_t, bits);
}
__device__ __forceinline__ uint32_t CountOf(uint64_t sum) { return static_cast<uint32_t>(sum >> kWeightBits); }
// In units of 2^-38: 2^52 and it are one double, bit for bit.
__device__ __forceinline__ double WeightOf(uint64_t sum) {
  const uint64_t whole = sum & ((uint64_t(1) << kWeightBits) - 1);
  return __builtin_bit_cast(double, whole | uint64_t(0x433) << 52) - 0x1p52;
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
  __device__ __forceinline__ float4 Load(int32_t i) const { return Checked(dev::LoadBuf4<0>(logits, 4u * static_cast<uint32_t>(i)), i); }
  __device__ __forceinline__ float4 Checked(float4 x, int32_t i) const {
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
    const float4 v = dev::LoadBuf4<0>(row.logits, 4u * static_cast<uint32_t>(slice * kSlice + i * kThreads + 4 * tid));
    x[i] = v.x, x[i + 1] = v.y, x[i + 2] = v.z, x[i + 3] = v.w;
  }
  const Setting set = SettingOf(a, row.r);
  const bool filters = !set.greedy && set.Filters();
  if (__builtin_expect(slice + 1 < a.slices, 1)) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) x[i] = Clean(x[i]);
  } else {  // the row may end in it
#pragma unroll
    for (int i = 0; i < kEach; i += 4) {
      const float4 v = row.Checked(make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]), slice * kSlice + i * kThreads + 4 * tid);
      x[i] = v.x, x[i + 1] = v.y, x[i + 2] = v.z, x[i + 3] = v.w;
    }
  }
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
        const bool live = x[i + c] > -INFINITY;
        const int j = live ? set.BinBelow(top_bin, x[i + c]) : kBins - 1;
        const uint64_t add = OneOf(near, (static_cast<double>(x[i + c]) - dtop) * set.by);
        if (live) {
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

// ---------------------------------------------------------------- the choice

// Sums over a wave: upto and with this lane.
__device__ __forceinline__ double WaveInclScanD(double v) {
  v += DppDbl<0x111>(v, 0.0);
  v += DppDbl<0x112>(v, 0.0);
  v += DppDbl<0x114>(v, 0.0);
  v += DppDbl<0x118>(v, 0.0);
  v += DppDbl<0x142, 0xA>(v, 0.0);
  return v + DppDbl<0x143, 0xC>(v, 0.0);
}
template <class T>
__device__ __forceinline__ T LastLane(T x) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(bits), 63);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(bits >> 32), 63);
  return __builtin_bit_cast(T, static_cast<uint64_t>(hi) << 32 | lo);
}

// The four waves of a SIMD take turns, so that what one wave can do (sums over slices and digits) is done by one, the
// others waiting at the barrier: sums over all sixteen took 4 us more for one row and 2 for 128.
constexpr int kRowThreads = 1024;
constexpr int kRowWaves = kRowThreads / 64;
constexpr int kJoiners = kRowThreads / kBins;  // threads to a bin, each for every kJoiners-th slice
// A bin's keys differ in some 19 bits. (128 rows of 2300 candidates: 23.8 us with digits of 7 or 8 bits, 24.6 with 9, 25.5
// with 10, which one wave sums up.)
constexpr int kDigitBits = 8;
constexpr int kDigits = 1 << kDigitBits;
constexpr int kLaneDigits = kDigits / 64;
static_assert(kDigits <= kRowThreads && kDigits % 64 == 0, "");
// Where digit d's amount is: from the highest down kLaneDigits to a lane, a lane's beside the next lane's.
__device__ __forceinline__ uint32_t DigitAt(uint32_t d) {
  const uint32_t down = kDigits - 1 - d;
  return down % kLaneDigits * 64 + down / kLaneDigits;
}

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
  uint64_t digits[kDigits];
  uint64_t sum[kMaxSlices];         // a slice's
  double scale[kMaxSlices];         // of its weights' units
  int32_t off[kMaxSlices];          // bins that its top one lies below the row's, at most all
  int32_t offsets[kMaxSlices + 1];  // of its candidates
  int32_t with[kMaxSlices];         // the slices that have some, `n_with` of them
  double kept[kMaxSlices];          // its weight
  uint64_t kept_in[kMaxSlices];     // that of its candidates, in whole units
  uint32_t ties[kMaxSlices];        // its candidates of the cut's key
  uint32_t first[kMaxSlices];       // of these those that are kept
  uint64_t found[2];
  uint64_t wave_sum[kRowWaves];
  uint32_t wave_last[kRowWaves];
  double weight_of_all;
  double before;
  float top;
  int32_t top_index;
  uint32_t low, high;
  uint32_t bin[3];
  int32_t n_with;
  uint32_t cut_key;
  uint64_t cut_ties;
  int32_t slice;
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

// The candidates' keys: in LDS where they fit.
struct Keys {
  uint32_t* lds;
  uint32_t* rest;
  bool in_lds;
  __device__ __forceinline__ uint32_t operator[](uint32_t i) const { return in_lds ? lds[i] : rest[i]; }
  __device__ __forceinline__ void Put(uint32_t i, uint32_t key) const {
    if (in_lds) {
      lds[i] = key;
    } else {
      rest[i] = key;
    }
  }
};

// The cut after the fewest first candidates, in order, whose amounts (1, or their weight) reach `goal` (or all of them),
// among those that `cut` keeps: radix selection from the upper of the `width` bits down in which keys, less the least,
// differ. The amounts of all ties of cut.key enter, which decides nothing: it is the last key. sh.digits are 0, and are so
// again.
__device__ __forceinline__ Cut Select(const Keys& keys, uint32_t n, uint32_t least, int width, const Units& units,
                                      bool by_weight, const Cut& cut, uint64_t goal, ChooseShared& sh) {
  uint32_t prefix = 0;
  if (threadIdx.x == 0) sh.found[0] = sh.found[1] = 0;  // candidates of no weight at all: the last
#pragma unroll 1
  for (bool first = true; width > 0; first = false) {
    const int bits = min(width, kDigitBits), shift = width - bits;
#pragma unroll 1
    for (uint32_t i = threadIdx.x; i < n; i += kRowThreads) {
      const uint32_t key = keys[i], part = key - least;
      if (key < cut.key || (!first && (part >> width) != prefix)) continue;
      atomicAdd(reinterpret_cast<unsigned long long*>(&sh.digits[DigitAt((part >> shift) & (kDigits - 1))]),
                static_cast<unsigned long long>(by_weight ? units.OfKey(key) : 1));
    }
    __syncthreads();
    if (threadIdx.x < 64) {  // some digits to a lane, from the highest down
      uint64_t d[kLaneDigits], mine = 0;
#pragma unroll
      for (int i = 0; i < kLaneDigits; ++i) {
        d[i] = sh.digits[64 * i + threadIdx.x];
        sh.digits[64 * i + threadIdx.x] = 0;
        mine += d[i];
      }
      const uint64_t upto = WaveInclScanU64(mine);
      if (first) goal = min(goal, LastLane(upto));
      uint64_t before = upto - mine;
#pragma unroll
      for (int i = 0; i < kLaneDigits; ++i) {
        if (before < goal && goal <= before + d[i]) {
          sh.found[0] = static_cast<uint64_t>(kDigits - 1 - (kLaneDigits * threadIdx.x + i));
          sh.found[1] = goal - before;
        }
        before += d[i];
      }
    }
    __syncthreads();
    prefix = prefix << bits | static_cast<uint32_t>(sh.found[0]);
    goal = sh.found[1];  // of what has this prefix
    width = shift;
  }
  __syncthreads();
  const uint32_t key = least + prefix;
  const uint64_t each = by_weight ? units.OfKey(key) : 1;
  return Cut{key, each > 0 ? (goal + each - 1) / each : 0};
}

// The same of up to 64 candidates, one to a lane of a wave: each lane sums what is above its own. A filter takes some 1 us
// so, and 2.6 by the digits above, whose rounds of atomics and barriers cost the same for few as for many (48 rows of 31999,
// top-k and top-p over some 35 candidates: the kernel 13.7 us against 18).
struct Few {
  uint32_t n, key;
  uint64_t weight;

  __device__ __forceinline__ Few(const Keys& keys, uint32_t count, const Units& units) : n(count) {
    const uint32_t lane = threadIdx.x & 63;
    key = lane < n ? keys[lane] : 0;  // of no candidate's: minus infinity's is above it
    weight = lane < n ? units.OfKey(key) : 0;
  }
  static __device__ __forceinline__ uint64_t FromLane(uint64_t x, uint32_t lane) {
    return static_cast<uint64_t>(__builtin_amdgcn_readlane(static_cast<uint32_t>(x >> 32), lane)) << 32 |
           static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<uint32_t>(x), lane));
  }
  __device__ __forceinline__ uint64_t WeightKept(const Cut& cut) const {
    const uint64_t ties = __ballot(key == cut.key);
    return LastLane(WaveInclScanU64(key > cut.key ? weight : 0)) +
           (ties != 0 ? cut.ties * FromLane(weight, __builtin_ctzll(ties)) : 0);
  }
  // (Four candidates a turn, whose steps overlap; those behind the last, of key and weight 0, change nothing.)
  __device__ __forceinline__ Cut SelectCount(uint64_t goal) const {
    uint32_t above = 0, alike = 0;
#pragma unroll 1
    for (uint32_t j = 0; j < n; j += 4) {
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) {
        const uint32_t other = __builtin_amdgcn_readlane(key, j + i);
        above += other > key ? 1 : 0;
        alike += other == key ? 1 : 0;
      }
    }
    const uint32_t want = static_cast<uint32_t>(min(goal, static_cast<uint64_t>(n)));
    const uint32_t lane = __builtin_ctzll(__ballot(key != 0 && above < want && want <= above + alike));
    return Cut{static_cast<uint32_t>(__builtin_amdgcn_readlane(key, lane)),
               want - static_cast<uint32_t>(__builtin_amdgcn_readlane(above, lane))};
  }
  __device__ __forceinline__ Cut SelectWeight(const Cut& cut, uint64_t goal, uint32_t least) const {
    const uint64_t each = key == 0 || key < cut.key ? 0 : weight;
    uint64_t above[2] = {0, 0};
    uint32_t alike = 0;
#pragma unroll 1
    for (uint32_t j = 0; j < n; j += 4) {
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) {
        const uint32_t other = __builtin_amdgcn_readlane(key, j + i);
        const uint64_t amount = FromLane(each, j + i);
        above[i & 1] += other > key ? amount : 0;
        alike += other == key ? 1 : 0;
      }
    }
    above[0] += above[1];
    goal = min(goal, LastLane(WaveInclScanU64(each)));
    const uint64_t here = __ballot(above[0] < goal && goal <= above[0] + alike * each);
    if (here == 0) return Cut{least, 0};  // candidates of no weight at all: the last
    const uint32_t lane = __builtin_ctzll(here);
    const uint64_t one = FromLane(each, lane);
    return Cut{static_cast<uint32_t>(__builtin_amdgcn_readlane(key, lane)), (goal - FromLane(above[0], lane) + one - 1) / one};
  }
};

// Of four bytes those in [from, from + span], as a 1 in each. (Bytes are subtracted and added without carries
// between them; a byte less `from` exceeds the span where adding 255 - span carries out.)
__device__ __forceinline__ uint32_t BytesWithin(uint32_t bytes, uint32_t from4, uint32_t beyond4) {
  constexpr uint32_t kHigh = 0x80808080u;
  const uint32_t less = ((bytes | kHigh) - (from4 & ~kHigh)) ^ ((bytes ^ ~from4) & kHigh);
  const uint32_t low = (less & ~kHigh) + (beyond4 & ~kHigh);
  return (~((less & beyond4) | ((less | beyond4) & low)) & kHigh) >> 7;
}

// The same of those that are the byte repeated in of4: of a byte and it the exclusive or is 0, and then no sum of its lower
// bits and 127 reaches the highest. (A third of the work; most cuts lie in one bin.)
__device__ __forceinline__ uint32_t BytesEqual(uint32_t bytes, uint32_t of4) {
  constexpr uint32_t kHigh = 0x80808080u;
  const uint32_t x = bytes ^ of4;
  return (~(((x & ~kHigh) + ~kHigh) | x) & kHigh) >> 7;
}
// Sixteen bits in order, of bytes that are in: sums of 1, 2, 4, ... for each.
template <class F>
__device__ __forceinline__ uint32_t BitsOf(const uint4& bytes, F in) {
  const uint32_t low =
      __builtin_amdgcn_udot4(in(bytes.x), 0x08040201u, __builtin_amdgcn_udot4(in(bytes.y), 0x80402010u, 0, false), false);
  const uint32_t high =
      __builtin_amdgcn_udot4(in(bytes.z), 0x08040201u, __builtin_amdgcn_udot4(in(bytes.w), 0x80402010u, 0, false), false);
  return high << 8 | low;
}

// Grid: rows.
__global__ __launch_bounds__(kRowThreads) void SampleChooseKernel(const SampleArgs a) {
  __shared__ ChooseShared sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Row row(a, blockIdx.x);
  SliceSums firsts{-INFINITY, 0, 0};  // of the first 64 slices, for the first wave
  if (tid < min(a.slices, 64)) firsts = row.Sums()[tid];
  const Setting set = SettingOf(a, row.r);
  const bool on_p = set.OnP(), on_m = set.m > 0.0f, filters = set.Filters();
  const auto slices64 = [&](auto f) {  // by the first wave
#pragma unroll 1
    for (int s0 = 0; s0 < a.slices; s0 += 64) f(s0 + lane, s0 + lane < a.slices);
  };

  // ---- the slices' largest, and what their weights are multiplied by
  if (wave == 0) {
    float top = firsts.top;
#pragma unroll 1
    for (int s = 64 + lane; s < a.slices; s += 64) top = fmaxf(top, row.Sums()[s].top);
    top = WaveMaxTo63(top);
    top = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(top), 63));
    int32_t index = 0x7FFFFFFF;
    const int32_t top_bin = set.BinOf(top);
    const Exp2Near<0> near;
    slices64([&](int s, bool there) {
      if (!there) return;
      const SliceSums mine = s < 64 ? firsts : row.Sums()[s];
      if (set.greedy) {
        if (mine.top == top) index = min(index, mine.top_index);
        return;
      }
      const bool any = mine.top > -INFINITY;
      sh.sum[s] = mine.sum;
      sh.scale[s] = any ? Exp2Down(near, (static_cast<double>(mine.top) - static_cast<double>(top)) * set.by, -kSliceUnits) : 0.0;
      sh.off[s] = any ? set.BinBelow(top_bin, mine.top) : kBins - 1;
      sh.kept_in[s] = 0;
      sh.ties[s] = 0;
      sh.first[s] = 0;
    });
    if (set.greedy) {
#pragma unroll
      for (int by = 32; by > 0; by >>= 1) index = min(index, __shfl_xor(index, by, 64));
    }
    if (lane == 0) {
      sh.top = top;
      sh.top_index = index;
      sh.low = 0xFFFFFFFFu;
      sh.high = 0;
      sh.slice = 0x7FFFFFFF;
    }
  } else if (tid < 64 + 3) {
    sh.bin[tid - 64] = kBins - 1;
  }
  if (tid < kDigits) sh.digits[tid] = 0;
  __syncthreads();
  const float top = sh.top;
  if (top == -INFINITY || set.greedy) {
    if (tid == 0) {
      a.tokens[row.r] = top == -INFINITY ? -1 : sh.top_index;
      if (a.probs != nullptr) a.probs[row.r] = top == -INFINITY ? 0.0f : 1.0f;
    }
    return;
  }
  const int32_t top_bin = set.BinOf(top);
  const Units units{Exp2Near<0>(), static_cast<double>(top), set.by, a.units};
  const double unit = __builtin_bit_cast(double, static_cast<uint64_t>(1023 - a.units) << 52);
  // a slice's sum over the row's bins down to j
  const auto sum_at = [&](int s, int j) -> uint64_t {
    const int in_slice = j == kBins - 1 ? j : j - sh.off[s];
    return in_slice >= 0 ? row.Bins(s)[in_slice] : 0;
  };

  // ---- between which bins the filters cut
  bool on_k = false;
  int hi = kBins, lo = -1;  // none: all that is live is above them
  bool cut_k = false, cut_p = false, cut_m = false;
  uint32_t base_count = 0;
  double base = 0.0, all_weight = 0.0;
  if (filters) {
    {
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
          if (s0 + i * kJoiners < a.slices) weight = fma(sh.scale[s0 + i * kJoiners], WeightOf(sums[i]), weight);
          count += CountOf(sums[i]);
        }
      }
      sh.join.weight[joiner][j] = weight;
      sh.join.count[joiner][j] = count;
    }
    __syncthreads();
    double weight = 0.0;
    uint32_t count = 0;
    if (tid < kBins) {
#pragma unroll
      for (int i = 0; i < kJoiners; ++i) {
        weight += sh.join.weight[i][tid];
        count += sh.join.count[i][tid];
      }
      sh.weight[tid] = weight;
      sh.count[tid] = count;
    }
    __syncthreads();
    on_k = set.k > 0 && static_cast<uint32_t>(set.k) < sh.count[kBins - 1];  // else it keeps all that is live
    const bool first_bin = tid == 0;
    // top_k's bin
    const uint32_t k = static_cast<uint32_t>(set.k);
    if (on_k) {
      if (tid < kBins && (first_bin ? 0 : sh.count[tid - 1]) < k && k <= count) sh.bin[0] = static_cast<uint32_t>(tid);
      __syncthreads();
    }
    const int bin_k = on_k ? static_cast<int>(sh.bin[0]) : kBins - 1;
    // top_p's: between those of the least and the most that what top_k leaves may weigh, and a rounding more
    if (on_p) {
      if (tid < kBins) {
        const double before = first_bin ? 0.0 : sh.weight[tid - 1];
        const double most = sh.weight[bin_k], least = !on_k ? most : bin_k == 0 ? 0.0 : sh.weight[bin_k - 1];
        const double p = static_cast<double>(set.p);
        const double goal_hi = p * least * (1.0 - 0x1p-40), goal_lo = fmin(p * most * (1.0 + 0x1p-40), most);
        if (weight >= goal_hi && (first_bin || before < goal_hi)) sh.bin[1] = static_cast<uint32_t>(tid);
        if (weight >= goal_lo && (first_bin || before < goal_lo)) sh.bin[2] = static_cast<uint32_t>(tid);
      }
      __syncthreads();
    }
    const int p_hi = static_cast<int>(sh.bin[1]), p_lo = static_cast<int>(sh.bin[2]);
    // min_p's: that of the nearest number to its border, and the next in either direction, where the border's rounding and its
    // number's may have it. The hardware's logarithm is within 2^-23 of its value from 2^-40 to 1, and a border further than
    // all bins, 32 octaves or (T above 1) 22 logits below the largest, is in the last: any other is off by at most 2^-18
    // octaves or logits, of which a bin is an eighth and a twelfth, at any temperature
    int m_hi = kBins - 1, m_lo = kBins - 1;
    if (on_m) {
      const double octaves = static_cast<double>(__builtin_amdgcn_logf(set.m));
      const double border = static_cast<double>(top) + octaves / set.by;
      const uint32_t near = KeyOf(static_cast<float>(fmax(border, -static_cast<double>(FLT_MAX))));
      m_hi = max(set.BinBelow(top_bin, fminf(ValueOf(near + 1), top)) - 1, 0);
      m_lo = min(set.BinBelow(top_bin, ValueOf(near - 1)) + 1, kBins - 1);
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
  if (wave == 0) {
    uint64_t placed = 0;
    int32_t n_with = 0;
    slices64([&](int s, bool there) {
      uint64_t in = 0;
      if (there) {
        uint64_t above = sh.sum[s];
        if (lo >= 0) {
          above = hi > 0 ? sum_at(s, hi - 1) : 0;
          in = CountOf(sum_at(s, lo)) - CountOf(above);
        }
        sh.kept[s] = sh.scale[s] * WeightOf(above);
      }
      const uint64_t upto = WaveInclScanU64(in);
      if (there) sh.offsets[s] = static_cast<int32_t>(placed + upto - in);
      placed += LastLane(upto);
      const uint64_t some = __ballot(in > 0);
      if (in > 0) sh.with[n_with + __builtin_popcountll(some & ((uint64_t(1) << lane) - 1))] = s;
      n_with += __builtin_popcountll(some);
    });
    if (lane == 0) {
      sh.offsets[a.slices] = static_cast<int32_t>(placed);
      sh.n_with = n_with;
    }
  }
  __syncthreads();
  const uint32_t n = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(sh.offsets[a.slices]));

  const double least = cut_m ? static_cast<double>(set.m) / unit : 0.0;  // in units
  Cut cut;
  uint64_t tie = 0;  // weight of a tie, if it counts
  if (n > 0) {
    // ---- the candidates, in index order: first where they are, a wave to a slice, 64 neighbours to a lane; then what they
    // are, all at once
    const Keys keys{sh.keys, row.Keys(), n <= kInLds};
    const int n_with = __builtin_amdgcn_readfirstlane(sh.n_with);
    const auto slice_of = [&](int i) { return __builtin_amdgcn_readfirstlane(sh.with[min(i, n_with - 1)]); };
    uint4 bytes[4];
    const auto load = [&](int s) {
      const uint4* const from = reinterpret_cast<const uint4*>(row.BytesOf(s)) + 4 * lane;
#pragma unroll
      for (int i = 0; i < 4; ++i) bytes[i] = from[i];
    };
    int s = slice_of(wave);
    if (wave < n_with) load(s);
#pragma unroll 1
    for (int i = wave; i < n_with; i += kRowWaves) {
      const int off = __builtin_amdgcn_readfirstlane(sh.off[s]);
      // in the slice's own bins, whose last is the row's last
      const int from = max(0, hi - off), upto = lo == kBins - 1 ? lo : lo - off;
      const uint32_t from4 = static_cast<uint32_t>(from) * 0x01010101u;
      const uint32_t beyond4 = static_cast<uint32_t>(255 - (upto - from)) * 0x01010101u;
      uint32_t part[4];
      if (upto == from) {
#pragma unroll
        for (int i = 0; i < 4; ++i) part[i] = BitsOf(bytes[i], [&](uint32_t x) { return BytesEqual(x, from4); });
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) part[i] = BitsOf(bytes[i], [&](uint32_t x) { return BytesWithin(x, from4, beyond4); });
      }
      uint64_t takes = static_cast<uint64_t>(part[3] << 16 | part[2]) << 32 | (part[1] << 16 | part[0]);
      const int32_t at = s * kSlice + 64 * lane;
      uint32_t next = static_cast<uint32_t>(sh.offsets[s]);
      if (i + kRowWaves < n_with) {
        s = slice_of(i + kRowWaves);
        load(s);
      }
      if (lo == kBins - 1) {  // minus infinity has the last bin's byte too
        for (uint64_t left = takes; left != 0; left &= left - 1) {
          const int c = __builtin_ctzll(left);
          if (row.LoadOne(at + c) == -INFINITY) takes &= ~(uint64_t(1) << c);
        }
      }
      const uint32_t count = static_cast<uint32_t>(__builtin_popcountll(takes));
      next += attn::ScanAdd(count) - count;
      for (; takes != 0; takes &= takes - 1) keys.Put(next++, static_cast<uint32_t>(at + __builtin_ctzll(takes)));
    }
    __syncthreads();
    {
      uint32_t low = 0xFFFFFFFFu, high = 0;
#pragma unroll 1
      for (uint32_t i0 = tid; i0 < n; i0 += 4 * kRowThreads) {
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t at = i0 + i * kRowThreads;
          x[i] = at < n ? row.LoadOne(static_cast<int32_t>(keys[at])) : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t at = i0 + i * kRowThreads;
          if (at < n) {
            keys.Put(at, KeyOf(x[i]));
            low = min(low, KeyOf(x[i]));
            high = max(high, KeyOf(x[i]));
          }
        }
      }
      // (a wave's first: a thousand atomics on one place took 5 us)
#pragma unroll
      for (int by = 32; by > 0; by >>= 1) {
        low = min(low, static_cast<uint32_t>(__shfl_xor(static_cast<int>(low), by, 64)));
        high = max(high, static_cast<uint32_t>(__shfl_xor(static_cast<int>(high), by, 64)));
      }
      if (lane == 0 && high != 0) {
        atomicMin(&sh.low, low);
        atomicMax(&sh.high, high);
      }
    }
    __syncthreads();

    // ---- the cut: first top_k's, then top_p's among what that keeps
    const auto goal_p = [&](double of_all) {
      const double of = ceil((static_cast<double>(set.p) * of_all - base) / unit);
      return of < 1.0 ? 1 : static_cast<uint64_t>(fmin(of, 0x1p62));
    };
    const uint64_t goal_k = static_cast<uint64_t>(set.k) - base_count;
    if (n <= 64) {
      if (wave == 0) {
        const Few few(keys, n, units);
        if (cut_k) cut = few.SelectCount(goal_k);
        if (cut_p) {
          const double of_all = on_k ? base + static_cast<double>(few.WeightKept(cut)) * unit : all_weight;
          cut = few.SelectWeight(cut, goal_p(of_all), sh.low);
        }
        if (lane == 0) {
          sh.cut_key = cut.key;
          sh.cut_ties = cut.ties;
        }
      }
      __syncthreads();
      cut = Cut{sh.cut_key, sh.cut_ties};
    } else {
      const int width = 32 - __builtin_clz((sh.high - sh.low) | 1);
#pragma unroll 1
      for (int filter = cut_k ? 0 : 1; filter < (cut_p ? 2 : 1); ++filter) {
        uint64_t goal = goal_k;
        if (filter == 1) {
          double of_all = all_weight;
          if (on_k) {
            if (tid == 0) sh.found[0] = 0;
            __syncthreads();
            uint64_t whole = 0;
#pragma unroll 1
            for (uint32_t i = tid; i < n; i += kRowThreads) {
              const uint32_t key = keys[i];
              if (key > cut.key) whole += units.OfKey(key);
            }
            if (whole != 0) {
              atomicAdd(reinterpret_cast<unsigned long long*>(&sh.found[0]), static_cast<unsigned long long>(whole));
            }
            __syncthreads();
            of_all = base + static_cast<double>(sh.found[0] + cut.ties * units.OfKey(cut.key)) * unit;
            __syncthreads();
          }
          goal = goal_p(of_all);
        }
        cut = Select(keys, n, sh.low, width, units, filter == 1, cut, goal, sh);
      }
    }
    if (cut.ties > 0) {
      const double of = units.Of(ValueOf(cut.key));
      tie = of >= least ? Units::Whole(of) : 0;
      if (of < least) cut.ties = 0;
    }

    // ---- what it keeps of each slice's candidates, a wave to a slice
#pragma unroll 1
    for (int i = wave; i < n_with; i += kRowWaves) {
      const int of = slice_of(i);
      const uint32_t end = static_cast<uint32_t>(sh.offsets[of + 1]);
      uint64_t kept = 0;
      uint32_t ties = 0;
#pragma unroll 1
      for (uint32_t c = static_cast<uint32_t>(sh.offsets[of]) + lane; c < end; c += 64) {
        const uint32_t key = keys[c];
        if (key == cut.key) ++ties;
        if (key > cut.key) {
          const double w = units.Of(ValueOf(key));
          if (w >= least) kept += Units::Whole(w);
        }
      }
      kept = WaveInclScanU64(kept);
      ties = attn::ScanAdd(ties);
      if (lane == 63) {
        sh.kept_in[of] = kept;
        sh.ties[of] = ties;
      }
    }
    __syncthreads();
  }

  // ---- u's slice, by sums in index order: the first whose end passes it, or the last that has any weight
  if (wave == 0) {
    uint64_t ties_before = 0;
    double all = 0.0;
    slices64([&](int s, bool there) {
      uint64_t ties = 0;
      if (n > 0) {
        ties = there ? sh.ties[s] : 0;
        const uint64_t upto = WaveInclScanU64(ties), before = ties_before + upto - ties;
        ties_before += LastLane(upto);
        ties = min(ties, before < cut.ties ? cut.ties - before : 0);
      }
      double kept = 0.0;
      if (there) {
        kept = sh.kept[s] + static_cast<double>(sh.kept_in[s] + ties * tie) * unit;
        sh.first[s] = static_cast<uint32_t>(ties);
      }
      const double upto = all + WaveInclScanD(kept);
      if (there) sh.kept[s] = kept > 0.0 ? upto : -1.0;  // where it ends
      all = LastLane(upto);
    });
    const double goal = (set.u > 0.0f ? fmin(static_cast<double>(set.u), 1.0) : 0.0) * all;
    int32_t found = 0x7FFFFFFF, last = 0;
    double end_before = 0.0, before = 0.0;  // the end of the last slice of any weight, and that before the one found
    slices64([&](int s, bool there) {
      const double end = there ? sh.kept[s] : -1.0;
      const uint64_t some = __ballot(end >= 0.0), past = __ballot(end > goal);
      if (found == 0x7FFFFFFF && past != 0) {
        const int at = __builtin_ctzll(past);
        const uint64_t earlier = some & ((uint64_t(1) << at) - 1);
        found = s - lane + at;
        before = earlier != 0 ? sh.kept[s - lane + 63 - __builtin_clzll(earlier)] : end_before;
      }
      if (some != 0) {
        last = s - lane + 63 - __builtin_clzll(some);
        end_before = sh.kept[last];
      }
    });
    if (lane == 0) {
      sh.slice = found != 0x7FFFFFFF ? found : last;
      sh.before = found != 0x7FFFFFFF ? floor((goal - before) / unit) : 0x1p63;  // u's place in it, in units
      sh.weight_of_all = all;
    }
  }
  __syncthreads();
  const int slice = __builtin_amdgcn_readfirstlane(sh.slice);
  const double inside = sh.before;
  const uint64_t place = inside < 0x1p63 ? static_cast<uint64_t>(inside) : ~uint64_t(0);

  // ---- the walk: four neighbours to a thread
  static_assert(kSlice == 4 * kRowThreads, "");
  const int at = slice * kSlice + 4 * tid;
  const float4 v = row.Load(at);
  const float x[4] = {v.x, v.y, v.z, v.w};
  const uint64_t ties_kept = sh.first[slice];
  const bool some_ties = ties_kept > 0 && ties_kept < sh.ties[slice];  // and not all: their order counts
  uint64_t tie_at = 0;
  if (some_ties) {
    uint64_t ties = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) ties += x[c] > -INFINITY && KeyOf(x[c]) == cut.key ? 1 : 0;
    const uint64_t upto = WaveInclScanU64(ties);
    if (lane == 63) sh.wave_sum[wave] = upto;
    __syncthreads();
    tie_at = upto - ties;
    for (int w = 0; w < wave; ++w) tie_at += sh.wave_sum[w];
    __syncthreads();
  }
  uint64_t w[4] = {0, 0, 0, 0}, sum = 0;
  double of[4];
  bool kept[4] = {false, false, false, false};
  int bin[4];
  bool some = false;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    bin[c] = x[c] > -INFINITY ? set.BinBelow(top_bin, x[c]) : 1 << 30;
    some = some || bin[c] < hi || bin[c] <= lo;
  }
  if (__any(some)) {  // in most waves nothing is kept
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint32_t key = KeyOf(x[c]);
      of[c] = units.Of(x[c]);
      bool keep = bin[c] < hi;
      if (!keep && bin[c] <= lo && of[c] >= least) {
        keep = key > cut.key;
        if (key == cut.key) {
          keep = some_ties ? tie_at < ties_kept : ties_kept > 0;
          ++tie_at;
        }
      }
      kept[c] = keep;
      w[c] = keep ? Units::Whole(of[c]) : 0;
      sum += w[c];
    }
  }
  const uint64_t upto = WaveInclScanU64(sum);
  if (lane == 63) sh.wave_sum[wave] = upto;
  __syncthreads();
  const uint64_t waves_upto = WaveInclScanU64(lane < kRowWaves ? sh.wave_sum[lane] : 0);
  const uint64_t total = LastLane(waves_upto);
  uint64_t seen = upto - sum + (wave > 0 ? Few::FromLane(waves_upto, wave - 1) : 0);
  const double weight = sh.weight_of_all;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    if (seen <= place && place < seen + w[c]) {
      a.tokens[row.r] = at + c;
      if (a.probs != nullptr) a.probs[row.r] = static_cast<float>(of[c] * unit / weight);
    }
    seen += w[c];
  }
  if (total > place) return;  // all of the workgroup, or none
  // rounding, u of 1, or weights of less than half a unit each, of which one is as near as another: the last kept one, those of
  // some weight before all of none
  uint32_t last = 0;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    if (kept[c]) last = max(last, (w[c] > 0 ? 0x80000000u : 0u) + static_cast<uint32_t>(at + c + 1));
  }
#pragma unroll
  for (int by = 32; by > 0; by >>= 1) last = max(last, static_cast<uint32_t>(__shfl_xor(static_cast<int>(last), by, 64)));
  if (lane == 0) sh.wave_last[wave] = last;
  __syncthreads();
  if (tid != 0) return;
  for (int i = 0; i < kRowWaves; ++i) last = max(last, sh.wave_last[i]);
  const int32_t token = static_cast<int32_t>(last & 0x7FFFFFFFu) - 1;
  a.tokens[row.r] = token;
  if (a.probs != nullptr) a.probs[row.r] = static_cast<float>(units.Of(row.LoadOne(token)) * unit / weight);
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
  RPG_CHECK(FitsLaunch(n_rows * slices, kThreads), "SampleBatch: %lld rows of %lld logits are too many for one call",
            static_cast<long long>(n_rows), static_cast<long long>(n));
  const SampleArgs a{logits_dev, row_stride, static_cast<int32_t>(n), slices, UnitsFor(n), opt.temperature, opt.top_k,
                     opt.top_p,  opt.min_p,  u_dev,                   tokens_dev, probs_dev, static_cast<char*>(workspace)};
  Launch("SampleSlicesKernel", SampleSlicesKernel, dim3(static_cast<unsigned>(n_rows * slices)), dim3(kThreads), a);
  Launch("SampleChooseKernel", SampleChooseKernel, dim3(static_cast<unsigned>(n_rows)), dim3(kRowThreads), a);
}

}  // namespace rpg
