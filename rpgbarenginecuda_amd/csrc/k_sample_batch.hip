// The next tokens of a batch of conversations, from given random numbers (the semantics
// are listed in sampler_gpu.h).
//
// Weights exp((x - max) / T) are formed in double, which on this card costs what fp32
// does, and rounded to integers of 2^-s: sums are exact from there on, in any order, so
// that atomics may add them and every border (top-k's, top-p's, u's) is the same from
// run to run.
#include <hip/hip_runtime.h>

#include <cmath>

#include "dev_util.h"
#include "kernels_gpu.h"
#include "launch.h"
#include "paged_kv.h"
#include "sampler_gpu.h"

namespace rpg {
namespace {

constexpr int kRowThreads = 1024;
constexpr int kRowWaves = kRowThreads / 64;
constexpr int kBins = 2048;

struct SampleArgs {
  const float* logits;
  int64_t row_stride;
  int32_t n;
  int32_t scale_bits;  // s: weights are whole numbers of 2^-s
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  const float* u;
  int32_t* tokens;
  float* probs;
};

// ---------------------------------------------------------------- order and weights

// Order-preserving map of float values onto uint32; both zeros alike, NaN 0.
constexpr uint32_t kDead = 0x007FFFFFu;  // minus infinity's: keys up to it have no weight
__device__ __forceinline__ uint32_t KeyOf(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float ValueOf(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7FFFFFFFu) : ~key);
}

constexpr double InverseFactorial(int n) { return n <= 1 ? 1.0 : InverseFactorial(n - 1) / n; }

// 2^v for v <= 0: the Taylor series of e^g at g = (v - round(v)) ln 2, |g| <= 0.35, whose
// first term left out, g^12 / 12!, is below 2^-47; 0 below 2^-1000 and for a NaN.
__device__ __forceinline__ double Exp2Down(double v) {
  if (!(v >= -1000.0)) return 0.0;
  const double k = rint(v);
  const double g = (v - k) * 0.69314718055994530942;
  double p = InverseFactorial(11);
#pragma unroll
  for (int i = 10; i >= 0; --i) p = fma(p, g, InverseFactorial(i));
  return ldexp(p, static_cast<int>(k));
}

// A row's weights: of a value x, relative to the largest.
struct Weights {
  float top;
  double by;     // log2(e) / T
  double units;  // 2^s

  __device__ __forceinline__ double Of(float x) const {
    const double d = x == top ? 0.0 : static_cast<double>(x) - static_cast<double>(top);
    return Exp2Down(d * by);
  }
  __device__ __forceinline__ uint64_t Whole(double w) const { return static_cast<uint64_t>(fma(w, units, 0.5)); }
};

// floor and ceil of f times whole, for 0 <= f < 1, without rounding.
__device__ __forceinline__ uint64_t Part(float f, uint64_t whole, bool up) {
  const uint32_t bits = __float_as_uint(f);
  const int e = static_cast<int>(bits >> 23);
  const uint64_t m = (bits & 0x7FFFFFu) | (e > 0 ? 0x800000u : 0u);
  const int shift = 150 - max(e, 1);  // f = m 2^-shift
  if (shift >= 90) return up && m != 0 && whole != 0 ? 1 : 0;  // m whole < 2^86
  const unsigned __int128 product = static_cast<unsigned __int128>(m) * whole;
  const unsigned __int128 more = up ? (static_cast<unsigned __int128>(1) << shift) - 1 : 0;
  return static_cast<uint64_t>((product + more) >> shift);
}

// ---------------------------------------------------------------- a row by one workgroup

struct RowShared {
  uint64_t bins[kBins];
  uint64_t parts[kRowWaves];
  uint64_t found[2];
};

__device__ __forceinline__ uint64_t WaveMax(uint64_t x) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const uint64_t o = __shfl_xor(x, off, 64);
    x = o > x ? o : x;
  }
  return x;
}
__device__ __forceinline__ uint64_t WaveSum(uint64_t x) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
  return x;
}
template <class F>
__device__ __forceinline__ uint64_t RowReduce(uint64_t x, RowShared& sh, F f) {
  if ((threadIdx.x & 63) == 0) sh.parts[threadIdx.x >> 6] = x;
  __syncthreads();
  uint64_t r = sh.parts[0];
#pragma unroll
  for (int w = 1; w < kRowWaves; ++w) r = f(r, sh.parts[w]);
  __syncthreads();
  return r;
}
__device__ __forceinline__ uint64_t RowMax(uint64_t x, RowShared& sh) {
  return RowReduce(WaveMax(x), sh, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
}
__device__ __forceinline__ uint64_t RowSum(uint64_t x, RowShared& sh) {
  return RowReduce(WaveSum(x), sh, [](uint64_t a, uint64_t b) { return a + b; });
}
// The sum over the threads before this one; *total that over all.
__device__ __forceinline__ uint64_t RowBefore(uint64_t x, RowShared& sh, uint64_t* total) {
  uint64_t upto = x;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint64_t o = __shfl_up(upto, off, 64);
    if ((threadIdx.x & 63) >= off) upto += o;
  }
  if ((threadIdx.x & 63) == 63) sh.parts[threadIdx.x >> 6] = upto;
  __syncthreads();
  uint64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kRowWaves; ++w) {
    if (w < static_cast<int>(threadIdx.x >> 6)) before += sh.parts[w];
    all += sh.parts[w];
  }
  __syncthreads();
  *total = all;
  return before + upto - x;
}

// Kept are the keys above `key`, and of those equal to it the first `ties` in index order.
struct Cut {
  uint32_t key;
  uint64_t ties;
};

// The cut after the fewest first elements, in order, whose amounts (1, or their weight) reach `goal`, among those that
// `cut` keeps. Radix select over the keys from their upper digits down, each a pass over the row. The amounts of all ties
// of cut.key enter, which decides nothing: it is the last key.
template <bool kByWeight>
__device__ Cut Select(const float* x, int32_t n, const Weights& weights, const Cut& cut, uint64_t goal, RowShared& sh) {
  uint32_t prefix = 0;
  uint64_t above = 0;
  int known = 0;  // bits of the key that are found
#pragma unroll 1
  for (int level = 0; level < 3; ++level) {
    const int bits = level < 2 ? 11 : 10, shift = 32 - known - bits;
    for (int i = threadIdx.x; i < kBins; i += kRowThreads) sh.bins[i] = 0;
    __syncthreads();
    for (int32_t i = threadIdx.x; i < n; i += kRowThreads) {
      const uint32_t key = KeyOf(x[i]);
      if (key <= kDead || key < cut.key) continue;
      if (known > 0 && (key >> (32 - known)) != prefix) continue;
      const uint64_t a = kByWeight ? weights.Whole(weights.Of(x[i])) : 1;
      if (a != 0) {
        atomicAdd(reinterpret_cast<unsigned long long*>(&sh.bins[(key >> shift) & ((1u << bits) - 1)]),
                  static_cast<unsigned long long>(a));
      }
    }
    __syncthreads();
    // two bins to a thread, from the highest down
    const int b = kBins - 1 - 2 * static_cast<int>(threadIdx.x);
    const uint64_t hi = sh.bins[b], lo = sh.bins[b - 1];
    uint64_t unused;
    const uint64_t before = above + RowBefore(hi + lo, sh, &unused);
    if (before < goal && goal <= before + hi + lo) {
      const bool first = goal <= before + hi;
      sh.found[0] = static_cast<uint64_t>(first ? b : b - 1);
      sh.found[1] = first ? before : before + hi;
    }
    __syncthreads();
    const uint32_t digit = static_cast<uint32_t>(sh.found[0]);
    above = sh.found[1];
    prefix = (prefix << bits) | digit;
    known += bits;
    __syncthreads();
  }
  const uint64_t each = kByWeight ? weights.Whole(weights.Of(ValueOf(prefix))) : 1;
  return Cut{prefix, (goal - above + each - 1) / each};
}

// The index behind the cut's last tie.
__device__ int32_t TiesEnd(const float* x, int32_t n, const Cut& cut, RowShared& sh) {
  uint64_t seen = 0;
#pragma unroll 1
  for (int32_t base = 0; base < n; base += kRowThreads) {
    const int32_t i = base + static_cast<int32_t>(threadIdx.x);
    const bool tie = i < n && KeyOf(x[i]) == cut.key;
    uint64_t total;
    const uint64_t before = seen + RowBefore(tie ? 1 : 0, sh, &total);
    if (tie && before + 1 == cut.ties) sh.found[0] = static_cast<uint64_t>(i);
    seen += total;
    if (seen >= cut.ties) {
      __syncthreads();
      return static_cast<int32_t>(sh.found[0]) + 1;
    }
  }
  return n;
}

__global__ __launch_bounds__(kRowThreads) void SampleRowKernel(const SampleArgs a) {
  __shared__ RowShared sh;
  const int64_t r = blockIdx.x;
  const float* x = a.logits + r * a.row_stride;
  const int32_t n = a.n;
  const auto out = [&](int32_t token, float prob) {
    a.tokens[r] = token;
    if (a.probs != nullptr) a.probs[r] = prob;
  };
  const float t = a.temperature != nullptr ? a.temperature[r] : 1.0f;

  uint64_t best = 0;  // the largest key, and of these the lowest index
  for (int32_t i = threadIdx.x; i < n; i += kRowThreads) {
    const uint64_t k = static_cast<uint64_t>(KeyOf(x[i])) << 32 | (0xFFFFFFFFu - static_cast<uint32_t>(i));
    best = k > best ? k : best;
  }
  best = RowMax(best, sh);
  const uint32_t top_key = static_cast<uint32_t>(best >> 32);
  if (top_key <= kDead || !(t > 0.0f)) {
    if (threadIdx.x == 0) {
      if (top_key <= kDead) {
        out(-1, 0.0f);
      } else {
        out(static_cast<int32_t>(0xFFFFFFFFu - static_cast<uint32_t>(best)), 1.0f);
      }
    }
    return;
  }
  const Weights weights{ValueOf(top_key), 1.4426950408889634 / static_cast<double>(t), ldexp(1.0, a.scale_bits)};

  Cut cut{kDead, 0};
  const int32_t k = a.top_k != nullptr ? a.top_k[r] : 0;
  if (k > 0 && k < n) {
    uint64_t live = 0;
    for (int32_t i = threadIdx.x; i < n; i += kRowThreads) live += KeyOf(x[i]) > kDead ? 1 : 0;
    live = RowSum(live, sh);
    if (live > static_cast<uint64_t>(k)) cut = Select<false>(x, n, weights, cut, k, sh);
  }
  const float p = a.top_p != nullptr ? a.top_p[r] : 1.0f;
  if (p > 0.0f && p < 1.0f) {
    uint64_t all = 0;
    for (int32_t i = threadIdx.x; i < n; i += kRowThreads) {
      if (KeyOf(x[i]) > cut.key) all += weights.Whole(weights.Of(x[i]));
    }
    all = RowSum(all, sh);
    if (cut.ties > 0) all += cut.ties * weights.Whole(weights.Of(ValueOf(cut.key)));
    cut = Select<true>(x, n, weights, cut, Part(p, all, true), sh);
  }
  const float m = a.min_p != nullptr ? a.min_p[r] : 0.0f;
  const double least = m > 0.0f ? fmin(static_cast<double>(m), 1.0) : 0.0;

  const int32_t ties_end = cut.ties > 0 ? TiesEnd(x, n, cut, sh) : 0;
  const auto kept = [&](int32_t i) -> uint64_t {
    const uint32_t key = KeyOf(x[i]);
    if (key < cut.key || key <= kDead || (key == cut.key && i >= ties_end)) return 0;
    const double w = weights.Of(x[i]);
    return w >= least ? weights.Whole(w) : 0;
  };
  uint64_t all = 0;
  for (int32_t i = threadIdx.x; i < n; i += kRowThreads) all += kept(i);
  all = RowSum(all, sh);
  const float u = a.u[r];
  uint64_t goal = u > 0.0f ? (u < 1.0f ? Part(u, all, false) : all - 1) : 0;
  goal = goal < all ? goal : all - 1;
  uint64_t seen = 0;
#pragma unroll 1
  for (int32_t base = 0; base < n; base += kRowThreads) {
    const int32_t i = base + static_cast<int32_t>(threadIdx.x);
    const uint64_t w = i < n ? kept(i) : 0;
    uint64_t total;
    const uint64_t before = seen + RowBefore(w, sh, &total);
    if (before <= goal && goal < before + w) {
      out(i, static_cast<float>(weights.Of(x[i]) / (static_cast<double>(all) / weights.units)));
    }
    seen += total;
    if (seen > goal) return;
  }
}

// ---------------------------------------------------------------- host side

int32_t ScaleBits(int64_t n) {
  int32_t bits = 0;
  while ((int64_t(1) << bits) < n) ++bits;
  return 62 - bits;
}

void CheckSizes(const char* what, int64_t n_rows, int64_t n) {
  RPG_CHECK(n > 0 && n <= kSamplerMaxVocab, "%s: %lld logits a row, the limit is %lld", what,
            static_cast<long long>(n), static_cast<long long>(kSamplerMaxVocab));
  RPG_CHECK(n_rows >= 0 && n_rows <= (1 << 20), "%s: %lld rows", what, static_cast<long long>(n_rows));
}

}  // namespace

size_t GpuSampleBatchWorkspaceBytes(int64_t n_rows, int64_t n) {
  CheckSizes("SampleBatchWorkspace", n_rows, n);
  return 256;
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
  const SampleArgs a{logits_dev, row_stride,  static_cast<int32_t>(n), ScaleBits(n), opt.temperature, opt.top_k,
                     opt.top_p,  opt.min_p,   u_dev,                   tokens_dev,   probs_dev};
  Launch("SampleRowKernel", SampleRowKernel, dim3(static_cast<unsigned>(n_rows)), dim3(kRowThreads), a);
}

}  // namespace rpg
