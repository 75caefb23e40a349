// Device argmax and token sampling: the step after lm_head.
//
// Same C++ signatures as the reference sampler (src/sampler_gpu.h:62-128,
// src/sampler.h:35-46) so the generate loop (src/qwen3_gpu.cu:416, :553) links
// unchanged; GpuArgMax itself is declared with the layer operators in
// kernels_gpu.h (reference src/kernels_gpu.h:131-143).
//
// Semantics (what the parity tests hold the kernels to):
//   * temperature <= 0 (or NaN) is greedy: FilterToProbs gives a one-hot at the
//     argmax, SampleToken is GpuArgMax and consumes no random number;
//   * logits are scaled by float(1/T) when T != 1;
//   * top_k (1 < k < n): the threshold is the k-th largest value in the total
//     order of float bit patterns; values below it (float compare) are dropped,
//     ties with it kept;
//   * softmax: e = expf(v - max), summed in double, p = e * float(1/sum);
//   * top_p (0 < p < 1): with S(t) = sum of p_i over bit-pattern keys <= t, the
//     cut is the largest key with S <= 1 - top_p; every p_i <= cut becomes 0;
//     if nothing is left the argmax gets 1; then p *= float(1/sum) again, the
//     sum of the kept p taken on the same 2^-62 grid (within n * 2^-62 of the
//     double sum);
//   * inverse transform: the first index whose running double sum of p exceeds
//     u; if none does, the first maximum of p;
//   * u = CounterUniform(seed, counter) = (SplitMix64 of seed + gamma*counter)
//     >> 40, times 2^-24.
#ifndef RPG_AMD_SAMPLER_GPU_H_
#define RPG_AMD_SAMPLER_GPU_H_

#include <cstddef>
#include <cstdint>

namespace rpg {

// Sampling parameters (reference src/sampler.h:35-46): temperature <= 0 is
// greedy; top_k 0 disables the top-k filter; top_p 1 disables the nucleus cut.
struct SampleOptions {
  float temperature = 1.0f;
  int32_t top_k = 0;
  float top_p = 1.0f;
};

// Largest vocabulary the device sampler accepts (the per-slice partials live
// in a fixed-size scratch block).
constexpr int64_t kSamplerMaxVocab = int64_t(1) << 22;

// Counter-based random source, host side (reference src/sampler_gpu.h:71-73).
uint64_t DevSplitMix64(uint64_t x);
uint64_t DevCounterRng(uint64_t seed, uint64_t counter);
float DevCounterUniform(uint64_t seed, uint64_t counter);

// logits -> filtered, normalised probabilities (reference src/sampler_gpu.h:86-87).
// probs_dev holds >= n floats; logits_dev is not modified.
void GpuFilterToProbs(const float* logits_dev, int64_t n, const SampleOptions& opt, float* probs_dev);

// Inverse transform with a host u in [0, 1) (reference src/sampler_gpu.h:95-96).
// Not capturable (u would be frozen into the graph): throws while the engine
// stream is capturing.
void GpuInverseSample(const float* probs_dev, int64_t n, float u, int32_t* out_idx_dev);

// One token: greedy -> GpuArgMax; otherwise FilterToProbs then the inverse
// transform with u = CounterUniform(seed, counter) (reference src/sampler_gpu.h:108-110).
void GpuSampleToken(const float* logits_dev, int64_t n, const SampleOptions& opt, uint64_t seed, uint64_t counter,
                    float* probs_dev, int32_t* out_idx_dev);

// The same with the counter read on the device (the pos0 staging scalar), so a
// captured graph draws a fresh u on every replay (reference src/sampler_gpu.h:124-126).
void GpuSampleTokenDev(const float* logits_dev, int64_t n, const SampleOptions& opt, uint64_t seed,
                       const uint64_t* counter_dev, float* probs_dev, int32_t* out_idx_dev);

// Allocates the sampler's scratch block; call once before capturing a graph
// that samples or takes an argmax (reference src/sampler_gpu.h:130).
void GpuSamplerWarmup();

// ---------------------------------------------------------------- a batch's next tokens
//
// One token for each row of logits ([n_rows], row_stride floats apart, n of them), from
// a given random number for each. Beside GpuSampleTokenDev, whose u is
// DevCounterUniform's; no counterpart in the reference, which samples one row.
//
// Semantics: tokens are ordered by falling logit, equal ones by rising index. With
// weights w = exp((x - max x) / temperature), kept are
//   * the first top_k in that order (0 < top_k; else all), ties cut by index (the one-row
//     sampler keeps all that are tied with the k-th),
//   * of these the fewest first ones whose weight is at least top_p times that of all
//     of these (0 < top_p < 1; else all),
//   * of these those of w >= min_p (0 < min_p, above 1 as 1; else all).
// The token is the first in index order up to which the kept weights add up to more
// than u times their sum. u is taken into [0, 1), a NaN as 0. temperature <= 0 or NaN
// takes the first in order, with probability 1. A NaN logit counts as minus infinity,
// whose weight is 0, plus infinity as the largest finite number; a row of nothing but
// minus infinity gives token -1 and probability 0.
//
// Weights are formed in double, within 2^-36 of their value, and summed in units of
// 2^-38 of the largest, as integers, so that no order of summing shows and ties add up
// to what they should: a sum of weights, and with it a border, lies within n 2^-39 +
// 2^-36 of the whole of where exact weights have it (typically within 10^-9).
struct SampleBatchOptions {
  // device arrays of n_rows, each may be null: 1, off, off, off
  const float* temperature = nullptr;
  const int32_t* top_k = nullptr;
  const float* top_p = nullptr;
  const float* min_p = nullptr;
};

// probs_dev (may be null): the token's share of the kept weight. All arrays are read on
// the device: a captured call holds for what stands there at replay. workspace:
// GpuSampleBatchWorkspaceBytes of device memory, 256-byte aligned, of any contents; it
// serves calls one after the other, of any n_rows and n that need no more. Calls that
// may run at the same time need a workspace each.
void GpuSampleBatch(const float* logits_dev, int64_t n_rows, int64_t n, int64_t row_stride,
                    const SampleBatchOptions& opt, const float* u_dev, int32_t* tokens_dev, float* probs_dev,
                    void* workspace, size_t workspace_bytes);
size_t GpuSampleBatchWorkspaceBytes(int64_t n_rows, int64_t n);

}  // namespace rpg

#endif  // RPG_AMD_SAMPLER_GPU_H_
