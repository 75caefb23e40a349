// GpuKvCache storage and the host-built RoPE table.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <limits>
#include <vector>

#include "kernels_gpu.h"

namespace rpg {

GpuKvCache::GpuKvCache(const ModelMeta& c, int64_t max_seq)
    : n_layers_(c.n_layers), n_kv_heads_(c.n_kv_heads), head_dim_(c.head_dim), max_seq_(max_seq) {
  if (n_layers_ <= 0 || n_kv_heads_ <= 0 || head_dim_ <= 0) {
    Throw("GpuKvCache needs a model shape with layers, kv heads and a head size; got %d / %d / %d", n_layers_,
          n_kv_heads_, head_dim_);
  }
  if (max_seq_ <= 0) Throw("GpuKvCache: a cache of %lld positions holds nothing", static_cast<long long>(max_seq_));
  // Element count of one plane and of the whole block, refusing anything whose
  // byte size would not fit a size_t (a corrupt model shape, not a real cache).
  const double total = 2.0 * n_layers_ * static_cast<double>(n_kv_heads_) * static_cast<double>(max_seq_) *
                       head_dim_ * sizeof(uint16_t);
  if (total > static_cast<double>(std::numeric_limits<int64_t>::max() / 2)) {
    Throw("GpuKvCache: %d layers x %d kv heads x %lld positions x %d is too large to address", n_layers_,
          n_kv_heads_, static_cast<long long>(max_seq_), head_dim_);
  }
  plane_elems_ = static_cast<int64_t>(n_kv_heads_) * max_seq_ * head_dim_;
  // The whole capacity is reserved now, so running out of device memory is an
  // error of session creation rather than of a later generation step. No
  // clearing: rows at positions >= len() are never read, and every position
  // below it has been written by the fused q/k kernel or GpuKvWrite.
  store_.Alloc(static_cast<size_t>(2 * n_layers_ * plane_elems_) * sizeof(uint16_t));
}

uint16_t* GpuKvCache::Plane(int32_t layer, int plane) const {
  if (layer < 0 || layer >= n_layers_) {
    Throw("GpuKvCache has layers 0..%d; layer %d was requested", n_layers_ - 1, layer);
  }
  uint16_t* base = static_cast<uint16_t*>(const_cast<void*>(store_.data()));
  return base + (static_cast<int64_t>(plane) * n_layers_ + layer) * plane_elems_;
}

void GpuKvCache::SetLen(int64_t n) {
  if (n < 0 || n > max_seq_) {
    Throw("GpuKvCache: cannot mark %lld positions as filled in a cache of %lld", static_cast<long long>(n),
          static_cast<long long>(max_seq_));
  }
  len_ = n;
}

std::string GpuKvCache::Describe() const {
  char text[224];
  std::snprintf(text, sizeof(text),
                "fp16 KV cache: %d layers, %d kv heads, head_dim %d, %lld positions (%lld filled), %.1f MiB in one "
                "block",
                n_layers_, n_kv_heads_, head_dim_, static_cast<long long>(max_seq_), static_cast<long long>(len_),
                static_cast<double>(bytes()) / (1024.0 * 1024.0));
  return text;
}

// tab[p][i] = cos(p * w_i), tab[p][head_dim/2 + i] = sin(p * w_i) with
// w_i = 1 / theta^(2i / head_dim), every angle in double and rounded to fp32 once
// (the table src/gpu_model.cu:90-120 uploads). The inverse frequency is formed as a
// reciprocal of the power, as the reference forms it: pow(theta, -2i/d) differs from
// it in the last double bit for about a third of the i, which moves some fp32 table
// entries at positions past ~6500.
std::vector<float> BuildRopeTable(int32_t head_dim, double theta, int64_t n_pos) {
  return BuildRopeTableScaled(head_dim, theta, n_pos, RopeScaling());
}

std::vector<float> BuildRopeTableScaled(int32_t rot_dim, double theta, int64_t n_pos, const RopeScaling& scaling) {
  RPG_CHECK(rot_dim > 0 && rot_dim % 2 == 0, "RoPE needs an even head size, got %d", rot_dim);
  RPG_CHECK(theta > 0.0, "RoPE base theta must be positive, got %g", theta);
  const uint32_t type = scaling.type;
  const double factor = scaling.factor;
  RPG_CHECK(type <= kRopeYarn, "RoPE scaling %u is none of plain, linear, NTK and YaRN", type);
  RPG_CHECK(type == kRopePlain || (factor >= 1.0 && std::isfinite(factor)), "RoPE scaling factor %g is not 1 or more",
            factor);
  RPG_CHECK(scaling.attention >= 0.0 && std::isfinite(scaling.attention), "RoPE attention factor %g is out of range",
            scaling.attention);
  const int64_t rows = n_pos > 0 ? n_pos : 1;
  RPG_CHECK(rows <= (int64_t(1) << 40) / rot_dim, "a RoPE table of %lld positions is too large",
            static_cast<long long>(rows));
  const int32_t pairs = rot_dim / 2;
  const double base =
      type == kRopeNtk && rot_dim > 2 ? theta * std::pow(factor, static_cast<double>(rot_dim) / (rot_dim - 2)) : theta;
  double from = 0.0, to = 0.0;  // YaRN: the pairs that the ramp lies between
  if (type == kRopeYarn) {
    RPG_CHECK(scaling.original_positions > 0 && scaling.beta_slow > 0.0 && scaling.beta_fast >= scaling.beta_slow &&
                  std::isfinite(scaling.beta_fast) && theta > 1.0,
              "YaRN needs the original number of positions, 0 < beta_slow <= beta_fast and theta above 1");
    const auto pair_of = [&](double turns) {
      return rot_dim * std::log(static_cast<double>(scaling.original_positions) / (turns * 2.0 * M_PI)) /
             (2.0 * std::log(theta));
    };
    from = std::max(std::floor(pair_of(scaling.beta_fast)), 0.0);
    to = std::min(std::ceil(pair_of(scaling.beta_slow)), rot_dim - 1.0);
  }
  std::vector<double> freq(static_cast<size_t>(pairs));
  for (int32_t i = 0; i < pairs; ++i) {
    double w = 1.0 / std::pow(base, static_cast<double>(2 * i) / static_cast<double>(rot_dim));
    if (type == kRopeLinear) w /= factor;
    if (type == kRopeYarn) {
      const double r = std::min(std::max((i - from) / std::max(to - from, 0.001), 0.0), 1.0);
      w = w / factor * r + w * (1.0 - r);
    }
    freq[static_cast<size_t>(i)] = w;
  }
  const double by = scaling.attention != 0.0 ? scaling.attention : type == kRopeYarn ? 0.1 * std::log(factor) + 1.0 : 1.0;
  std::vector<float> tab(static_cast<size_t>(rows * rot_dim));
  float* out = tab.data();
  for (int64_t p = 0; p < rows; ++p, out += rot_dim) {
    for (int32_t i = 0; i < pairs; ++i) {
      const double angle = static_cast<double>(p) * freq[static_cast<size_t>(i)];
      out[i] = static_cast<float>(by * std::cos(angle));
      out[pairs + i] = static_cast<float>(by * std::sin(angle));
    }
  }
  return tab;
}

}  // namespace rpg
