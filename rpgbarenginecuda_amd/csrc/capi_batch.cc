// The table of functions that include/rpg_batch.h declares: each forwards to the
// C++ operator layer and converts exceptions into the negative-status /
// thread-local-message convention.
#include "../../include/rpg_batch.h"

#include <cstring>
#include <exception>
#include <new>

#include "common.h"
#include "kernels_gpu.h"
#include "sampler_gpu.h"

namespace {

template <typename F>
int32_t Guard(F&& f) {
  try {
    f();
    return RPG_OPS_OK;
  } catch (const rpg::Error&) {
    return -1;  // Throw already recorded the message
  } catch (const std::bad_alloc&) {
    rpg::SetLastError("out of host memory");
    return -2;
  } catch (const std::exception& e) {
    rpg::SetLastError(e.what());
    return -3;
  } catch (...) {
    rpg::SetLastError("unknown error");
    return -4;
  }
}

int32_t RopeTable(int32_t rot_dim, double theta, int64_t n_pos, const rpg_rope_scaling_t* scaling, float* out) {
  return Guard([&] {
    RPG_CHECK(out != nullptr && n_pos > 0, "rope_table needs n_pos > 0 and an output buffer");
    rpg::RopeScaling s;
    if (scaling != nullptr) {
      s.type = scaling->type;
      s.factor = scaling->factor;
      s.original_positions = scaling->original_positions;
      s.beta_fast = scaling->beta_fast;
      s.beta_slow = scaling->beta_slow;
      s.attention = scaling->attention;
    }
    const std::vector<float> t = rpg::BuildRopeTableScaled(rot_dim, theta, n_pos, s);
    std::memcpy(out, t.data(), t.size() * sizeof(float));
  });
}

int32_t RopeRows(const float* q, const float* k, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim,
                 int32_t rot_dim, int32_t interleaved, const float* rope_tab, int64_t rope_rows,
                 const int32_t* positions, int64_t n_rows, float* q_out, float* k_out) {
  return Guard([&] {
    rpg::GpuRopeRows(q, k, n_heads, n_kv_heads, head_dim, rot_dim, interleaved != 0, rope_tab, rope_rows, positions,
                     n_rows, q_out, k_out);
  });
}

int32_t Sample(const float* logits, int64_t n_rows, int64_t n, int64_t row_stride, const float* temperature,
               const int32_t* top_k, const float* top_p, const float* min_p, const float* u, int32_t* tokens,
               float* probs, void* workspace, int64_t workspace_bytes) {
  return Guard([&] {
    RPG_CHECK(workspace_bytes >= 0, "SampleBatch: a workspace of negative size");
    rpg::GpuSampleBatch(logits, n_rows, n, row_stride, rpg::SampleBatchOptions{temperature, top_k, top_p, min_p}, u,
                        tokens, probs, workspace, static_cast<size_t>(workspace_bytes));
  });
}

int64_t SampleWorkspace(int64_t n_rows, int64_t n) {
  int64_t bytes = 0;
  const int32_t rc = Guard([&] { bytes = static_cast<int64_t>(rpg::GpuSampleBatchWorkspaceBytes(n_rows, n)); });
  return rc < 0 ? rc : bytes;
}

}  // namespace

// hipcc passes over a .cc for the device too and would place a constant there.
#ifndef __HIP_DEVICE_COMPILE__
extern "C" {
const rpg_batch_ops_t rpg_batch_ops = {sizeof(rpg_batch_ops_t), RopeTable, RopeRows, Sample, SampleWorkspace};
}
#endif
