// The table of functions that include/rpg_paged.h declares: each forwards to the
// C++ operator layer and converts exceptions into the negative-status /
// thread-local-message convention.
#include "../../include/rpg_paged.h"

#include <exception>
#include <new>

#include "common.h"
#include "kernels_gpu.h"

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

rpg::GpuPagedKv Kv(const rpg_paged_kv_t* kv) {
  RPG_CHECK(kv != nullptr, "null paged cache");
  rpg::GpuPagedKv out;
  out.type = kv->type;
  out.n_kv_heads = kv->n_kv_heads;
  out.head_dim = kv->head_dim;
  out.page_size = kv->page_size;
  out.n_pages = kv->n_pages;
  out.k = kv->k;
  out.v = kv->v;
  out.k_scale = kv->k_scale;
  out.v_scale = kv->v_scale;
  return out;
}

rpg::GpuPageTable Table(const rpg_page_table_t* t) {
  RPG_CHECK(t != nullptr, "null page table");
  return rpg::GpuPageTable{t->pages, t->n_seqs, t->max_pages};
}

int32_t KvWrite(const rpg_paged_kv_t* kv, const rpg_page_table_t* table, const int32_t* seq_ids,
                const int32_t* positions, const float* k, const float* v, int64_t n_tokens) {
  return Guard([&] { rpg::GpuKvWritePaged(Kv(kv), Table(table), seq_ids, positions, k, v, n_tokens); });
}

int32_t QkNormRopeKv(const rpg_paged_kv_t* kv, const rpg_page_table_t* table, const int32_t* seq_ids,
                     const int32_t* positions, const float* q, const float* k, const float* v, const float* q_norm,
                     const float* k_norm, int32_t n_heads, const float* rope_tab, int64_t rope_rows, int64_t n_tokens,
                     float eps, float* q_out) {
  return Guard([&] {
    rpg::GpuQkNormRopeKvPaged(Kv(kv), Table(table), seq_ids, positions, q, k, v, q_norm, k_norm, n_heads, rope_tab,
                              rope_rows, n_tokens, eps, q_out);
  });
}

int32_t KvRead(const rpg_paged_kv_t* kv, const rpg_page_table_t* table, const int32_t* seq_ids,
               const int32_t* positions, int64_t n_tokens, int32_t out_f32, void* k_out, void* v_out,
               int64_t token_stride, int64_t head_stride) {
  return Guard([&] {
    rpg::GpuKvReadPaged(Kv(kv), Table(table), seq_ids, positions, n_tokens, out_f32 != 0, k_out, v_out, token_stride,
                        head_stride);
  });
}

int32_t Attention(const rpg_paged_kv_t* kv, const rpg_page_table_t* table, const int32_t* seq_ids,
                  const int32_t* lens, const float* q, int32_t n_heads, int64_t n_rows, float* out, void* workspace,
                  int64_t workspace_bytes) {
  return Guard([&] {
    RPG_CHECK(workspace_bytes >= 0, "AttentionPaged: a workspace of negative size");
    rpg::GpuAttentionPaged(Kv(kv), Table(table), seq_ids, lens, q, n_heads, n_rows, out, workspace,
                           static_cast<size_t>(workspace_bytes));
  });
}

int64_t AttentionWorkspace(int32_t n_heads, int32_t n_kv_heads, int32_t head_dim) {
  int64_t bytes = 0;
  const int32_t rc = Guard([&] {
    bytes = static_cast<int64_t>(rpg::GpuAttentionPagedWorkspaceBytes(n_heads, n_kv_heads, head_dim));
  });
  return rc < 0 ? rc : bytes;
}

int32_t AttentionWorkspaceInit(void* workspace, int64_t bytes) {
  return Guard([&] {
    RPG_CHECK(bytes >= 0, "AttentionPagedWorkspaceInit: a workspace of negative size");
    rpg::GpuAttentionPagedWorkspaceInit(workspace, static_cast<size_t>(bytes));
  });
}

}  // namespace

// hipcc passes over a .cc for the device too and would place a constant there.
#ifndef __HIP_DEVICE_COMPILE__
extern "C" {
const rpg_paged_ops_t rpg_paged_ops = {sizeof(rpg_paged_ops_t), KvWrite,   QkNormRopeKv,       KvRead,
                                       Attention,               AttentionWorkspace, AttentionWorkspaceInit};
}
#endif
