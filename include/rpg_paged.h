/* rpg_paged.h -- C ABI of the operators over a paged KV cache.
 *
 * librpg_ops.so exports them as one table of functions, rpg_paged_ops, beside
 * the functions of rpg_ops.h, whose conventions hold here too: device pointers
 * of the caller's, asynchronous launches on the engine stream, status 0 or
 * negative with the reason in rpg_ops_last_error(), argument errors found before
 * anything is launched, no C++ exception across the boundary.
 *
 * The cache of a batch of sequences lies in pages of page_size positions, taken
 * from one pool per layer: position p of sequence s is slot p % page_size of page
 * pages[s * max_pages + p / page_size]. A slot holds one position's row of every
 * kv head, as fp16 or as 8-bit codes with an fp32 scale per row:
 *   scale = max|x| * fl(1/127), code = round(x * (1 / scale)), ties to even,
 * and the row stands for code * scale. A row whose scale would be subnormal is
 * kept as zeros, one that holds an infinity or a NaN as a NaN scale.
 *
 * seq_ids[t] (NULL: t itself) names row t's sequence, positions[t] its position;
 * both are device arrays, which like lengths and tables must stay as they are
 * while the call runs. A negative seq_id is padding: no slot is read or written
 * for that row, and no output. A row that names no slot (a sequence, position or
 * page out of range) stores nothing in the cache, and what the call gives back
 * for it is NaN. Rows of one call that name the same slot leave a mixture there.
 *
 * No counterparts in the reference, whose cache holds one sequence
 * (src/kv_cache_gpu.h:1-30); each entry names the operator it stands beside.
 */
#ifndef RPG_PAGED_H
#define RPG_PAGED_H

#include "rpg_ops.h"

#ifdef __cplusplus
extern "C" {
#endif

#define RPG_KV_F16 0u
#define RPG_KV_Q8 1u

/* One layer's pages. */
typedef struct {
  uint32_t type;      /* RPG_KV_F16 or RPG_KV_Q8 */
  int32_t n_kv_heads;
  int32_t head_dim;   /* 64 or 128 */
  int32_t page_size;  /* a power of two, 16 to 256 */
  int64_t n_pages;    /* at most 2^31 - 1 */
  void* k;            /* [n_pages][n_kv_heads][page_size][head_dim], 16-byte aligned: fp16 bits or int8 codes */
  void* v;
  float* k_scale;     /* RPG_KV_Q8: [n_pages][n_kv_heads][page_size], 16-byte aligned */
  float* v_scale;
} rpg_paged_kv_t;

/* pages [n_seqs][max_pages], on the device. */
typedef struct {
  const int32_t* pages;
  int64_t n_seqs;
  int64_t max_pages;
} rpg_page_table_t;

typedef struct {
  /* sizeof(rpg_paged_ops_t) of the library: what lies past it is not there. */
  int64_t size;

  /* Rows of k and v ([n_tokens][n_kv_heads][head_dim] fp32) into the cache.
   * Beside rpg_op_kv_write. */
  int32_t (*kv_write)(const rpg_paged_kv_t* kv, const rpg_page_table_t* table, const int32_t* seq_ids,
                      const int32_t* positions, const float* k, const float* v, int64_t n_tokens);

  /* q_out <- RoPE(RMSNorm(q) * q_norm) at each row's position (q_out may be q),
   * RoPE(RMSNorm(k) * k_norm) and v into the cache. q [n_tokens][n_heads][head_dim],
   * rope_tab [rope_rows][head_dim] (cos | sin). Beside rpg_op_qk_norm_rope_kv,
   * with its bits at head_dim 128. */
  int32_t (*qk_norm_rope_kv)(const rpg_paged_kv_t* kv, const rpg_page_table_t* table, const int32_t* seq_ids,
                             const int32_t* positions, const float* q, const float* k, const float* v,
                             const float* q_norm, const float* k_norm, int32_t n_heads, const float* rope_tab,
                             int64_t rope_rows, int64_t n_tokens, float eps, float* q_out);

  /* The rows back: element d of row t of kv head h to out[t * token_stride +
   * h * head_stride + d], fp16 bits (out_f32 0) or fp32 (1). Strides are in
   * elements, multiples of 8, and rows must not overlap, nor those of k_out those
   * of v_out (which may lie between them). (head_dim, max_seq * head_dim) gives a
   * layer of an rpg_kv. */
  int32_t (*kv_read)(const rpg_paged_kv_t* kv, const rpg_page_table_t* table, const int32_t* seq_ids,
                     const int32_t* positions, int64_t n_tokens, int32_t out_f32, void* k_out, void* v_out,
                     int64_t token_stride, int64_t head_stride);

  /* Row r of q ([n_rows][n_heads][head_dim]) attends to positions [0, lens[r]) of
   * its sequence; length 0 gives zeros. Scores, weights and sums have fp32's
   * precision, with three limits: what a query holds below 2^-30 of its row's largest
   * element does not count; values past 2^93 may add up to an infinity; an infinite
   * value of a weight below 2^-23 of the largest may give NaN in place of the
   * infinity. A captured call holds for any lengths,
   * tables and seq_ids at replay. out must not overlap q. Calls that may run at
   * the same time need a workspace each. Beside rpg_op_attention_from_cache. */
  int32_t (*attention)(const rpg_paged_kv_t* kv, const rpg_page_table_t* table, const int32_t* seq_ids,
                       const int32_t* lens, const float* q, int32_t n_heads, int64_t n_rows, float* out,
                       void* workspace, int64_t workspace_bytes);
  /* Bytes of an attention workspace for these heads (negative on error), and the
   * zeroing of one (256-byte aligned) that it needs before its first call. */
  int64_t (*attention_workspace)(int32_t n_heads, int32_t n_kv_heads, int32_t head_dim);
  int32_t (*attention_workspace_init)(void* workspace, int64_t bytes);
} rpg_paged_ops_t;

RPG_OPS_API extern const rpg_paged_ops_t rpg_paged_ops;

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* RPG_PAGED_H */
