/* rpg_batch.h -- C ABI of the operators for a step of many conversations, beside
 * those over their paged cache (rpg_paged.h): rotation of queries and keys at any
 * positions and in any of the usual forms, and the choice of every conversation's
 * next token.
 *
 * librpg_ops.so exports them as one table of functions, rpg_batch_ops, with the
 * conventions of rpg_ops.h: device pointers of the caller's, asynchronous launches
 * on the engine stream, status 0 or negative with the reason in
 * rpg_ops_last_error(), argument errors found before anything is launched, no C++
 * exception across the boundary.
 *
 * No counterparts in the reference, which serves one conversation; each entry names
 * the operator it stands beside.
 */
#ifndef RPG_BATCH_H
#define RPG_BATCH_H

#include "rpg_ops.h"

#ifdef __cplusplus
extern "C" {
#endif

#define RPG_ROPE_PLAIN 0u
#define RPG_ROPE_LINEAR 1u /* positions divided by factor */
#define RPG_ROPE_NTK 2u    /* theta * factor^(rot_dim / (rot_dim - 2)) */
#define RPG_ROPE_YARN 3u   /* slow pairs' frequencies divided, fast ones' kept */

typedef struct {
  uint32_t type;
  double factor;             /* at least 1 */
  int64_t original_positions; /* YARN: the length that the model was trained on */
  double beta_fast;          /* YARN: pairs of more turns than this over that length keep their frequency (32) */
  double beta_slow;          /* YARN: pairs of fewer turns than this have theirs divided (1) */
  double attention;          /* what cos and sin are multiplied by; 0: 0.1 ln(factor) + 1 for YARN, else 1 */
} rpg_rope_scaling_t;

typedef struct {
  /* sizeof(rpg_batch_ops_t) of the library: what lies past it is not there. */
  int64_t size;

  /* A rotation table [n_pos][rot_dim] (cos | sin), on the host; scaling NULL gives
   * rpg_ops_build_rope_table's bits. Beside that function. */
  int32_t (*rope_table)(int32_t rot_dim, double theta, int64_t n_pos, const rpg_rope_scaling_t* scaling, float* out);

  /* q_out <- q ([n_rows][n_heads][head_dim]) and k_out <- k ([n_rows][n_kv_heads]
   * [head_dim]), the first rot_dim elements of every head rotated by the row's
   * position: pairs (i, i + rot_dim / 2), or (2 i, 2 i + 1) if interleaved. The
   * rest of a head is copied. rope_tab [rope_rows][rot_dim] (cos | sin). A position
   * outside [0, rope_rows) gives NaN in the rotated elements. An output may be its
   * input; else it overlaps neither input nor the other output. k and k_out may be
   * NULL with n_kv_heads 0. At most 2^31 - 1 heads in all, 2^28 - 4 where head_dim or
   * rot_dim is no multiple of 8 or a buffer not 16-byte aligned. Beside rpg_op_rope. */
  int32_t (*rope_rows)(const float* q, const float* k, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim,
                       int32_t rot_dim, int32_t interleaved, const float* rope_tab, int64_t rope_rows,
                       const int32_t* positions, int64_t n_rows, float* q_out, float* k_out);

  /* tokens[r] <- a token of row r of logits ([n_rows], row_stride floats apart, n
   * of them), chosen by u[r]; probs[r] (may be NULL) <- its share of the weight
   * that the filters leave. temperature, top_k, top_p and min_p are device arrays
   * of n_rows, each NULL for 1, off, off, off; all are read on the device, so that
   * a captured call holds for what stands there at replay.
   *
   * Tokens are ordered by falling logit, equal ones by rising index; with weights
   * exp((x - max x) / temperature), kept are the first top_k (if 0 < top_k), of
   * these the fewest first ones of at least top_p times their weight (if 0 < top_p
   * < 1), and of these those of at least min_p (if 0 < min_p) times the largest;
   * the first always is. The token is the first in index order up to which the kept
   * weights add up to more than u times their sum; u is taken into [0, 1).
   * temperature <= 0 or NaN takes the first in order, with probability 1. A logit
   * that is a NaN counts as minus infinity, plus infinity as the largest finite
   * number; a row of nothing but minus infinity gives token -1 and probability 0.
   * Beside rpg_op_sample_token_dev, whose random numbers rpg_sample_counter_uniform
   * gives.
   *
   * workspace: sample_workspace bytes (negative on error), 256-byte aligned, of any
   * contents; calls that may run at the same time need one each. */
  int32_t (*sample)(const float* logits, int64_t n_rows, int64_t n, int64_t row_stride, const float* temperature,
                    const int32_t* top_k, const float* top_p, const float* min_p, const float* u, int32_t* tokens,
                    float* probs, void* workspace, int64_t workspace_bytes);
  int64_t (*sample_workspace)(int64_t n_rows, int64_t n);
} rpg_batch_ops_t;

RPG_OPS_API extern const rpg_batch_ops_t rpg_batch_ops;

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* RPG_BATCH_H */
