// Hot-path operators of the Qwen3 layer, MI355X (gfx950) implementation.
//
// The seven reference operators keep their exact C++ signatures
// (reference src/kernels_gpu.h), so the engine code that sequences them
// (src/qwen3_gpu.cu:47-109, 139-140, 168) links against this library unchanged:
//   GpuDequantRow        src/kernels_gpu.h:39-40
//   GpuRmsNorm           src/kernels_gpu.h:65-66
//   GpuRope              src/kernels_gpu.h:71-72
//   GpuKvWrite           src/kernels_gpu.h:97-99
//   GpuSiluMulInPlace    src/kernels_gpu.h:147
//   GpuVecAddInPlace     src/kernels_gpu.h:150
//   GpuEmbeddingLookup   src/kernels_gpu.h:153-154
// and three fused operators replace the unfused sequences of GpuForwardLayer:
//   GpuAddRmsNorm        GpuVecAddInPlace(x += d) ; GpuRmsNorm(x -> out)
//                        (src/qwen3_gpu.cu:100 -> 103, and :108 -> next layer's :69)
//   GpuQkNormRopeKv      GpuRmsNorm(q), GpuRmsNorm(k), GpuRope(q), GpuRope(k),
//                        GpuKvWrite(k, v)   (src/qwen3_gpu.cu:77-91)
//   GpuSiluMulInPlace    already one kernel in the reference (src/qwen3_gpu.cu:106)
//
// Conventions (same as the reference operator layer):
//   * every pointer is a device pointer; the caller owns all buffers;
//   * launches are asynchronous on EngineStream(); nothing synchronises;
//   * argument errors throw rpg::Error before anything is launched;
//   * out may alias x for RMSNorm / RoPE / SiLU-mul / add.
//
// Numerics (what the parity tests hold each operator to):
//   * dequant / gather: bit-exact with the reference CPU dequant (quant.cc):
//     Q4_K y = (d*sc)*q - (dmin*m), Q6_K y = (d*sc)*q, each op rounded
//     separately (the library is built with -ffp-contract=off);
//   * residual add: one IEEE fp32 add, bit-exact;
//   * fp16 KV store: IEEE round-to-nearest-even, bit-exact;
//   * RMSNorm: sum of squares accumulated in double, scale = float(1/sqrt(ss/n + eps)),
//     out = (x*scale)*w in fp32;  RoPE: a*c - b*s, b*c + a*s;  SiLU-mul: v/(1+exp(-v))*up.
#ifndef RPG_AMD_KERNELS_GPU_H_
#define RPG_AMD_KERNELS_GPU_H_

#include <cstdint>
#include <string>
#include <vector>

#include "hip_common.h"
#include "quant_types.h"

namespace rpg {

// ---------------------------------------------------------------- shapes

// Shapes and hyper-parameters of a model, with the reference's field names and
// types (src/model_meta.h:27-65); filled from a GGUF by ReadModelMeta
// (gpu_model.h) or by hand for single-operator use.
struct ModelMeta {
  std::string arch;  // "qwen3"
  std::string name;

  int32_t n_layers = 0;
  int32_t hidden = 0;
  int32_t n_heads = 0;
  int32_t n_kv_heads = 0;
  int32_t head_dim = 0;   // qwen3.attention.key_length
  int32_t value_dim = 0;  // qwen3.attention.value_length (== head_dim)
  int32_t intermediate = 0;
  int32_t vocab = 0;  // rows of token_embd
  int32_t context_length = 0;

  float rope_theta = 10000.0f;
  float rms_eps = 1e-6f;

  bool tied_embeddings = false;  // no output.weight / lm_head.weight: lm_head is token_embd

  int32_t bos_id = -1;
  int32_t eos_id = -1;
  int32_t pad_id = -1;
  bool add_bos = false;

  int64_t weight_bytes = 0;  // sum of every tensor's bytes in the file

  int32_t q_dim() const { return n_heads * head_dim; }
  int32_t kv_dim() const { return n_kv_heads * head_dim; }
  int32_t heads_per_kv() const { return n_kv_heads > 0 ? n_heads / n_kv_heads : 0; }
};

// A weight tensor resident in device memory as its raw GGUF bytes
// (reference src/gpu_model.h:42-55).
struct GpuTensor {
  DeviceBuffer buf;
  uint32_t type = kGgmlF32;
  bool matrix = false;
  int64_t rows = 0;  // dims[1]
  int64_t cols = 0;  // dims[0]
  int64_t n_elements = 0;

  bool valid() const { return !buf.empty(); }
  const char* type_name() const { return TypeName(type); }
  int64_t bytes() const { return static_cast<int64_t>(buf.size()); }
  int64_t row_bytes() const { return TypeRowBytes(type, cols); }
};

// Device-resident fp16 KV cache with the reference's layout: K, and V, each
// [n_layers][n_kv_heads][max_seq][head_dim] (src/kv_cache_gpu.h:1-30, :50-100),
// reached through the per-layer bases. The interface is the reference's; the
// storage is one device block per cache (all K layers, then all V layers), so
// a session costs a single allocation.
class GpuKvCache {
 public:
  GpuKvCache() = default;
  GpuKvCache(const ModelMeta& c, int64_t max_seq);

  int64_t len() const { return len_; }
  int64_t max_seq() const { return max_seq_; }
  int32_t n_layers() const { return n_layers_; }
  int32_t n_kv_heads() const { return n_kv_heads_; }
  int32_t head_dim() const { return head_dim_; }
  bool valid() const { return max_seq_ > 0; }

  // Base of layer `layer`: [n_kv_heads][max_seq][head_dim] fp16 bits.
  uint16_t* k_layer(int32_t layer) { return Plane(layer, 0); }
  uint16_t* v_layer(int32_t layer) { return Plane(layer, 1); }
  const uint16_t* k_layer(int32_t layer) const { return Plane(layer, 0); }
  const uint16_t* v_layer(int32_t layer) const { return Plane(layer, 1); }

  // Positions [0, len()) hold valid K / V rows; nothing else is ever read.
  void Reset() { len_ = 0; }
  void SetLen(int64_t n);
  void AddLen(int64_t n) { SetLen(len_ + n); }
  int64_t bytes() const { return static_cast<int64_t>(store_.size()); }
  std::string Describe() const;

 private:
  // Base of `layer` in plane 0 (K) or 1 (V).
  uint16_t* Plane(int32_t layer, int plane) const;

  int32_t n_layers_ = 0;
  int32_t n_kv_heads_ = 0;
  int32_t head_dim_ = 0;
  int64_t max_seq_ = 0;
  int64_t len_ = 0;
  int64_t plane_elems_ = 0;  // n_kv_heads * max_seq * head_dim
  DeviceBuffer store_;
};

// Host-built RoPE table, [n_pos][head_dim] fp32, cos in the first half of a row and
// sin in the second; angles computed in double (reference src/gpu_model.cu:90-120).
// n_pos = min(max_pos, context_length), at least 1.
std::vector<float> BuildRopeTable(int32_t head_dim, double theta, int64_t n_pos);

// The same for contexts longer than the model was trained on. With w_i = 1 /
// theta^(2i / rot_dim), the frequency of pair i is
//   kRopePlain   w_i (BuildRopeTable's bits);
//   kRopeLinear  w_i / factor, as if positions were divided;
//   kRopeNtk     w_i of theta * factor^(rot_dim / (rot_dim - 2)) (rot_dim 2: w_i),
//                so that the slowest pair's is divided and the fastest one's stays;
//   kRopeYarn    w_i (r / factor + 1 - r), r rising from 0 to 1 between the pairs that
//                turn beta_fast and beta_slow times over the original positions (their
//                indices floored and rounded up; Peng et al., YaRN, 2023).
// cos and sin are multiplied by `attention`, or where that is 0 by 0.1 ln(factor) + 1
// (kRopeYarn) or 1. The table serves every operator that takes one.
enum RopeScalingType : uint32_t { kRopePlain = 0, kRopeLinear = 1, kRopeNtk = 2, kRopeYarn = 3 };
struct RopeScaling {
  uint32_t type = kRopePlain;
  double factor = 1.0;  // at least 1
  int64_t original_positions = 0;
  double beta_fast = 32.0;
  double beta_slow = 1.0;
  double attention = 0.0;
};
std::vector<float> BuildRopeTableScaled(int32_t rot_dim, double theta, int64_t n_pos, const RopeScaling& scaling);

// ---------------------------------------------------------------- reference operators

void GpuDequantRow(uint32_t type, const uint8_t* src_dev, int64_t n_elems, float* dst_dev);

void GpuRmsNorm(const float* x, const float* w, int64_t n_rows, int64_t n, int64_t stride, float eps,
                float* out);

void GpuRope(float* x, int32_t n_heads, int32_t head_dim, const float* rope_tab, int64_t pos0,
             int64_t n_rows);

void GpuKvWrite(const float* k_dev, const float* v_dev, int32_t n_kv_heads, int32_t head_dim, int64_t pos0,
                int64_t seq, uint16_t* k_cache_layer, uint16_t* v_cache_layer, int64_t max_seq);

void GpuSiluMulInPlace(float* gate_dev, const float* up_dev, int64_t n);

void GpuVecAddInPlace(float* a_dev, const float* b_dev, int64_t n);

void GpuEmbeddingLookup(const GpuTensor& emb, const int32_t* toks_dev, int64_t seq, float* x_dev);

// GpuRope for rows at any positions and in any of the usual forms, queries and keys
// in one launch: q_out <- q ([n_rows][n_heads][head_dim]) and k_out <- k
// ([n_rows][n_kv_heads][head_dim]), where the first rot_dim elements of a head are
// rotated in pairs (i, i + rot_dim / 2), interleaved (2i, 2i + 1), by
//   a <- a cos - b sin,  b <- b cos + a sin
// with row positions[r] of rope_tab ([rope_rows][rot_dim], cos | sin), and the others
// copied. A position outside [0, rope_rows) gives NaN in the rotated elements. An
// output may be its input; else it must overlap neither an input nor the other
// output. k and k_out may be null with n_kv_heads 0. A call may have 2^31 - 1 heads in
// all, 2^28 - 4 where head_dim or rot_dim is no multiple of 8 or a buffer not 16-byte
// aligned. No counterpart in the reference,
// whose rows stand at consecutive positions (src/kernels_gpu.h:71-72).
void GpuRopeRows(const float* q, const float* k, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim,
                 int32_t rot_dim, bool interleaved, const float* rope_tab, int64_t rope_rows,
                 const int32_t* positions, int64_t n_rows, float* q_out, float* k_out);

// ---------------------------------------------------------------- fused operators

// x[r] += d[r] (one IEEE add, written back to x), then out[r] = RMSNorm(x[r]) * w.
// Rows are contiguous with stride n. out must not alias x or d.
void GpuAddRmsNorm(float* x, const float* d, const float* w, int64_t n_rows, int64_t n, float eps, float* out);

// Per token t (position pos0 + t):
//   q[t,h,:]  <- RoPE(RMSNorm(q[t,h,:]) * q_norm)          in place, h < n_heads
//   k'        <- RoPE(RMSNorm(k[t,h,:]) * k_norm)          h < n_kv_heads
//   k_layer[h][pos0+t][:] <- fp16_rne(k');  v_layer[h][pos0+t][:] <- fp16_rne(v[t,h,:])
//   if write_k_f32: k[t,h,:] <- k' (needed only by the no-cache attention path)
// rope_rows is the number of rows in rope_tab (bounds check on pos0 + seq).
void GpuQkNormRopeKv(float* q, float* k, const float* v, const float* q_norm, const float* k_norm,
                     int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, const float* rope_tab,
                     int64_t rope_rows, int64_t pos0, int64_t seq, float eps, uint16_t* k_cache_layer,
                     uint16_t* v_cache_layer, int64_t max_seq, bool write_k_f32);

// Embedding gather from a raw (non-owning) device table; GpuEmbeddingLookup
// forwards here. Token ids outside [0, rows) produce a zero row instead of an
// out-of-bounds read.
void GpuEmbeddingLookupRaw(uint32_t type, const uint8_t* emb_dev, int64_t rows, int64_t cols,
                           const int32_t* toks_dev, int64_t seq, float* x_dev);

// ---------------------------------------------------------------- attention

// Causal attention over the fp16 KV cache (src/kernels_gpu.h:113-116): for token
// t (absolute position pos0 + t) and query head h, softmax((q . k_j) / sqrt(d))
// over the cached positions j <= pos0 + t of kv head h / (n_heads / n_kv_heads),
// then the weighted sum of the v rows. q and out are [seq][n_heads][head_dim]
// fp32; k_layer / v_layer are one layer of the cache, [n_kv_heads][max_seq][d]
// fp16 bits. sh_positions > 0 fixes the position budget (needed under graph
// capture, where pos0 is read from the staging scalar at replay); otherwise
// pos0 + seq. head_dim must be 128.
void GpuAttentionFromCache(const ModelMeta& c, int64_t pos0, const float* q_dev, int64_t seq, const uint16_t* k_layer,
                           const uint16_t* v_layer, int64_t max_seq, float* out_dev, int64_t sh_positions = -1);

// One token at position pos0: GpuQkNormRopeKv (q / k per-head RMSNorm with
// q_norm / k_norm and eps = c.rms_eps, RoPE at pos0, k and v rounded to fp16
// into k_layer / v_layer at pos0) and GpuAttentionFromCache in one decode launch
// (plus the chunk merge when the keys are split), bit-identical to the two
// calls; q, k, v are the projections' raw [heads][128] rows and are not
// modified. Returns false, having launched nothing, when the shape has no fused
// kernel (head_dim != 128, a GQA group other than 1, 2, 4, pointers not 16-byte
// aligned); the caller then makes the two calls. No counterpart in the
// reference (src/qwen3_gpu.cu:77-96 runs norm, RoPE, KV write and attention as
// separate launches).
bool GpuQkNormRopeKvAttention(const ModelMeta& c, int64_t pos0, const float* q_dev, const float* k_dev,
                              const float* v_dev, const float* q_norm, const float* k_norm, const float* rope_tab,
                              int64_t rope_rows, uint16_t* k_layer, uint16_t* v_layer, int64_t max_seq,
                              float* out_dev, int64_t sh_positions = -1);

// Causal attention without a cache (src/kernels_gpu.h:82-84): the same maths
// over the segment's own fp32 rows, k / v [seq][n_kv_heads][head_dim], token t
// attending to tokens 0..t. The no-cache forward uses it; the difference from
// GpuAttentionFromCache on the same tokens is the fp16 rounding of k and v only.
void GpuCausalAttention(const ModelMeta& c, const float* q_dev, const float* k_dev, const float* v_dev, int64_t seq,
                        float* out_dev);

// GpuAttentionFromCache for callers that cannot allocate (code under HIP graph
// capture, serving loops that forbid hipMalloc): the same kernels and results,
// with the chunk partials in a fixed 8 MiB device array of the library instead
// of the grow-only buffer, so nothing is ever allocated. A call whose key split
// needs more partials than that (seq * n_heads * chunks * 132 floats > 2^21;
// the split aims at ~2048 waves, so this is reached only with GQA groups of 4
// and more than ~2000 (token, kv head) pairs) is rejected before anything
// launches. Every call on a device shares that
// device's array: calls that overlap on one device (two streams) race. No
// counterpart in the reference.
void GpuAttentionFromCacheNoAlloc(const ModelMeta& c, int64_t pos0, const float* q_dev, int64_t seq,
                                  const uint16_t* k_layer, const uint16_t* v_layer, int64_t max_seq, float* out_dev,
                                  int64_t sh_positions = -1);
// Looks up the fixed array's address on the current device (once per device;
// the entry point does it on first use if this was not called).
void GpuAttentionNoAllocInit();
size_t GpuAttentionNoAllocScratchBytes();

// Sizes the attention's partials buffer for up to sh_positions cached positions
// (decode calls), so that a graph capture of the decode step allocates nothing
// (src/kernels_gpu.h:128; there it raises the shared-memory limit instead).
void GpuAttentionWarmupShmem(int64_t sh_positions);

// ---------------------------------------------------------------- paged KV cache
//
// The cache of a batch of sequences, in pages of page_size positions taken from
// one pool per layer: position p of sequence s is slot p % page_size of page
// pages[s * max_pages + p / page_size]. A slot holds one position's row of every
// kv head, as fp16 or as 8-bit codes with an fp32 scale per row. All of it is
// device memory of the caller's. No counterpart in the reference, whose cache
// holds one sequence.
//
// Q8: a row x is kept as scale = max|x| * fl(1/127) and code = round(x * (1 /
// scale)) (ties to even, at most 127 either way); it stands for code * scale. A
// row whose scale would be subnormal is kept as zeros, one that holds an
// infinity or a NaN as a NaN scale, so that it reads back as NaN.
enum GpuKvType : uint32_t { kKvF16 = 0, kKvQ8 = 1 };

struct GpuPagedKv {
  uint32_t type = kKvF16;
  int32_t n_kv_heads = 0;
  int32_t head_dim = 0;   // 64 or 128
  int32_t page_size = 0;  // a power of two, 16 to 256
  int64_t n_pages = 0;    // at most 2^31 - 1
  void* k = nullptr;      // [n_pages][n_kv_heads][page_size][head_dim] fp16 bits or int8 codes
  void* v = nullptr;
  float* k_scale = nullptr;  // Q8: [n_pages][n_kv_heads][page_size]; F16: unused
  float* v_scale = nullptr;
};

struct GpuPageTable {
  const int32_t* pages = nullptr;  // [n_seqs][max_pages]; entries no token reaches are never read as pages
  int64_t n_seqs = 0;
  int64_t max_pages = 0;
};

// Where each row of a call goes is device data: seq_ids[t] (nullptr: t itself)
// names the sequence and positions[t] the position; they, like the lengths and
// the table, must stay as they are while the call runs. A negative seq_id is
// padding: no slot is read or written for that row, and no output. A row that
// names no slot
// (a sequence, position or page out of range) stores nothing in the cache, and
// what the call gives back for it is NaN. Two rows that name the same slot in
// one call leave it holding a mixture of both.

// Rows of k and v ([n_tokens][n_kv_heads][head_dim] fp32) into the cache.
void GpuKvWritePaged(const GpuPagedKv& kv, const GpuPageTable& table, const int32_t* seq_ids,
                     const int32_t* positions, const float* k_dev, const float* v_dev, int64_t n_tokens);

// GpuQkNormRopeKv over pages: q_out[t,h,:] <- RoPE(RMSNorm(q[t,h,:]) * q_norm) at
// the row's position (q_out may be q), RoPE(RMSNorm(k) * k_norm) and v into the
// cache; k and v are not modified, nor may q_out overlap them. At head_dim 128 q_out and an F16 cache hold
// the bits that GpuQkNormRopeKv leaves. A position at or past rope_rows is out of
// range.
void GpuQkNormRopeKvPaged(const GpuPagedKv& kv, const GpuPageTable& table, const int32_t* seq_ids,
                          const int32_t* positions, const float* q_dev, const float* k_dev, const float* v_dev,
                          const float* q_norm, const float* k_norm, int32_t n_heads, const float* rope_tab,
                          int64_t rope_rows, int64_t n_tokens, float eps, float* q_out);

// The rows back out of the cache: element d of row t of kv head h goes to
// out[t * token_stride + h * head_stride + d], as fp16 bits (out_f32 false) or
// fp32. Strides (in elements) are multiples of 8, and rows must not overlap:
// either whole tokens or whole heads follow each other. Rows of v_out may lie
// between those of k_out, but not over them. token_stride = head_dim,
// head_stride = max_seq * head_dim is one layer of a contiguous GpuKvCache.
void GpuKvReadPaged(const GpuPagedKv& kv, const GpuPageTable& table, const int32_t* seq_ids,
                    const int32_t* positions, int64_t n_tokens, bool out_f32, void* k_out, void* v_out,
                    int64_t token_stride, int64_t head_stride);

// Attention of one new token per row over the paged cache: row r (q and out
// [n_rows][n_heads][head_dim] fp32) attends to positions [0, lens[r]) of its
// sequence, softmax((q . k_j) / sqrt(head_dim)) over them, query head h reading kv
// head h / (n_heads / n_kv_heads). A row of length 0 gives zeros; padding
// (negative seq_id) leaves its out row as it was; a length below 0 or past the
// table's row, a sequence out of range, or a page out of range among the row's
// positions gives NaN. out must not overlap q. The work is shared out on the
// device from the lengths themselves, so a captured call holds for any lengths,
// tables and seq_ids that stand there at replay. A call whose rows have room for
// 2^31 units (32 positions of a kv head and 8 of its query heads) is refused.
//
// Scores, weights and sums have fp32's precision, within these limits: of a query,
// what is below 2^-30 of its row's largest element (fp16 pages: 2^-38) does not
// count; a weight below 2^-120 of the row's largest may count as none, and over fp16 pages
// any weight is off by up to 2^-39 of it; weights times
// values that add up to more than fp32 holds before the sum of weights divides them
// (values past 2^93) may give an infinity; an infinite value whose weight is below
// 2^-23 of the largest may give NaN instead of the infinity.
//
// workspace: GpuAttentionPagedWorkspaceBytes of device memory, 256-byte aligned,
// whose bytes are zero before the first call (GpuAttentionPagedWorkspaceInit
// does that); each call leaves it ready for the next on the same stream. Calls
// that may run at the same time need a workspace each.
void GpuAttentionPaged(const GpuPagedKv& kv, const GpuPageTable& table, const int32_t* seq_ids, const int32_t* lens,
                       const float* q_dev, int32_t n_heads, int64_t n_rows, float* out_dev, void* workspace,
                       size_t workspace_bytes);
size_t GpuAttentionPagedWorkspaceBytes(int32_t n_heads, int32_t n_kv_heads, int32_t head_dim);
void GpuAttentionPagedWorkspaceInit(void* workspace, size_t bytes);

// GpuAttentionPaged for a batch whose sequences share their beginnings (a system
// prompt, a world's description): rows [group_rows[g], group_rows[g + 1]) form group
// g, whose sequences' tables begin with the same group_pages[g] pages. These are
// attended to once for the group, what is behind them by each row. group_rows
// ([n_groups + 1]) and group_pages ([n_groups]) are device arrays, read when the call
// runs as lens and tables are; n_groups is at most 64.
//
// Which pages a group shares is read from the table of its first row that has them
// all; the tables of the others have to name the same ones. A row that does not reach
// behind them, or is in no group, is attended to by itself; one in several groups
// belongs to the first of these. Of a group out of range, what lies inside [0, n_rows)
// counts; one of no pages, fewer or more than a table has, shares none. Results and limits are
// GpuAttentionPaged's, but that an infinity or a NaN among a group's keys and values,
// or a page out of range, may give NaN in all of the group's rows whose output it
// reaches. At shared positions queries and weights count to 2^-22 of their value; over
// 8-bit pages weight times scale to 2^-37 of the largest besides.
//
// Sharing pays where it saves much reading: groups that together save less than
// least_saving bytes of keys and values (of each group all rows but one, times its
// pages) share nothing, and each row is attended to by itself. Rows that stand idle or
// do not reach behind the shared pages count with the others there: where a batch has
// many, least_saving is the caller's to set. A negative least_saving
// stands for what was measured to break even, 144 MB and one more for each row; 0
// shares always. Where not even all rows with all pages of a table would save as much,
// the call is GpuAttentionPaged's one launch. One that may share is refused where its
// outputs reach 2^34 elements, or where the groups, each of all rows, would have room
// for 2^31 units (128 positions of a kv head, for 128 rows times query heads).
//
// workspace: GpuAttentionPagedSharedWorkspaceBytes for n_rows or more, else as for
// GpuAttentionPaged (GpuAttentionPagedWorkspaceInit zeroes it).
void GpuAttentionPagedShared(const GpuPagedKv& kv, const GpuPageTable& table, const int32_t* seq_ids,
                             const int32_t* lens, const int32_t* group_rows, const int32_t* group_pages,
                             int32_t n_groups, const float* q_dev, int32_t n_heads, int64_t n_rows, float* out_dev,
                             void* workspace, size_t workspace_bytes, int64_t least_saving = -1);
size_t GpuAttentionPagedSharedWorkspaceBytes(int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, int64_t n_rows);

// ---------------------------------------------------------------- quantised matmul

// OUT[t, r] = dot(row r of W, row t of X), i.e. OUT = X . W^T (src/kernels_gpu.h:42-49):
//   W   [rows, cols] quantised (raw GGUF bytes on the device, Q4_K / Q6_K / F32)
//   X   [n_tokens, cols] fp32, row-major
//   OUT [n_tokens, rows] fp32, row-major
// Weights are dequantised bit-exactly and accumulated in fp32 (fused multiply-add).
void GpuMatMulQuant(const GpuTensor& w, const float* X_dev, int64_t n_tokens, float* OUT_dev);

// Path-equivalence switch (src/kernels_gpu.h:51-58): while set, GpuMatMulQuant
// and the grouped / fused matmul entry points run the generic kernel
// (MatMulGenericKernel: per-element decode, one wave per output) instead of the
// decode, tiled and matrix-core kernels; the norm-fused entry points then
// return false. For verification only: the specialised kernels are checked bit
// for bit against it on inputs where every summation order is exact. Off by
// default; the flag is process-wide.
void GpuSetForceGenericMatMul(bool force);
bool GpuForceGenericMatMul();

// GpuMatMulQuant over several matrices that read the same X (a layer's q / k / v,
// or gate / up): OUT_i = X . W_i^T. At n_tokens = 1, up to 4 Q4_K / Q6_K
// matrices (either type or both) are decoded in one launch, else each run of
// consecutive same-type matrices is; on the matrix-core path
// X is split once for all the matrices; otherwise one call per matrix. Every
// output is bit-identical to its own GpuMatMulQuant call. No counterpart in the
// reference (which launches once per matrix).
void GpuMatMulQuantGroup(const GpuTensor* const* ws, int32_t n_mats, const float* X_dev, int64_t n_tokens,
                         float* const* OUTs);

// The layer's gate / up projections and SwiGLU (src/qwen3_gpu.cu:104-106):
// gate <- silu(X . W_gate^T) * (X . W_up^T); up is scratch (it holds X . W_up^T
// after a multi-token call, and is left untouched at one token). At one token on
// same-type matrices of <= 2048 columns it is one launch: each wave computes
// row p of both matrices and writes the SwiGLU of the two totals. Bit-identical
// to GpuMatMulQuantGroup({gate, up}) + GpuSiluMulInPlace. No counterpart in the
// reference.
void GpuMatMulQuantSwiGLU(const GpuTensor& w_gate, const GpuTensor& w_up, const float* X_dev, int64_t n_tokens,
                          float* gate_dev, float* up_dev);

// The sub-layer norm in front of a one-token matmul (the reference runs
// GpuVecAddInPlace, GpuRmsNorm and the matmul as separate launches,
// src/qwen3_gpu.cu:69-76,100-104,168): v = x + d (d == nullptr: v = x),
// h = RMSNorm(v) * w as GpuAddRmsNorm computes it, and the matmul of h. Each
// launch forms h itself, so no h buffer is written; x_out (optional) receives v,
// bit-exact, and must not alias x or d. The scale's double sum of squares is
// taken in another order than GpuAddRmsNorm's, so h can differ from it in the
// last fp32 bit. All of x, d, w, x_out 16-byte aligned.
struct GpuNormIn {
  const float* x;
  const float* d;
  const float* w;
  float eps;
  float* x_out;
};

// GpuMatMulQuantGroup at one token on RMSNorm(x + d) * w. Returns false, having
// launched nothing, when the group has no fused form (a matrix that is not
// Q4_K / Q6_K, more than 2048 columns, misaligned pointers); the caller then
// runs GpuAddRmsNorm and GpuMatMulQuantGroup. No counterpart in the reference.
bool GpuNormMatMulQuantGroup(const GpuNormIn& in, const GpuTensor* const* ws, int32_t n_mats, float* const* OUTs);

// GpuMatMulQuantSwiGLU at one token on RMSNorm(x + d) * w; false as above. No
// counterpart in the reference.
bool GpuNormMatMulQuantSwiGLU(const GpuNormIn& in, const GpuTensor& w_gate, const GpuTensor& w_up, float* gate_dev,
                              float* up_dev);

// The same on a raw (non-owning) weight pointer; GpuMatMulQuant forwards here.
void GpuMatMulQuantRaw(uint32_t type, const uint8_t* w_dev, int64_t rows, int64_t cols, const float* x_dev,
                       int64_t n_tokens, float* out_dev);

// ---------------------------------------------------------------- argmax

// Index of the largest of x[0..n) (src/kernels_gpu.h:131-143): only values above
// -FLT_MAX count (none -> 0), ties go to the smallest index, NaN never wins.
// n <= kSamplerMaxVocab (sampler_gpu.h, which declares the sampler around it).
void GpuArgMax(const float* x_dev, int64_t n, int32_t* out_idx_dev);

// ---------------------------------------------------------------- measurement / verification

// Streaming copy of `bytes` (multiple of 16) used to calibrate bandwidth and
// HBM counters (the reference's streaming-bandwidth probe, tools/matmul_bench.cu:230-289).
void GpuStreamCopy(const void* src, void* dst, int64_t bytes);

// Write-only probe: every 32-bit word of dst <- pattern (`bytes` a multiple of 16).
void GpuStreamFill(void* dst, int64_t bytes, uint32_t pattern);

// Read-only probe: reads `bytes` (a multiple of 16) of src and writes nothing
// unless the XOR fold of some thread's words equals `key` (then that fold goes to
// *sink). The reference's read probe (BwReadKernel, tools/matmul_bench.cu:239-250).
void GpuStreamRead(const void* src, int64_t bytes, uint32_t key, uint32_t* sink);

// out[i] = binary16 bits i converted to fp32, i in [0, 65536): exhaustive check
// of the device f16 -> f32 conversion (tools/dequant_check.cu:44-48).
void GpuF16Sweep(float* out_dev);

}  // namespace rpg

#endif  // RPG_AMD_KERNELS_GPU_H_
