// Attention of one new token per row over a paged cache whose rows share their beginnings:
// here the shared positions, once for all rows of a group, and the join with what each row's own
// positions came to, which k_attention_paged.hip has left in the output just before.
//
// For row r of a group, query head h, over the group's positions j < pages * page_size:
//   m = max_j s_j,  l = sum_j 2^(s_j - m),  o = sum_j 2^(s_j - m) v_j,  s_j = (q . k_j) log2(e) / sqrt(D),
// over its own ones m', l' and the output o' / l'; joined (o f + o' f') / (l f + l' f') with f = 2^(m - M),
// f' = 2^(m' - M), M the larger of m and m'.
//
// Keys and values are read once for up to 128 columns (the queries of a kv head: rows times heads of a group). Queries and
// weights, which are fp32, enter the matrix cores as two fp16 terms of 11 bits each, together 22, so that each product runs
// twice. Over 8-bit pages codes are fp16 numbers as they are; keys' scales multiply the scores, and weights times values'
// scales are brought to fp16's range by a power of two of the column's, relative to the largest yet and what that counts for
// now: a row of a large scale that has lost its weight costs the others nothing.
//
// A workgroup takes steps of 128 positions through LDS, two of them at a time (one being read, one being filled), for a
// tile of up to 128 columns; of its eight waves each has 16 columns and all of a step's keys, a half or a quarter of them
// where the tile has no more than 64 or 32 columns. The products are those of k_attention_paged.hip: rows of S = K Q^T are
// 16 keys, rows of O^T = V^T P^T 16 elements, so that a lane ends the first with the weights of the keys that it holds in
// the second. The units (kv head, column tile, step) of all groups are shared out evenly and contiguously. A tile that one
// workgroup holds it joins with the rows' own parts by itself; the parts of others are left in the workspace for a small
// kernel that joins them in order, over all compute units: the last workgroup of a tile to arrive, on its one, took 18 us for
// four parts of 128 columns where that takes 4.
//
// What bounds it: 32 positions of 128 columns take a compute unit some 2750 cycles, of which the matrix cores are busy for
// 1030 and vector arithmetic for 1360, by two waves that mostly wait for the same; 32 columns to a wave (half the reads of LDS)
// and sixteen waves were no faster, and their code and joins cost the short pieces 4 us. Behind few columns it is memory
// (4 TB/s), and for one or two steps the chain of groups, lengths, table, keys and the first pass through the code, 8 us.
// 128 rows and 4 heads to a kv head over 8192 positions in 8 bits 59 us (0.58 PFLOP/s of formed products), 8 rows over
// 32768 26 us, 32 rows and 2 heads over 2816 in fp16 10.8 us.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "attention_dev.h"
#include "dev_util.h"
#include "kernels_gpu.h"
#include "launch.h"
#include "paged_kv.h"

namespace rpg {
namespace {

using namespace attn;
using dev::PagedView;

constexpr int kWaves = 8;
constexpr int kThreads = 64 * kWaves;
constexpr int kCols = 128;     // columns of a tile
constexpr int kStep = 128;     // positions of a unit: 16 for each wave to bring in
constexpr int kGroups = 256;   // workgroups: one to a compute unit
constexpr int kJoinThreads = 64;

// What a workgroup leaves of a tile that it has a part of: o [column][D], then (m, l) [column].
__host__ __device__ constexpr uint32_t SlotBytes(int d) { return kCols * (4u * d + 8u); }

struct PrefixArgs {
  PagedView view;
  PagedPrefix prefix;
  const int32_t* seq_ids;
  const int32_t* lens;
  const float* q;
  float* out;
  char* workspace;  // slots: two of a workgroup, for the first tile that it has a part of and for another
  int32_t n_rows;
  int32_t capacity;  // positions that a table row has pages for, at most the largest int32
  int32_t n_heads;
  int32_t group;  // query heads of a kv head
  float scale_log2;
};

// The two fp16 terms of a pair of values times `by`, a power of two: rounded to 11 bits, and what that leaves rounded to 11.
// (Instructions that multiply, add and round to either half of a register: two for each value.)
struct Terms {
  uint32_t hi, lo;
};
__device__ __forceinline__ Terms TermsOf(float a, float b, float by) {
  const Half2 hi = {static_cast<_Float16>(fmaf(a, by, 0.0f)), static_cast<_Float16>(fmaf(b, by, 0.0f))};
  const Half2 lo = {static_cast<_Float16>(fmaf(a, by, -static_cast<float>(hi[0]))),
                    static_cast<_Float16>(fmaf(b, by, -static_cast<float>(hi[1])))};
  return Terms{Bits(hi), Bits(lo)};
}

// Four codes as fp16: 1024 + 128 + code by their bits, less 1152.
__device__ __forceinline__ uint2 CodesToHalves(uint32_t codes) {
  const uint32_t u = codes ^ 0x80808080u;
  const Half2 by = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
  const Half2 lo = __builtin_bit_cast(Half2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + by;
  const Half2 hi = __builtin_bit_cast(Half2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + by;
  return make_uint2(Bits(lo), Bits(hi));
}
// What row_head's own positions came to: the maximum and the sum of its output, which is divided by that.
struct Own {
  float m, l;
};
__device__ __forceinline__ Own OwnOf(const PrefixArgs& a, int64_t row_head) {
  const float2 ml = *reinterpret_cast<const float2*>(a.prefix.ml + 2 * row_head);
  return Own{ml.x, ml.y};
}
// The two joined. (An own part of no weight, all of whose scores are minus infinity, is no number: it is left out.)
struct Both {
  float of_own, of_shared;
  bool none;
  __device__ __forceinline__ Both(const Own& own, float m, float l) {
    const float top = fmaxf(own.m, m);
    const float safe = top == -INFINITY ? 0.0f : top;
    const float f = own.l * __builtin_amdgcn_exp2f(own.m - safe), g = __builtin_amdgcn_exp2f(m - safe);
    const float inv = 1.0f / fmaf(l, g, f);
    of_own = f * inv;
    of_shared = g * inv;
    none = own.l == 0.0f;
  }
  __device__ __forceinline__ float4 Of(float4 own, float4 o) const {
    if (none) own = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    return make_float4(fmaf(own.x, of_own, o.x * of_shared), fmaf(own.y, of_own, o.y * of_shared),
                       fmaf(own.z, of_own, o.z * of_shared), fmaf(own.w, of_own, o.w * of_shared));
  }
};

// What a workgroup does of a tile: steps [c0, c1) of its `steps`.
struct Piece {
  uint32_t first_unit, c0, c1, steps;
  int32_t of;  // group
  int32_t first_row, last_row, pages, positions;
  int32_t kv_head, tile, cols;  // cols: of the tile
  bool leads;  // the first thing that the workgroup does
};

// Products of queries' and keys' codes, below 2^29, times scales up to this stay in fp32's range.
constexpr float kFarScale = 0x1p60f;

template <int D, bool kQ8>
struct Stage {
  static constexpr int kRow = 2 * D;
  alignas(16) char k[kStep * kRow];
  alignas(16) char v[kStep * kRow];
  float k_scale[kQ8 ? kStep : 4], v_scale[kQ8 ? kStep : 4];
  uint32_t bad[kStep / 16];  // 1: pages out of range, 2: keys' scales past kFarScale
};

// The groups' units, a group to a lane: those of kv head, column tile and step count up, in this order.
struct Units {
  dev::SharedGroups groups;
  uint32_t cols, tiles, steps, amount, upto;
  uint32_t all, sharers;  // the workgroups that share them out

  __device__ __forceinline__ Units(const PrefixArgs& a, int lane)
      : groups(a.prefix.group_rows, a.prefix.group_pages, a.prefix.n_groups, a.prefix.least, a.n_rows, a.view.max_pages, lane) {
    cols = static_cast<uint32_t>(groups.last - groups.first) * a.group;
    tiles = (cols + kCols - 1) / kCols;
    steps = (PositionsOf(a, groups.pages) + kStep - 1) / kStep;
    amount = tiles * steps * a.view.n_kv;
    upto = ScanAdd(amount);
    all = __builtin_amdgcn_readlane(upto, 63);
    sharers = min(static_cast<uint32_t>(kGroups), all);
  }
  static __device__ __forceinline__ uint32_t PositionsOf(const PrefixArgs& a, int32_t pages) {
    return pages <= (a.capacity >> a.view.page_shift) ? static_cast<uint32_t>(pages) << a.view.page_shift : 0u;
  }
};

// x, from which what follows is worked out where it stands: hoisted out of the loop of steps, the addresses that come of it
// take more registers than there are, and a value that comes back from memory waits for all loads before it.
template <class T>
__device__ __forceinline__ T Afresh(T x) {
  asm volatile("" : "+v"(x));
  return x;
}

// A row, the lane's, as asked for: requested apart from where it is looked at, so that other loads go out in between.
struct AskedRow {
  int32_t seq = -1, len = 0;
  __device__ __forceinline__ AskedRow(const PrefixArgs& a, int32_t r, bool there) {
    if (there) {
      seq = a.seq_ids != nullptr ? a.seq_ids[r] : r;
      len = a.lens[r];
    }
  }
  // whether it begins with all of its group's pages
  __device__ __forceinline__ bool BeginsWith(const PrefixArgs& a, int32_t pages) const {
    return seq >= 0 && seq < a.view.n_seqs && len >= 0 && len <= a.capacity && dev::TakesPart(pages, a.view.page_shift, len);
  }
};
// Whether r, among the rows that group `of` names, is its own: no earlier group's. Of all lanes at once, as OfLane is.
__device__ __forceinline__ bool IsOf(const dev::SharedGroups& groups, int32_t r, int32_t of, bool there) {
  const bool own = groups.n == 1 || groups.OfLane(there ? r : -1) == of;
  return there && own;
}

template <int D, bool kQ8>
__device__ __forceinline__ void AttendPiece(const PrefixArgs& args, const dev::SharedGroups& groups, uint32_t me,
                                            const Piece& piece, const int32_t* table, Stage<D, kQ8> (&stages)[2]) {
  constexpr int kRow = 2 * D;              // bytes of a row in LDS
  constexpr int kPieces = kRow / 16;       // of 16 bytes
  constexpr int kSource = kQ8 ? D : 2 * D;  // bytes of a cached row
  constexpr int kLoads = kSource / 64;     // loads of 64 pieces for 16 rows
  constexpr int kSourcePieces = kSource / 16;
  constexpr int kSteps = D / 32;           // products of 16 keys
  constexpr int kE = D / 16;               // tiles of 16 elements of a value row
  constexpr int kTiles = kStep / 16;
  constexpr int kPart = D + 4;             // floats of a joined column: o, m, l
  constexpr int kWaveCols = 16;
  static_assert(kTiles == kWaves, "a wave brings in 16 positions");
  static_assert(3 * 32 * kPart * 4 <= sizeof(stages), "joins fit where keys were");

  const PagedView& view = args.view;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int n = lane & 15;
  const int g = lane >> 4;
  const int32_t positions = piece.positions, kh = piece.kv_head;
  const uint32_t c0 = piece.c0, c1 = piece.c1;

  // ---- bringing in: this wave's 16 positions of a step, their pieces permuted as the reads below need them
  const auto k_swap = [](int r) { return kPieces == 16 ? r & 15 : r & 7; };
  const auto v_swap = [](int r) { return 2 * (r & (kPieces == 16 ? 7 : 3)); };
  struct Loaded {
    float4 k[kLoads], v[kLoads];
    float k_scale, v_scale;  // of row lane % 16
    uint32_t bad;
    bool got;
  };
  Loaded loaded;
  const auto page_of = [&](uint32_t c) {
    const int32_t pos = static_cast<int32_t>(c * kStep) + 16 * wave;
    return c < c1 && pos < positions ? ScalarLoad(table + (pos >> view.page_shift)) : 0;
  };
  const auto load = [&](Loaded& to, uint32_t c, int32_t page) {
    const int32_t pos = static_cast<int32_t>(c * kStep) + 16 * wave;
    to.got = c < c1 && pos < positions;
    to.bad = 0;
    if (!to.got) return;
    const bool fine = static_cast<uint32_t>(page) < static_cast<uint32_t>(view.n_pages);
    to.bad = fine ? 0 : 1;
    const int64_t at = ((static_cast<int64_t>(fine ? page : 0) * view.n_kv + kh) << view.page_shift) +
                       (pos & ((1 << view.page_shift) - 1));
    const auto rows = [&](const void* base, int64_t bytes) {
      return dev::OutResource(const_cast<char*>(static_cast<const char*>(base)) + at * bytes, static_cast<uint32_t>(16 * bytes));
    };
    const __amdgpu_buffer_rsrc_t k = rows(view.k, kSource), v = rows(view.v, kSource);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      to.k[i] = dev::LoadBuf4<0>(k, 1024u * i + 16u * lane);
      to.v[i] = dev::LoadBuf4<0>(v, 1024u * i + 16u * lane);
    }
    if constexpr (kQ8) {
      to.k_scale = dev::LoadBuf1<0>(rows(view.k_scale, 4), 4u * n);
      to.v_scale = dev::LoadBuf1<0>(rows(view.v_scale, 4), 4u * n);
    }
  };
  const auto store = [&](Loaded& from, Stage<D, kQ8>& st) {
    if (!from.got) {  // positions behind the last: weights of 0 times values of 0
#pragma unroll
      for (int i = 0; i < kLoads; ++i) from.k[i] = from.v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      from.k_scale = from.v_scale = 0.0f;
    }
    const int own = Afresh(lane);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = (64 * i + own) / kSourcePieces, p = (64 * i + own) % kSourcePieces;
      char* const k = st.k + (16 * wave + r) * kRow;
      char* const v = st.v + (16 * wave + r) * kRow;
      if constexpr (!kQ8) {
        *reinterpret_cast<float4*>(k + 16 * (p ^ k_swap(r))) = from.k[i];
        *reinterpret_cast<float4*>(v + 16 * (p ^ v_swap(r))) = from.v[i];
      } else {
        const float kw[4] = {from.k[i].x, from.k[i].y, from.k[i].z, from.k[i].w};
        const float vw[4] = {from.v[i].x, from.v[i].y, from.v[i].z, from.v[i].w};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint2 a = CodesToHalves(__float_as_uint(kw[2 * h])), b = CodesToHalves(__float_as_uint(kw[2 * h + 1]));
          *reinterpret_cast<uint4*>(k + 16 * ((2 * p + h) ^ k_swap(r))) = make_uint4(a.x, a.y, b.x, b.y);
          const uint2 c = CodesToHalves(__float_as_uint(vw[2 * h])), d = CodesToHalves(__float_as_uint(vw[2 * h + 1]));
          *reinterpret_cast<uint4*>(v + 16 * ((2 * p + h) ^ v_swap(r))) = make_uint4(c.x, c.y, d.x, d.y);
        }
      }
    }
    if constexpr (kQ8) {
      from.bad |= __any(fabsf(from.k_scale) > kFarScale) ? 2 : 0;
      if (own < 16) {
        st.k_scale[16 * wave + own] = from.k_scale;
        st.v_scale[16 * wave + own] = from.v_scale;
      }
    }
    if (own == 0) st.bad[wave] = from.bad;
  };

  // ---- this wave's columns and part of the keys; its queries are requested before the first keys, which take longer
  const int col_waves = piece.cols > 64 ? 8 : piece.cols > 32 ? 4 : piece.cols > 16 ? 2 : 1;
  const int key_waves = min(kWaves / col_waves, 4);
  const int col_wave = wave % col_waves, key_wave = wave / col_waves;
  const bool works = key_wave < key_waves && col_wave * kWaveCols < piece.cols;
  float to_score, m, l;
  int q_exp;  // 8 bits: the power of two that to_score gives back to queries
  bool rounds = false;  // whether scores are rounded as m is
  float down;  // the power of two that weights enter multiplied by
  F32x4 acc[kE];
  Half8 q_hi[kSteps], q_lo[kSteps];
  int64_t row_head;
  bool there;
  int32_t next_page;
  {
    float4 raw[kSteps][2];
    const int32_t in_tile = col_wave * kWaveCols + n;
    const int32_t col = piece.tile * kCols + in_tile;
    const bool a_column = works && in_tile < piece.cols;
    const int32_t in_group = a_column ? col / args.group : 0, row = piece.first_row + in_group;
    row_head = static_cast<int64_t>(row) * args.n_heads + kh * args.group + (a_column ? col - in_group * args.group : 0);
    const float* qr = args.q + row_head * D;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      raw[s][0] = dev::Load4(qr + (4 * s + g) * 8);
      raw[s][1] = dev::Load4(qr + (4 * s + g) * 8 + 4);
    }
    const AskedRow asked(args, row, a_column);
    load(loaded, c0, page_of(c0));
    next_page = page_of(c0 + 1);
    there = IsOf(groups, row, piece.of, a_column);
    there = asked.BeginsWith(args, piece.pages) && there;
    float x[kSteps][8];
    float top = 0.0f;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float e[4] = {raw[s][i].x, raw[s][i].y, raw[s][i].z, raw[s][i].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          x[s][4 * i + k] = there ? e[k] : 0.0f;
          top = fmaxf(top, fabsf(x[s][4 * i + k]));
        }
      }
    }
    top = MaxAcrossRows(top);
    q_exp = 127;
    if constexpr (kQ8) {  // keys of 8 bits may make scores of queries that 2^127 does not bring to [2^14, 2^15)
      if (__any(top < 0x1p-112f)) {
        const float first = top < 0x1p-112f ? 0x1p40f : 1.0f;
        q_exp = top < 0x1p-112f ? 127 - 40 : 127;
        top *= first;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[s][i] *= first;
        }
      }
    }
    const int e = min(max(268 - (__float_as_int(top) >> 23), 1), 254);  // brings top to [2^14, 2^15)
    const float up = __int_as_float(e << 23);
    q_exp -= e;
    to_score = ldexpf(args.scale_log2, max(q_exp, -140));  // below, scores of scales up to kFarScale count for nothing
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      Terms w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = TermsOf(x[s][2 * i], x[s][2 * i + 1], up);
      q_hi[s] = AsHalf8(w[0].hi, w[1].hi, w[2].hi, w[3].hi);
      q_lo[s] = AsHalf8(w[0].lo, w[1].lo, w[2].lo, w[3].lo);
    }
#pragma unroll
    for (int i = 0; i < kE; ++i) acc[i] = F32x4{0.0f, 0.0f, 0.0f, 0.0f};
    m = -INFINITY;
    l = 0.0f;
    down = kQ8 ? 0x1p126f : 0x1p14f;
  }

  // ---- two tiles of 16 keys, from tile `from` of a step, against 16 columns
  const uint32_t k_lane = static_cast<uint32_t>(n * kRow + 16 * (g ^ k_swap(n)));
  const uint32_t v_lane = static_cast<uint32_t>((4 * g + (n >> 2)) * kRow + 16 * (((n & 3) >> 1) ^ v_swap(4 * g + (n >> 2))) + 8 * (n & 1));
  const auto attend = [&](const Stage<D, kQ8>& st, uint32_t c, int from) {
    const int valid = min(kTiles, (positions - static_cast<int32_t>(c * kStep)) / 16) - from;
    if (valid <= 0) return;
    const uint32_t k_at = Afresh(k_lane), v_at = Afresh(v_lane);
    // All that the products read is requested ahead of them: left to itself, the compiler saves registers by reading each
    // operand just before its product, and waits for every one.
    Half8 k[2][kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
#pragma unroll
      for (int j = 0; j < 2; ++j) k[j][i] = *reinterpret_cast<const Half8*>(st.k + (from + j) * 16 * kRow + (k_at ^ (64u * i)));
    }
    const uint32_t bads[2] = {st.bad[from], st.bad[from + 1]};
    float4 ks[2], vs[2];
    if constexpr (kQ8) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        ks[j] = *reinterpret_cast<const float4*>(st.k_scale + 16 * (from + j) + 4 * g);
        vs[j] = *reinterpret_cast<const float4*>(st.v_scale + 16 * (from + j) + 4 * g);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    F32x4 s[2] = {};
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
#pragma unroll
      for (int j = 0; j < 2; ++j) s[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[j][i], q_hi[i], s[j], 0, 0, 0);
#pragma unroll
      for (int j = 0; j < 2; ++j) s[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[j][i], q_lo[i], s[j], 0, 0, 0);
    }
    uint2 v[kE][2];
#pragma unroll
    for (int i = 0; i < kE; ++i) {
      const char* at = st.v + from * 16 * kRow + (v_at ^ (32u * i));
      v[i][0] = ReadHalvesAcross(at);
      v[i][1] = ReadHalvesAcross(at + 16 * kRow);
    }
    __builtin_amdgcn_sched_barrier(0);
    const uint32_t bad = Scalar(bads[0] | bads[1] << 2);
    float by = to_score;  // what makes scores of s
    if (__builtin_expect(valid < 2 || bad != 0, 0)) {
      if constexpr (kQ8) {
        if (bad & 10) {  // small queries' power of two goes to the scales
          const int first = min(q_exp, 0);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            ks[j] = make_float4(ldexpf(ks[j].x, first), ldexpf(ks[j].y, first), ldexpf(ks[j].z, first), ldexpf(ks[j].w, first));
          }
          by = ldexpf(args.scale_log2, q_exp - first);
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (bad >> (2 * j) & 1) s[j] = F32x4{NAN, NAN, NAN, NAN};
        if (j >= valid) {
          s[j] = F32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          if constexpr (kQ8) ks[j] = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
        }
      }
    }
    if constexpr (kQ8) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float scales[4] = {ks[j].x, ks[j].y, ks[j].z, ks[j].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) s[j][i] *= scales[i];
      }
    }
    // Weights are relative to a maximum that moves only where a score exceeds it by 4 (a factor of 16), over fp16 values by
    // 1: there they enter multiplied by 2^14, with the factor half of fp16's largest, and the low end loses less than 2^-38.
    constexpr float kLag = kQ8 ? 4.0f : 1.0f;
    uint32_t w[2][4];
    float top = s[0][0];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, s[j][i]);
    }
    top = MaxAcrossRows(top) * by;
    const bool moves = __any(top - m > kLag);
    float rise = 0.0f;  // of m, with its sign turned
    if (moves) {
      const float to = top - m > kLag ? top : m;
      rise = m - (to == -INFINITY ? 0.0f : to);
      const float back = __builtin_amdgcn_exp2f(rise);
      m = to;
      l *= back;
      if constexpr (!kQ8) {
#pragma unroll
        for (int i = 0; i < kE; ++i) acc[i] *= back;
      }
      rounds = __any(fabsf(m) >= 0x1p22f);
    }
    // m is a score as rounded. From 2^22 on, where the rounding is half an octave and more, the others are rounded too: not
    // rounded, their weights could pass what they have room for.
    if (__builtin_expect(rounds, 0)) {
#pragma unroll
      for (int j = 0; j < 2; ++j) s[j] *= by;
      by = 1.0f;
    }
    const float less = m == -INFINITY ? 0.0f : m;
    float p[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[j][i] = __builtin_amdgcn_exp2f(fmaf(s[j][i], by, -less));
        l += p[j][i];
      }
    }
    if constexpr (kQ8) {
      // Weights times scales, brought to fp16's range by a power of two that rises with m and falls where they pass it, so
      // that the largest yet, by what it counts for now, enters as 2^12 to 2^15. The two terms end at 2^-24: each is off by
      // at most 2^-37 of that largest.
      float big = 0.0f;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float by[4] = {vs[j].x, vs[j].y, vs[j].z, vs[j].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[j][i] *= by[i];
          big = fmaxf(big, fabsf(p[j][i]));
        }
      }
      big = MaxAcrossRows(big);
      if (moves || __any(big * down > 0x1p15f)) {
        const int from = static_cast<int>(__float_as_uint(down) >> 23);
        int to = min(from + static_cast<int>(fminf(-rise, 300.0f)), 253);
        if (ldexpf(big, to - 127) > 0x1p15f) to = max(266 - static_cast<int>(__float_as_uint(big) >> 23), 1);  // to [2^12, 2^13)
        const float back = __builtin_amdgcn_exp2f(rise + static_cast<float>(to - from));
        down = __int_as_float(to << 23);
#pragma unroll
        for (int i = 0; i < kE; ++i) acc[i] *= back;
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const Terms a = TermsOf(p[j][0], p[j][1], down), b = TermsOf(p[j][2], p[j][3], down);
      w[0][2 * j] = a.hi;
      w[0][2 * j + 1] = b.hi;
      w[1][2 * j] = a.lo;
      w[1][2 * j + 1] = b.lo;
    }
#pragma unroll
    for (int i = 0; i < kE; ++i) {
#pragma unroll
      for (int term = 0; term < 2; ++term) {
        const Half8 p = AsHalf8(w[term][0], w[term][1], w[term][2], w[term][3]);
        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(AsHalf8(v[i][0].x, v[i][0].y, v[i][1].x, v[i][1].y), p, acc[i], 0, 0, 0);
      }
    }
  };

  // ---- the steps: one being attended to in one stage, the next on its way into the other
  store(loaded, stages[0]);
  __syncthreads();
  const int each = kTiles / key_waves;
#pragma unroll 1
  for (uint32_t c = c0; c < c1; ++c) {
    load(loaded, c + 1, next_page);
    next_page = page_of(c + 2);
    if (works) {
#pragma unroll 1
      for (int from = key_wave * each; from < (key_wave + 1) * each; from += 2) attend(stages[(c - c0) & 1], c, from);
    }
    if (c + 1 < c1) store(loaded, stages[(c + 1 - c0) & 1]);
    __syncthreads();
  }

  // ---- the waves' parts of a column joined, in order
  const bool whole = c0 == 0 && c1 == piece.steps;
  float* const joins = reinterpret_cast<float*>(stages);  // [key wave - 1][column]
  const auto join_at = [&](int from) {
    return joins + ((from - 1) * (col_waves * kWaveCols) + col_wave * kWaveCols + n) * kPart;
  };
  l = SumAcrossRows(l);
  const float by = 1.0f / down;
#pragma unroll
  for (int i = 0; i < kE; ++i) acc[i] *= by;
  if (works && key_wave > 0) {
    float* to = join_at(key_wave);
#pragma unroll
    for (int i = 0; i < kE; ++i) *reinterpret_cast<F32x4*>(to + 16 * i + 4 * g) = acc[i];
    if (g == 0) {
      to[D] = m;
      to[D + 1] = l;
    }
  }
  __syncthreads();
  const __amdgpu_buffer_rsrc_t rs = dev::OutResource(args.workspace, 2 * kGroups * SlotBytes(D));
  const uint32_t my_slot = (2 * me + (piece.leads ? 0 : 1)) * SlotBytes(D);
  if (works && key_wave == 0) {
    Own own{};
    float4 own_o[kE];
    if (whole && there) {  // requested before the join
      own = OwnOf(args, row_head);
#pragma unroll
      for (int i = 0; i < kE; ++i) own_o[i] = dev::Load4(args.out + row_head * D + 16 * i + 4 * g);
    } else {
#pragma unroll
      for (int i = 0; i < kE; ++i) own_o[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
#pragma unroll 1
    for (int k = 1; k < key_waves; ++k) {
      const float* from = join_at(k);
      const float m2 = from[D], l2 = from[D + 1];
      const float to = fmaxf(m, m2);
      const float safe = to == -INFINITY ? 0.0f : to;
      const float f = __builtin_amdgcn_exp2f(m - safe), f2 = __builtin_amdgcn_exp2f(m2 - safe);
      m = to;
      l = fmaf(l2, f2, l * f);
#pragma unroll
      for (int i = 0; i < kE; ++i) {
        const F32x4 x = *reinterpret_cast<const F32x4*>(from + 16 * i + 4 * g);
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][r] = fmaf(x[r], f2, acc[i][r] * f);
      }
    }
    if (whole && there) {
      const Both both(own, m, l);
#pragma unroll
      for (int i = 0; i < kE; ++i) {
        dev::Store4(args.out + row_head * D + 16 * i + 4 * g,
                    both.Of(own_o[i], make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3])));
      }
    } else if (there) {
      const int32_t in_tile = col_wave * kWaveCols + n;
#pragma unroll
      for (int i = 0; i < kE; ++i) {
        dev::StoreBuf4<0>(rs, my_slot + 4u * (in_tile * D + 16 * i + 4 * g),
                          make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]));
      }
      if (g == 0) {
        dev::StoreBufU2<0>(rs, my_slot + 4u * kCols * D + 8u * in_tile,
                           make_uint2(__float_as_uint(m), __float_as_uint(l)));
      }
    }
  }
}

template <int D, bool kQ8>
__global__ __launch_bounds__(kThreads, 2) void SharedPrefixKernel(const PrefixArgs args) {
  __shared__ Stage<D, kQ8> stages[2];
  const PagedView& view = args.view;
  const int lane = threadIdx.x & 63;

  const Units units(args, lane);
  const uint32_t sharers = units.sharers;
  if (sharers == 0) return;
  const Share share(units.all, sharers);
  // Workgroups are dealt out to the eight dies in turn: with all of them at work those of one die take neighbouring shares,
  // whose tiles read the same keys and values through its cache.
  const uint32_t me = sharers == kGroups ? (blockIdx.x % 8) * (kGroups / 8) + blockIdx.x / 8 : blockIdx.x;
  if (me >= sharers) return;
  const uint32_t begin = share.Begin(me), end = share.Begin(me + 1);
  uint32_t u = begin;
#pragma unroll 1
  while (u < end) {
    Piece piece;
    const int of = static_cast<int>(__builtin_popcountll(__ballot(units.upto <= u)));
    const uint32_t before = __builtin_amdgcn_readlane(units.upto - units.amount, of);
    const uint32_t tiles = __builtin_amdgcn_readlane(units.tiles, of), cols = __builtin_amdgcn_readlane(units.cols, of);
    piece.of = of;
    piece.steps = __builtin_amdgcn_readlane(units.steps, of);
    piece.first_row = __builtin_amdgcn_readlane(units.groups.first, of);
    piece.last_row = __builtin_amdgcn_readlane(units.groups.last, of);
    piece.pages = __builtin_amdgcn_readlane(units.groups.pages, of);
    piece.positions = static_cast<int32_t>(Units::PositionsOf(args, piece.pages));
    const uint32_t pair = Scalar((u - before) / piece.steps);
    piece.first_unit = before + pair * piece.steps;
    piece.c0 = u - piece.first_unit;
    piece.c1 = min(piece.steps, piece.c0 + (end - u));
    piece.kv_head = static_cast<int32_t>(Scalar(pair / tiles));
    piece.tile = static_cast<int32_t>(pair) - piece.kv_head * static_cast<int32_t>(tiles);
    piece.cols = min(kCols, static_cast<int32_t>(cols) - piece.tile * kCols);
    piece.leads = u == begin;
    u += piece.c1 - piece.c0;

    // the sequence whose table names the group's pages: the first row's that takes part
    int32_t leader = -1;
#pragma unroll 1
    for (int32_t r = piece.first_row; r < piece.last_row && leader < 0; r += 64) {
      const AskedRow asked(args, r + lane, r + lane < piece.last_row);
      const uint64_t good =
          __ballot(IsOf(units.groups, r + lane, of, r + lane < piece.last_row) && asked.BeginsWith(args, piece.pages));
      if (good != 0) leader = __builtin_amdgcn_readlane(asked.seq, __builtin_ctzll(good));
    }
    if (leader < 0) continue;  // the same for every workgroup that has a part of the tile
    const int32_t* table = view.pages + static_cast<int64_t>(leader) * view.max_pages;
    AttendPiece<D, kQ8>(args, units.groups, me, piece, table, stages);
    __syncthreads();  // before the next piece's keys
  }
}

// The parts of tiles that several workgroups have held joined, in order, and with the rows' own part: four elements of a
// column to a thread.
template <int D>
__global__ __launch_bounds__(kJoinThreads) void SharedJoinKernel(const PrefixArgs args) {
  constexpr int kLanes = D / 4;  // of a column
  constexpr int kBatch = 16;     // parts under way
  const int lane = threadIdx.x & 63;
  const int64_t row_head = static_cast<int64_t>(blockIdx.x) * (kJoinThreads / kLanes) + threadIdx.x / kLanes;
  const int32_t d = 4 * (threadIdx.x % kLanes);
  const int32_t row = static_cast<int32_t>(row_head / args.n_heads), head = static_cast<int32_t>(row_head % args.n_heads);
  const bool there = row < args.n_rows;
  const AskedRow asked(args, row, there);
  Own own{};
  float4 own_o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float* const to = args.out + row_head * D + d;
  if (there) {
    own = OwnOf(args, row_head);
    own_o = dev::Load4(to);
  }
  const Units units(args, lane);
  if (units.sharers == 0) return;
  const int32_t in = units.groups.OfLane(there ? row : -1), of = max(in, 0);
  const int32_t pages = __shfl(units.groups.pages, of);
  const bool takes = in >= 0 && asked.BeginsWith(args, pages);
  const uint32_t steps = __shfl(units.steps, of), tiles = __shfl(units.tiles, of);
  const uint32_t before = __shfl(units.upto - units.amount, of);
  const int32_t first_row = __shfl(units.groups.first, of);
  if (!takes) return;

  const int32_t kh = head / args.group, col = (row - first_row) * args.group + (head - kh * args.group);
  const uint32_t tile = static_cast<uint32_t>(col) / kCols, in_tile = static_cast<uint32_t>(col) % kCols;
  const uint32_t first_unit = before + (kh * tiles + tile) * steps;
  const Share share(units.all, units.sharers);
  const uint32_t wa = share.HolderOfLane(first_unit);
  const uint32_t parts = share.HolderOfLane(first_unit + steps - 1) - wa + 1;
  if (parts == 1) return;  // joined where it was made
  const uint32_t first_slot = 2 * wa + (share.Begin(wa) == first_unit ? 0 : 1);
  const __amdgpu_buffer_rsrc_t rs = dev::OutResource(args.workspace, 2 * kGroups * SlotBytes(D));
  float top = -INFINITY, sum = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
  for (uint32_t p = 0; p < parts; p += kBatch) {
    uint2 ml[kBatch];
    float4 x[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const uint32_t part = min(p + k, parts - 1);  // the last once more behind the last, for nothing
      const uint32_t from = (part == 0 ? first_slot : 2 * (wa + part)) * SlotBytes(D);
      ml[k] = dev::LoadBufU2<0>(rs, from + 4u * kCols * D + 8u * in_tile);
      x[k] = dev::LoadBuf4<0>(rs, from + 4u * (in_tile * D + d));
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (p + k < parts) {
        const float m2 = __uint_as_float(ml[k].x), most = fmaxf(top, m2);
        const float safe = most == -INFINITY ? 0.0f : most;
        const float f = __builtin_amdgcn_exp2f(top - safe), f2 = __builtin_amdgcn_exp2f(m2 - safe);
        top = most;
        sum = fmaf(__uint_as_float(ml[k].y), f2, sum * f);
        o = make_float4(fmaf(x[k].x, f2, o.x * f), fmaf(x[k].y, f2, o.y * f), fmaf(x[k].z, f2, o.z * f),
                        fmaf(x[k].w, f2, o.w * f));
      }
    }
  }
  dev::Store4(to, Both(own, top, sum).Of(own_o, o));
}

// The bytes of keys and values from which on it pays to share them, 144 MB and one more for each row. Three kernels instead
// of one cost some 15 us, and 10 more for many rows, whose queries and outputs pass through two of them; the kernel of single
// rows reads what neighbours have just read at some 6 TB/s. Shared against by themselves, us, at 96 / 128 / 160 / 192 / 256 MB
// saved: 16 query and 8 kv heads of 128, fp16, 4 rows 27:30 32:36 33:42 31:48 38:60, 16 rows 23:18 25:29 25:28 26:32 28:44,
// 64 rows 28:16 29:26 30:28 30:31 30:35, 128 rows 36:26 36:29 37:32 37:34 37:40; 32 and 8 heads in 8 bits, 4 rows 31:24 37:41
// 39:44 39:52 46:67, 16 rows 28:20 32:28 33:28 34:35 35:46, 64 rows 31:18 32:27 32:29 33:31 34:34; 32 and 4 heads of 64,
// fp16, 8 rows 32:19 32:34 32:34 33:43 38:54, 32 rows 25:17 29:24 30:24 32:29 32:37. One line in rows for all of these:
// it takes the slower side for 4 rows at 96 (fp16) and 128, for 16 at 128 (fp16) and 160 (8 bits), for heads of 64 at 128 (8
// rows) and 192 (32 rows), and for 64 and 128 rows where both are alike, by 3 to 18%. Rows are counted without their
// lengths: those of a batch that stand idle save nothing, but count.
int64_t LeastSaving(int64_t n_rows) { return (144 + n_rows) << 20; }

int64_t JoinGroups(int64_t n_rows, int32_t n_heads, int32_t head_dim) {
  return (n_rows * n_heads * (head_dim / 4) + kJoinThreads - 1) / kJoinThreads;
}

size_t MlBytes(int32_t n_heads, int64_t n_rows) {
  return (static_cast<size_t>(n_rows) * n_heads * 8 + 255) / 256 * 256;
}
size_t PrefixBytes(int32_t n_heads, int32_t head_dim, int64_t n_rows) {
  return 2 * kGroups * static_cast<size_t>(SlotBytes(head_dim)) + MlBytes(n_heads, n_rows);
}

}  // namespace

void CheckPrefix(const GpuPagedKv& kv, const GpuPageTable& table, int32_t n_heads, int64_t n_rows, char* workspace,
                 PagedPrefix* prefix) {
  const int64_t capacity = std::min<int64_t>(table.max_pages * kv.page_size, 0x7FFFFFFF);
  const int64_t group = n_heads / kv.n_kv_heads;
  const int64_t most = ((n_rows * group + kCols - 1) / kCols) * kv.n_kv_heads * (capacity / kStep + 1);
  RPG_CHECK(n_rows * group <= 0x7FFFFFFF && most <= 0x7FFFFFFF / std::max(prefix->n_groups, 1),
            "AttentionPagedShared: %d groups of %lld rows of up to %lld positions are too many for one call",
            prefix->n_groups, static_cast<long long>(n_rows), static_cast<long long>(capacity));
  RPG_CHECK(FitsLaunch(JoinGroups(n_rows, n_heads, kv.head_dim), kJoinThreads),
            "AttentionPagedShared: %lld rows of %d heads are too many for one call", static_cast<long long>(n_rows), n_heads);
  // slots, (m, l)
  prefix->workspace = workspace;
  prefix->ml = reinterpret_cast<float*>(workspace + 2 * kGroups * static_cast<size_t>(SlotBytes(kv.head_dim)));
}

void AttendPrefix(const GpuPagedKv& kv, const GpuPageTable& table, const int32_t* seq_ids, const int32_t* lens,
                  const float* q_dev, int32_t n_heads, int64_t n_rows, float* out_dev, const PagedPrefix& prefix) {
  const float scale_log2 = static_cast<float>(1.4426950408889634 / std::sqrt(static_cast<double>(kv.head_dim)));
  const bool q8 = kv.type == kKvQ8;
  auto* kern = kv.head_dim == 128 ? (q8 ? SharedPrefixKernel<128, true> : SharedPrefixKernel<128, false>)
                                  : (q8 ? SharedPrefixKernel<64, true> : SharedPrefixKernel<64, false>);
  const PrefixArgs args{dev::ViewOf(kv, table), prefix, seq_ids, lens, q_dev, out_dev, prefix.workspace,
                        static_cast<int32_t>(n_rows),
                        static_cast<int32_t>(std::min<int64_t>(table.max_pages * kv.page_size, 0x7FFFFFFF)), n_heads,
                        n_heads / kv.n_kv_heads, scale_log2};
  Launch("SharedPrefixKernel", kern, dim3(kGroups), dim3(kThreads), args);
  Launch("SharedJoinKernel", kv.head_dim == 128 ? SharedJoinKernel<128> : SharedJoinKernel<64>,
         dim3(static_cast<uint32_t>(JoinGroups(n_rows, n_heads, kv.head_dim))), dim3(kJoinThreads), args);
}

size_t GpuAttentionPagedSharedWorkspaceBytes(int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, int64_t n_rows) {
  const size_t own = GpuAttentionPagedWorkspaceBytes(n_heads, n_kv_heads, head_dim);
  RPG_CHECK(n_rows >= 0 && n_rows <= 0x7FFFFFFF / n_heads, "AttentionPagedSharedWorkspace: %lld rows of %d heads",
            static_cast<long long>(n_rows), n_heads);
  return own + PrefixBytes(n_heads, head_dim, n_rows);
}

void GpuAttentionPagedShared(const GpuPagedKv& kv, const GpuPageTable& table, const int32_t* seq_ids,
                             const int32_t* lens, const int32_t* group_rows, const int32_t* group_pages,
                             int32_t n_groups, const float* q_dev, int32_t n_heads, int64_t n_rows, float* out_dev,
                             void* workspace, size_t workspace_bytes, int64_t least_saving) {
  RPG_CHECK(n_groups >= 0 && n_groups <= dev::kMaxSharedGroups, "AttentionPagedShared: %d groups, at most %d", n_groups,
            dev::kMaxSharedGroups);
  RPG_CHECK(n_groups == 0 || (group_rows != nullptr && group_pages != nullptr), "AttentionPagedShared got null groups");
  RPG_CHECK(((reinterpret_cast<uintptr_t>(group_rows) | reinterpret_cast<uintptr_t>(group_pages)) & 3) == 0,
            "AttentionPagedShared: groups have to be 4-byte aligned");
  if (least_saving < 0) least_saving = LeastSaving(n_rows);
  const int64_t row = int64_t{kv.type == kKvQ8 ? kv.head_dim + 4 : 2 * kv.head_dim} * 2;  // a position's of a kv head
  const int64_t page = std::max<int64_t>(row * std::max(kv.page_size, 1) * std::max(kv.n_kv_heads, 1), 1);
  const int64_t least = least_saving / page + (least_saving % page != 0 ? 1 : 0);
  PagedPrefix prefix{group_rows, group_pages, n_groups, std::min(least, kMostSaving)};
  AttendPaged(kv, table, seq_ids, lens, q_dev, n_heads, n_rows, out_dev, workspace, workspace_bytes, &prefix);
}

}  // namespace rpg
