// Attention of one new token per row over the paged KV cache.
//
// For row r, query head h of kv head h / G, over the positions j < lens[r]:
//   s_j = (q . k_j) / sqrt(D),  out = sum_j exp(s_j - max s) v_j / sum_j exp(s_j - max s)
// in one pass over the cache, with the running maximum m and sum l: on a new
// maximum the sum and the accumulated output are scaled by exp(m_old - m_new).
// Exponentials are taken as powers of two, with log2(e) in the scores' scale.
//
// What bounds it: the cache is read once, 2 D (+ 4) bytes of keys and values a
// position and kv head, and 4 D G operations are done on them. Vector arithmetic
// would take G multiply-adds an element beside its conversion, too much from G = 8
// on for 8-bit rows (39e12 lane operations a second against some 6e12 bytes), so
// both products run on the matrix cores, where the G query heads of a kv head are
// columns of one 16-column tile.
//
// Products (16x16x32, fp16 operands, fp32 sums). Keys and values enter as they are
// kept: halves, or codes, which are exact in fp16. Queries and weights are fp32 and
// enter as two fp16 terms of 11 bits, hi + lo, in columns n and n + 8 of the same
// tile, which a tile of at most 8 heads leaves free: 22 bits for no further matrix
// instruction. A query row is first scaled by a power of two to a largest magnitude
// in [2^14, 2^15), weights by 2^14 (8-bit values: with their row's scale, relative
// to a power of two above the largest scale so far), so that what is lost at fp16's
// low end is below 2^-38 of the largest. hi is cut off from slightly below the
// value, so that both terms have its sign and neither is zero: infinities in the
// cache then give what the one product would (weights below 2^-23 of the largest
// excepted, which may turn an infinite value into NaN).
//   S = K Q^T: rows are 16 keys (a lane loads 16 contiguous bytes of a key's row),
//     columns heads; a lane ends with 4 keys of one column.
//   O^T = V^T P^T: rows are D / 16 sets of 16 elements, the sum runs over 32 keys.
//     Which of them a lane group holds is free, so it holds those whose weights it
//     has from S, and loads their rows D / 16 contiguous elements wide; the
//     transposition is byte permutes within the lane.
//
// Sharing out: work is counted in units of 64 positions of one (row, kv head, tile
// of up to 8 heads). Every wave adds up the rows' units by itself from lens and
// takes an equal, contiguous share of them, so that ragged batches and single long
// rows fill the card alike and nothing about the lengths is needed on the host. A
// wave writes what it holds whole; where a (row, tile) is split over waves of one
// workgroup they join in LDS, and where it is split over workgroups each leaves its
// part in the workspace and the last to arrive joins them, in order.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "dev_util.h"
#include "kernels_gpu.h"
#include "launch.h"
#include "paged_kv.h"

namespace rpg {
namespace {

using dev::PagedView;

constexpr int kWaves = 4;
constexpr int kUnitShift = 6;  // 64 positions to a unit
constexpr int kTileHeads = 8;
// Workgroups at most; a workspace has two part slots and a counter for each.
constexpr int kMaxGroups = 768;
// Bytes between two counters: on lines of their own, as the decode attention's.
constexpr size_t kCounterBytes = 256;

using Half2 = _Float16 __attribute__((ext_vector_type(2)));
using Half8 = _Float16 __attribute__((ext_vector_type(8)));
using F32x4 = float __attribute__((ext_vector_type(4)));

constexpr int PartFloats(int d) { return d + 4; }  // o[d], m, l, and two to keep rows 16-byte aligned

// ---------------------------------------------------------------- lane exchange

// x of the lane 8 further on in its row of 16.
__device__ __forceinline__ float Ror8(float x) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x128, 0xF, 0xF, false));
}

// f over the four lanes l, l ^ 16, l ^ 32, l ^ 48; every one of them has the result.
template <class F>
__device__ __forceinline__ float AcrossRows(float x, F f) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_int(x), __float_as_int(x), false, false);
  x = f(__int_as_float(a[0]), __int_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false, false);
  return f(__int_as_float(b[0]), __int_as_float(b[1]));
}
__device__ __forceinline__ float MaxAcrossRows(float x) {
  return AcrossRows(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float SumAcrossRows(float x) {
  return AcrossRows(x, [](float a, float b) { return a + b; });
}

// ---------------------------------------------------------------- conversions

__device__ __forceinline__ uint32_t Bits(Half2 h) { return __builtin_bit_cast(uint32_t, h); }

// The hi (want_lo false) or lo terms of two values, packed.
__device__ __forceinline__ uint32_t Term2(float a, float b, bool want_lo) {
  const auto below = [](float x) {
    const int u = __float_as_int(x);
    const int mag = max((u & 0x7FFFFFFF) - 0x100, 0);
    return __int_as_float((u & static_cast<int>(0x80000000u)) | mag);
  };
  const auto hi = __builtin_amdgcn_cvt_pkrtz(below(a), below(b));
  const Half2 lo = {static_cast<_Float16>(a - static_cast<float>(hi[0])),
                    static_cast<_Float16>(b - static_cast<float>(hi[1]))};
  return want_lo ? Bits(lo) : __builtin_bit_cast(uint32_t, hi);
}

__device__ __forceinline__ Half8 AsHalf8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  const dev::U32x4 w = {a, b, c, d};
  return __builtin_bit_cast(Half8, w);
}

// Two codes (bytes 2 i, 2 i + 1 of w, sign bit flipped) as halves: 1024 + u, less 1152.
template <int kI>
__device__ __forceinline__ uint32_t CodePair(uint32_t flipped) {
  const uint32_t x = __builtin_amdgcn_perm(0x64646464u, flipped, kI == 0 ? 0x04010400u : 0x04030402u);
  const Half2 bias = {static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
  return Bits(__builtin_bit_cast(Half2, x) - bias);
}

// Byte kI of two words (sign bit flipped) as halves, times 2^-9: as a subnormal the
// byte u stands for u 2^-24, and u 2^-9 - 2^-2 = (u - 128) 2^-9 is one exact fma.
template <int kI>
__device__ __forceinline__ uint32_t CodeOfTwo(uint32_t w0, uint32_t w1) {
  const uint32_t x = __builtin_amdgcn_perm(w1, w0, 0x0C000C00u | kI | ((4 + kI) << 16));
  const Half2 up = {static_cast<_Float16>(32768.0f), static_cast<_Float16>(32768.0f)};
  const Half2 off = {static_cast<_Float16>(-0.25f), static_cast<_Float16>(-0.25f)};
  return Bits(__builtin_elementwise_fma(__builtin_bit_cast(Half2, x), up, off));
}

// ---------------------------------------------------------------- sharing out

// Everything here is the same in every lane of a wave.
struct Share {
  int64_t total;  // units
  int64_t per;    // a workgroup's units: per, and one more in the first `rem` of them
  int64_t rem;
  int32_t groups;

  __device__ __forceinline__ int64_t Begin(int64_t w) const { return w * per + (w < rem ? w : rem); }
  // The workgroup whose share holds unit x.
  __device__ __forceinline__ int64_t Holder(int64_t x) const {
    const int64_t big = rem * (per + 1);
    if ((total >> 32) == 0) {
      return x < big ? static_cast<uint32_t>(x) / static_cast<uint32_t>(per + 1)
                     : rem + static_cast<uint32_t>(x - big) / static_cast<uint32_t>(per);
    }
    return x < big ? x / (per + 1) : rem + (x - big) / per;
  }
};

struct Rows {
  const int32_t* seq_ids;
  const int32_t* lens;
  int64_t n_seqs;
  int64_t capacity;  // positions that a table row has pages for
  int32_t n_rows;
  int32_t pairs;  // (kv head, tile) pairs of a row

  __device__ __forceinline__ int64_t Seq(int32_t r) const { return seq_ids != nullptr ? seq_ids[r] : r; }
  __device__ __forceinline__ bool Fine(int64_t seq, int32_t len) const {
    return seq >= 0 && seq < n_seqs && len >= 0 && len <= capacity;
  }
  // Units of one pair of row r; none for a row that is padding, empty or out of range.
  __device__ __forceinline__ int32_t UnitsOf(int32_t r) const {
    const int32_t len = lens[r];
    return Fine(Seq(r), len) ? static_cast<int32_t>((static_cast<int64_t>(len) + 63) >> kUnitShift) : 0;
  }
};

// Units of rows [lo, hi), taken `each` to a lane: what lies before this lane's rows.
__device__ __forceinline__ int64_t UnitsBefore(const Rows& rows, int32_t lo, int32_t hi, int32_t each, int lane,
                                               int64_t* total) {
  int64_t own = 0;
  const int64_t first = lo + static_cast<int64_t>(lane) * each;
  for (int32_t i = 0; i < each; ++i) {
    if (first + i < hi) own += rows.UnitsOf(static_cast<int32_t>(first + i));
  }
  own *= rows.pairs;
  int64_t sum = own;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int64_t up = __shfl_up(sum, off, 64);
    if (lane >= off) sum += up;
  }
  *total = __shfl(sum, 63, 64);
  return sum - own;
}

__device__ __forceinline__ int64_t Uniform(int64_t x) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(x));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(x >> 32));
  return static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
}

// Row that holds unit x, and what of x lies in it (*rest), from the units before
// each lane's `each` rows of [lo, hi).
__device__ __forceinline__ int32_t RowOfUnit(const Rows& rows, int64_t before, int32_t each, int lane, int64_t x,
                                             int64_t* rest) {
  int32_t lo = 0, hi = rows.n_rows;
  while (true) {
    // before does not fall from lane to lane, and the last one at or below x is not of an empty set of rows
    const int at = static_cast<int>(__builtin_popcountll(__ballot(before <= x))) - 1;
    x -= Uniform(__shfl(before, at, 64));
    const int64_t begin = lo + static_cast<int64_t>(at) * each;
    hi = static_cast<int32_t>(min(begin + each, static_cast<int64_t>(hi)));
    lo = static_cast<int32_t>(begin);
    if (each == 1) break;
    each = (hi - lo + 63) / 64;
    int64_t unused;
    before = UnitsBefore(rows, lo, hi, each, lane, &unused);
  }
  *rest = x;
  return lo;
}

// ---------------------------------------------------------------- the kernel

// What a wave or workgroup holds of a (row, pair): its units [c0, c1) of n.
struct Piece {
  int64_t first;  // number of the pair's first unit
  int32_t row, pair, c0, c1, n;
};

// In scalar registers: a buffer descriptor made from vector ones would be looped over.
__device__ __forceinline__ Piece UniformPiece(const Piece& p) {
  return Piece{Uniform(p.first),
               __builtin_amdgcn_readfirstlane(p.row),
               __builtin_amdgcn_readfirstlane(p.pair),
               __builtin_amdgcn_readfirstlane(p.c0),
               __builtin_amdgcn_readfirstlane(p.c1),
               __builtin_amdgcn_readfirstlane(p.n)};
}

template <int D, bool kQ8>
__global__ __launch_bounds__(64 * kWaves) void PagedAttentionKernel(PagedView view, Rows rows,
                                                                    const float* __restrict__ q, int32_t n_heads,
                                                                    int32_t tiles, int32_t tile_heads, float scale_log2,
                                                                    float* __restrict__ out,
                                                                    char* __restrict__ workspace) {
  constexpr int kBytes = kQ8 ? 1 : 2;
  constexpr int kSub = D == 128 && !kQ8 ? 2 : 4;  // 16-key tiles of a step: 32 registers of keys at most
  constexpr int kStep = 16 * kSub;
  constexpr int kRow = D * kBytes;        // bytes of a key's row
  constexpr int kKLoads = kRow / 64;      // 16-byte loads of a lane for 16 keys
  constexpr int kSteps = D / 32;          // matrix products of 16 keys
  constexpr int kE = D / 16;              // elements of a value row to a lane
  constexpr int kVWords = kE * kBytes / 4;
  constexpr int kPart = PartFloats(D);
  static_assert((1 << kUnitShift) % kStep == 0, "a unit is whole steps");

  __shared__ __attribute__((aligned(16))) float part[kWaves][2][kTileHeads][kPart];
  __shared__ Piece pieces[kWaves][2];
  __shared__ int held[kWaves];
  __shared__ int last_flag;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int n = lane & 15;
  const int g = lane >> 4;
  const bool is_lo = n >= 8;
  const int32_t group = n_heads / view.n_kv;

  // the batch's units, and this wave's share
  Share share;
  const int32_t each = (rows.n_rows + 63) / 64;
  const int64_t before = UnitsBefore(rows, 0, rows.n_rows, each, lane, &share.total);
  share.total = Uniform(share.total);
  share.groups = static_cast<int32_t>(min(static_cast<int64_t>(gridDim.x), (share.total + kWaves - 1) / kWaves));
  const int64_t me = blockIdx.x;
  int64_t begin = 0, end = 0;
  if (me < share.groups) {
    if ((share.total >> 32) == 0) {
      const uint32_t t = static_cast<uint32_t>(share.total), w = static_cast<uint32_t>(share.groups);
      share.per = t / w;
      share.rem = t % w;
    } else {
      share.per = share.total / share.groups;
      share.rem = share.total % share.groups;
    }
    begin = share.Begin(me);
    end = share.Begin(me + 1);
  }
  int64_t u = Uniform(begin + (((end - begin) * wave) >> 2));
  const int64_t u_end = Uniform(begin + (((end - begin) * (wave + 1)) >> 2));
  static_assert(kWaves == 4, "a wave's share of its workgroup's");

  int my_held = 0;
  if (u < u_end) {
    int64_t rest;
    int32_t row = __builtin_amdgcn_readfirstlane(RowOfUnit(rows, before, each, lane, u, &rest));
    rest = Uniform(rest);
    int32_t units = __builtin_amdgcn_readfirstlane(rows.UnitsOf(row));
    int32_t pair = 0, c0 = 0;
    if ((rest >> 32) == 0) {
      pair = static_cast<int32_t>(static_cast<uint32_t>(rest) / static_cast<uint32_t>(units));
      c0 = static_cast<int32_t>(static_cast<uint32_t>(rest) % static_cast<uint32_t>(units));
    } else {
      pair = static_cast<int32_t>(rest / units);
      c0 = static_cast<int32_t>(rest % units);
    }
    while (true) {
      const int32_t c1 = static_cast<int32_t>(min(static_cast<int64_t>(units), c0 + (u_end - u)));
      const int64_t seq = rows.Seq(row);
      const int32_t len = rows.lens[row];
      const int32_t* table = view.pages + seq * view.max_pages;
      const int32_t kh = pair / tiles;
      const int32_t h0 = (pair - kh * tiles) * tile_heads;
      const int32_t heads = min(tile_heads, group - h0);
      const int64_t head_row = static_cast<int64_t>(row) * n_heads + kh * group + h0;

      // rows of the pool that the 16-key tiles of a step start at; a tile past the end repeats the step's first, a
      // page out of range is read as page 0 and its tile marked in *bad
      auto find = [&](int32_t pos, int64_t (&at)[kSub]) {
        int bad = 0;
#pragma unroll
        for (int j = 0; j < kSub; ++j) {
          const int32_t p = pos + 16 * j < len ? pos + 16 * j : pos;
          int32_t page = table[p >> view.page_shift];
          if (page < 0 || page >= view.n_pages) {
            page = 0;
            bad |= 1 << j;
          }
          at[j] = ((static_cast<int64_t>(page) * view.n_kv + kh) << view.page_shift) +
                  (p & ((1 << view.page_shift) - 1));
        }
        return bad;
      };
      uint4 kw[kSub][kKLoads];
      const uint32_t k_lane = static_cast<uint32_t>(n * kRow + 16 * g);
      auto load_k = [&](const int64_t (&at)[kSub]) {
#pragma unroll
        for (int j = 0; j < kSub; ++j) {
          const char* p = static_cast<const char*>(view.k) + at[j] * kRow;
#pragma unroll
          for (int i = 0; i < kKLoads; ++i) kw[j][i] = *reinterpret_cast<const uint4*>(p + (k_lane + 64u * i));
        }
      };

      int32_t pos = c0 << kUnitShift;
      const int32_t stop = static_cast<int32_t>(min(static_cast<int64_t>(len), static_cast<int64_t>(c1) << kUnitShift));
      int64_t at[kSub];
      int bad = find(pos, at);
      load_k(at);

      // the queries' terms: column n is head n % 8, hi below 8 and lo above
      Half8 qt[kSteps];
      float to_score;
      {
        const bool there = (n & 7) < heads;
        const float* qr = q + (head_row + (there ? n & 7 : 0)) * D;
        float x[kSteps][8];
        float top = 0.0f;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          const int d = kQ8 ? 64 * (s / 2) + 16 * g + 8 * (s & 1) : 32 * s + 8 * g;
          const float4 a = dev::Load4(qr + d), b = dev::Load4(qr + d + 4);
          const float e[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            x[s][i] = there ? e[i] : 0.0f;
            top = fmaxf(top, fabsf(x[s][i]));
          }
        }
        top = MaxAcrossRows(top);
        const int e = min(max(268 - (__float_as_int(top) >> 23), 1), 254);  // biased exponent of 2^14 over top's
        const float up = __int_as_float(e << 23);
        to_score = ldexpf(scale_log2, 127 - e);
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = Term2(x[s][2 * i] * up, x[s][2 * i + 1] * up, is_lo);
          qt[s] = AsHalf8(w[0], w[1], w[2], w[3]);
        }
      }

      float m = -INFINITY, l = 0.0f;
      float ref = 0.0f;  // 8-bit values: what acc's weights are relative to, a power of two above the scales so far
      F32x4 acc[kE];
#pragma unroll
      for (int i = 0; i < kE; ++i) acc[i] = F32x4{0.0f, 0.0f, 0.0f, 0.0f};

      for (; pos < stop; pos += kStep) {
        const bool tail = pos + kStep > len;
        // this step's values and scales
        uint32_t vw[kSub][4][kVWords];
        const uint32_t v_lane = static_cast<uint32_t>(4 * g * kRow + n * kE * kBytes);
#pragma unroll
        for (int j = 0; j < kSub; ++j) {
          const char* p = static_cast<const char*>(view.v) + at[j] * kRow;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const char* a = p + (v_lane + static_cast<uint32_t>(i * kRow));
            if constexpr (kVWords == 4) {
              const uint4 w = *reinterpret_cast<const uint4*>(a);
              vw[j][i][0] = w.x, vw[j][i][1] = w.y, vw[j][i][2] = w.z, vw[j][i][3] = w.w;
            } else if constexpr (kVWords == 2) {
              const uint2 w = *reinterpret_cast<const uint2*>(a);
              vw[j][i][0] = w.x, vw[j][i][1] = w.y;
            } else {
              vw[j][i][0] = *reinterpret_cast<const uint32_t*>(a);
            }
          }
        }
        float4 ks[kQ8 ? kSub : 1], vs[kQ8 ? kSub : 1];
        if constexpr (kQ8) {
#pragma unroll
          for (int j = 0; j < kSub; ++j) {
            ks[j] = dev::Load4(view.k_scale + at[j] + 4 * g);
            vs[j] = dev::Load4(view.v_scale + at[j] + 4 * g);
          }
        }
        // scores
        F32x4 s4[kSub];
#pragma unroll
        for (int j = 0; j < kSub; ++j) {
          s4[j] = F32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int i = 0; i < kKLoads; ++i) {
            const uint4 w = kw[j][i];
            if constexpr (kQ8) {
              const uint32_t f[4] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u, w.z ^ 0x80808080u, w.w ^ 0x80808080u};
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const Half8 a = AsHalf8(CodePair<0>(f[2 * h]), CodePair<1>(f[2 * h]), CodePair<0>(f[2 * h + 1]),
                                        CodePair<1>(f[2 * h + 1]));
                s4[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qt[2 * i + h], s4[j], 0, 0, 0);
              }
            } else {
              s4[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(AsHalf8(w.x, w.y, w.z, w.w), qt[i], s4[j], 0, 0, 0);
            }
          }
        }
        // the next step's keys
        const int this_bad = bad;
        if (pos + kStep < stop) {
          bad = find(pos + kStep, at);
          load_k(at);
        }
        float s[kSub][4];
        float top = m;
#pragma unroll
        for (int j = 0; j < kSub; ++j) {
          const float by[4] = {kQ8 ? ks[kQ8 ? j : 0].x : 0.0f, kQ8 ? ks[kQ8 ? j : 0].y : 0.0f,
                               kQ8 ? ks[kQ8 ? j : 0].z : 0.0f, kQ8 ? ks[kQ8 ? j : 0].w : 0.0f};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float x = (s4[j][i] + Ror8(s4[j][i])) * to_score;
            if constexpr (kQ8) x *= by[i];
            if (this_bad & (1 << j)) x = NAN;
            if (tail && pos + 16 * j + 4 * g + i >= len) x = -INFINITY;
            s[j][i] = x;
            top = fmaxf(top, x);
          }
        }
        top = MaxAcrossRows(top);
        const float safe = top == -INFINITY ? 0.0f : top;
        float back = __builtin_amdgcn_exp2f(m - safe);
        m = top;
        l *= back;
        float up = 0x1p14f;
        if constexpr (kQ8) {
          if (tail) {
#pragma unroll
            for (int j = 0; j < kSub; ++j) {
              const int32_t p = pos + 16 * j + 4 * g;
              vs[j].x = p < len ? vs[j].x : 0.0f;
              vs[j].y = p + 1 < len ? vs[j].y : 0.0f;
              vs[j].z = p + 2 < len ? vs[j].z : 0.0f;
              vs[j].w = p + 3 < len ? vs[j].w : 0.0f;
            }
          }
          float big = 0.0f;
#pragma unroll
          for (int j = 0; j < kSub; ++j) big = fmaxf(big, fmaxf(fmaxf(vs[j].x, vs[j].y), fmaxf(vs[j].z, vs[j].w)));
          big = MaxAcrossRows(big);
          if (big >= ref) {  // the same in every lane
            const int e = min(max((__float_as_int(big) >> 23) + 1, 27), 254);
            const float to = __int_as_float(e << 23);
            back *= ref * __int_as_float((254 - e) << 23);  // ref / to
            ref = to;
          }
          up *= __int_as_float((254 << 23) - __float_as_int(ref));  // 2^14 / ref
        }
        if (__any(back != 1.0f)) {
#pragma unroll
          for (int i = 0; i < kE; ++i) acc[i] *= back;
        }
        // weights: p, and its terms in the order of the lane's keys
        uint32_t pt[kSub][2];
#pragma unroll
        for (int j = 0; j < kSub; ++j) {
          float w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            w[i] = __builtin_amdgcn_exp2f(s[j][i] - safe);
            l += w[i];
          }
          if constexpr (kQ8) {
            w[0] *= vs[j].x, w[1] *= vs[j].y, w[2] *= vs[j].z, w[3] *= vs[j].w;
          }
          pt[j][0] = Term2(w[0] * up, w[1] * up, is_lo);
          pt[j][1] = Term2(w[2] * up, w[3] * up, is_lo);
        }
        if (tail) {  // what stands behind the last position is not even a number
#pragma unroll
          for (int j = 0; j < kSub; ++j) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const bool keep = pos + 16 * j + 4 * g + i < len;
#pragma unroll
              for (int w = 0; w < kVWords; ++w) vw[j][i][w] = keep ? vw[j][i][w] : 0u;
            }
          }
        }
#pragma unroll
        for (int t = 0; t < kSub / 2; ++t) {
          const Half8 b = AsHalf8(pt[2 * t][0], pt[2 * t][1], pt[2 * t + 1][0], pt[2 * t + 1][1]);
          auto& v0 = vw[2 * t];
          auto& v1 = vw[2 * t + 1];
          if constexpr (kQ8) {
#pragma unroll
            for (int w = 0; w < kVWords; ++w) {
              uint32_t f[8];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                f[i] = v0[i][w] ^ 0x80808080u;
                f[4 + i] = v1[i][w] ^ 0x80808080u;
              }
              auto one = [&](auto byte) {
                constexpr int kI = decltype(byte)::value;
                const Half8 a = AsHalf8(CodeOfTwo<kI>(f[0], f[1]), CodeOfTwo<kI>(f[2], f[3]),
                                        CodeOfTwo<kI>(f[4], f[5]), CodeOfTwo<kI>(f[6], f[7]));
                acc[4 * w + kI] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, acc[4 * w + kI], 0, 0, 0);
              };
              one(std::integral_constant<int, 0>{});
              one(std::integral_constant<int, 1>{});
              one(std::integral_constant<int, 2>{});
              one(std::integral_constant<int, 3>{});
            }
          } else {
#pragma unroll
            for (int i = 0; i < kE; ++i) {
              const uint32_t sel = i & 1 ? 0x07060302u : 0x05040100u;
              const int w = i / 2;
              const Half8 a = AsHalf8(__builtin_amdgcn_perm(v0[1][w], v0[0][w], sel),
                                      __builtin_amdgcn_perm(v0[3][w], v0[2][w], sel),
                                      __builtin_amdgcn_perm(v1[1][w], v1[0][w], sel),
                                      __builtin_amdgcn_perm(v1[3][w], v1[2][w], sel));
              acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, acc[i], 0, 0, 0);
            }
          }
        }
      }

      // the piece's (m, l, o): out, or to LDS where it is not the whole of its pair
      const float total = SumAcrossRows(l);
      const bool whole = c0 == 0 && c1 == units;
      const float unit = kQ8 ? ref * 0x1p-5f : 0x1p-14f;
      const float by = whole ? unit / total : unit;
      float* to = whole ? out + (head_row + n) * D : &part[wave][my_held][n & 7][0];
      float o[4][kE];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
#pragma unroll
        for (int i = 0; i < kE; ++i) o[r][i] = (acc[i][r] + Ror8(acc[i][r])) * by;
      }
      if (n < heads) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
#pragma unroll
          for (int i = 0; i < kE; i += 4) {
            *reinterpret_cast<float4*>(to + kE * (4 * g + r) + i) =
                make_float4(o[r][i], o[r][i + 1], o[r][i + 2], o[r][i + 3]);
          }
        }
        if (!whole && g == 0) {
          to[D] = m;
          to[D + 1] = total;
        }
      }
      if (!whole) {
        if (lane == 0) {
          pieces[wave][my_held] = Piece{u - c0, row, pair, c0, c1, units};
        }
        ++my_held;
      }
      u += c1 - c0;
      if (u >= u_end) break;
      c0 = 0;
      if (++pair == rows.pairs) {
        pair = 0;
        do {
          ++row;
          units = row < rows.n_rows ? __builtin_amdgcn_readfirstlane(rows.UnitsOf(row)) : 1;
        } while (units == 0);
        if (row >= rows.n_rows) break;  // only if the lengths change while this runs
      }
    }
  }
  if (lane == 0) held[wave] = my_held;
  __syncthreads();

  // The workgroup's pieces in order, neighbours of one pair joined.
  float* const slots = reinterpret_cast<float*>(workspace + kMaxGroups * kCounterBytes);
  const int64_t slot_floats = static_cast<int64_t>(tile_heads) * kPart;
  int from = 0;  // wave * 2 + which
  while (from < 2 * kWaves) {
    if ((from & 1) >= held[from >> 1]) {
      ++from;
      continue;
    }
    Piece run = UniformPiece(pieces[from >> 1][from & 1]);
    int list = 1 << from;
    int to = from + 1;
    for (; to < 2 * kWaves; ++to) {
      if ((to & 1) >= held[to >> 1]) continue;
      const Piece next = UniformPiece(pieces[to >> 1][to & 1]);
      if (next.first != run.first) break;
      run.c1 = next.c1;
      list |= 1 << to;
    }
    from = to;
    const int32_t kh = run.pair / tiles;
    const int32_t h0 = (run.pair - kh * tiles) * tile_heads;
    const int32_t heads = min(tile_heads, group - h0);
    const int64_t head_row = static_cast<int64_t>(run.row) * n_heads + kh * group + h0;
    const bool whole = run.c0 == 0 && run.c1 == run.n;
    const bool leads = run.first + run.c0 == begin;  // the workgroup's first piece
    float* slot = slots + (2 * me + (leads ? 0 : 1)) * slot_floats;
    const __amdgpu_buffer_rsrc_t rs = dev::OutResource(slot, static_cast<uint32_t>(slot_floats * 4));
    for (int i = threadIdx.x; i < heads * (D / 4); i += 64 * kWaves) {
      const int h = i / (D / 4), d = 4 * (i % (D / 4));
      float top = -INFINITY;
      for (int k = 0; k < 2 * kWaves; ++k) {
        if (list >> k & 1) top = fmaxf(top, part[k >> 1][k & 1][h][D]);
      }
      const float safe = top == -INFINITY ? 0.0f : top;
      float l = 0.0f;
      float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int k = 0; k < 2 * kWaves; ++k) {
        if (!(list >> k & 1)) continue;
        const float* p = part[k >> 1][k & 1][h];
        const float f = __builtin_amdgcn_exp2f(p[D] - safe);
        const float4 x = *reinterpret_cast<const float4*>(p + d);
        l = fmaf(p[D + 1], f, l);
        o = make_float4(fmaf(x.x, f, o.x), fmaf(x.y, f, o.y), fmaf(x.z, f, o.z), fmaf(x.w, f, o.w));
      }
      if (whole) {
        const float inv = 1.0f / l;
        dev::Store4(out + (head_row + h) * D + d, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
      } else {
        dev::StoreBuf4<dev::kStoreDeviceThroughPolicy>(rs, 4u * static_cast<uint32_t>(h * kPart + d), o);
        if (d == 0) {
          dev::StoreBufU2<dev::kStoreDeviceThroughPolicy>(rs, 4u * static_cast<uint32_t>(h * kPart + D),
                                                          make_uint2(__float_as_uint(top), __float_as_uint(l)));
        }
      }
    }
    if (whole) continue;
    // Device-scope write-through stores, acknowledged before the count: what the last workgroup of the pair to arrive
    // then reads, with device-coherent loads, is all there. No workgroup waits for another.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    const int64_t wa = share.Holder(run.first), wb = share.Holder(run.first + run.n - 1);
    uint32_t* counter = reinterpret_cast<uint32_t*>(workspace + wa * kCounterBytes);
    if (threadIdx.x == 0) {
      last_flag = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                  static_cast<uint32_t>(wb - wa);
    }
    __syncthreads();
    if (last_flag) {
      // wa's part is in its first slot only if the pair starts where its share does
      const bool first_leads = share.Begin(wa) == run.first;
      const __amdgpu_buffer_rsrc_t all =
          dev::OutResource(slots + 2 * wa * slot_floats, static_cast<uint32_t>((2 * (wb - wa) + 2) * slot_floats * 4));
      const int parts = static_cast<int>(wb - wa) + 1;
      auto slot_at = [&](int w) {
        return static_cast<uint32_t>((2 * w + (w == 0 && !first_leads ? 1 : 0)) * slot_floats * 4);
      };
      for (int i = threadIdx.x; i < heads * (D / 4); i += 64 * kWaves) {
        const int h = i / (D / 4), d = 4 * (i % (D / 4));
        const uint32_t ml = 4u * static_cast<uint32_t>(h * kPart + D), at = 4u * static_cast<uint32_t>(h * kPart + d);
        float top = -INFINITY;
        for (int w = 0; w < parts; ++w) {
          top = fmaxf(top, dev::LoadBuf1<dev::kLoadDevicePolicy>(all, slot_at(w) + ml));
        }
        const float safe = top == -INFINITY ? 0.0f : top;
        float l = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int w = 0; w < parts; ++w) {
          const uint2 x2 = dev::LoadBufU2<dev::kLoadDevicePolicy>(all, slot_at(w) + ml);
          const float f = __builtin_amdgcn_exp2f(__uint_as_float(x2.x) - safe);
          const float4 x = dev::LoadBuf4<dev::kLoadDevicePolicy>(all, slot_at(w) + at);
          l = fmaf(__uint_as_float(x2.y), f, l);
          o = make_float4(fmaf(x.x, f, o.x), fmaf(x.y, f, o.y), fmaf(x.z, f, o.z), fmaf(x.w, f, o.w));
        }
        const float inv = 1.0f / l;
        dev::Store4(out + (head_row + h) * D + d, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
      }
      // every workgroup of the pair has counted in: ready for the next call
      if (threadIdx.x == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();  // last_flag is read before the next run writes it
  }

  // rows with nothing to attend to: zeros, or NaN where the row is out of range
  for (int64_t r = me; r < rows.n_rows; r += gridDim.x) {
    const int64_t seq = rows.Seq(static_cast<int32_t>(r));
    const int32_t len = rows.lens[r];
    if (seq < 0) continue;
    const bool fine = rows.Fine(seq, len);
    if (fine && len > 0) continue;
    const float x = fine ? 0.0f : NAN;
    for (int64_t i = threadIdx.x; i < static_cast<int64_t>(n_heads) * (D / 4); i += 64 * kWaves) {
      dev::Store4(out + r * n_heads * D + 4 * i, make_float4(x, x, x, x));
    }
  }
}

// ---------------------------------------------------------------- host side

void CheckHeads(const char* what, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim) {
  RPG_CHECK(head_dim == 64 || head_dim == 128, "%s: head_dim %d is neither 64 nor 128", what, head_dim);
  RPG_CHECK(n_kv_heads > 0 && n_heads > 0 && n_heads <= (1 << 20) && n_heads % n_kv_heads == 0,
            "%s: %d query heads do not divide among %d kv heads", what, n_heads, n_kv_heads);
}

// A kv head's query heads in tiles of at most kTileHeads, as even as they go.
void TilesOf(int32_t group, int32_t* tiles, int32_t* tile_heads) {
  *tiles = (group + kTileHeads - 1) / kTileHeads;
  *tile_heads = (group + *tiles - 1) / *tiles;
}

}  // namespace

size_t GpuAttentionPagedWorkspaceBytes(int32_t n_heads, int32_t n_kv_heads, int32_t head_dim) {
  CheckHeads("AttentionPagedWorkspace", n_heads, n_kv_heads, head_dim);
  int32_t tiles, tile_heads;
  TilesOf(n_heads / n_kv_heads, &tiles, &tile_heads);
  return kMaxGroups * (kCounterBytes + 2 * sizeof(float) * static_cast<size_t>(tile_heads) *
                                           static_cast<size_t>(PartFloats(head_dim)));
}

void GpuAttentionPagedWorkspaceInit(void* workspace, size_t bytes) {
  RPG_CHECK(workspace != nullptr && bytes > 0 && bytes % 16 == 0 && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0,
            "AttentionPagedWorkspaceInit: a workspace is 256-byte aligned and a multiple of 16 bytes");
  GpuStreamFill(workspace, static_cast<int64_t>(bytes), 0);
}

void GpuAttentionPaged(const GpuPagedKv& kv, const GpuPageTable& table, const int32_t* seq_ids, const int32_t* lens,
                       const float* q_dev, int32_t n_heads, int64_t n_rows, float* out_dev, void* workspace,
                       size_t workspace_bytes) {
  CheckPagedKv("AttentionPaged", kv, table);
  CheckHeads("AttentionPaged", n_heads, kv.n_kv_heads, kv.head_dim);
  RPG_CHECK(n_rows >= 0 && n_rows <= 0x7FFFFFFF, "AttentionPaged: %lld rows", static_cast<long long>(n_rows));
  if (n_rows == 0) return;
  RPG_CHECK(lens != nullptr && q_dev != nullptr && out_dev != nullptr && workspace != nullptr,
            "AttentionPaged got a null pointer");
  RPG_CHECK(seq_ids != nullptr || n_rows <= table.n_seqs, "AttentionPaged: %lld rows without seq_ids, but %lld sequences",
            static_cast<long long>(n_rows), static_cast<long long>(table.n_seqs));
  RPG_CHECK(((reinterpret_cast<uintptr_t>(q_dev) | reinterpret_cast<uintptr_t>(out_dev)) & 15) == 0,
            "AttentionPaged: q and out have to be 16-byte aligned");
  const int64_t q_bytes = n_rows * n_heads * kv.head_dim * 4;
  RPG_CHECK(!Overlap(q_dev, q_bytes, out_dev, q_bytes), "AttentionPaged: out must not overlap q");
  const size_t need = GpuAttentionPagedWorkspaceBytes(n_heads, kv.n_kv_heads, kv.head_dim);
  RPG_CHECK((reinterpret_cast<uintptr_t>(workspace) & 255) == 0 && workspace_bytes >= need,
            "AttentionPaged: a workspace of %zu bytes, 256-byte aligned, is needed (%zu given)", need, workspace_bytes);
  int32_t tiles, tile_heads;
  TilesOf(n_heads / kv.n_kv_heads, &tiles, &tile_heads);
  const Rows rows{seq_ids, lens, table.n_seqs, table.max_pages * kv.page_size, static_cast<int32_t>(n_rows),
                  kv.n_kv_heads * tiles};
  // no more workgroups than the longest possible rows would give four units to
  const int64_t most = (std::min<int64_t>(rows.capacity, 0x7FFFFFFF) + 63) / 64;
  int64_t groups = kMaxGroups;
  if (most * rows.pairs < int64_t{4} * kMaxGroups) {
    groups = std::min<int64_t>(groups, (n_rows * most * rows.pairs + kWaves - 1) / kWaves);
  }
  const float scale_log2 =
      static_cast<float>(1.4426950408889634 / std::sqrt(static_cast<double>(kv.head_dim)));
  const bool q8 = kv.type == kKvQ8;
  auto* kern = kv.head_dim == 128 ? (q8 ? PagedAttentionKernel<128, true> : PagedAttentionKernel<128, false>)
                                  : (q8 ? PagedAttentionKernel<64, true> : PagedAttentionKernel<64, false>);
  Launch("PagedAttentionKernel", kern, dim3(static_cast<unsigned>(groups)), dim3(64 * kWaves), dev::ViewOf(kv, table),
         rows, q_dev, n_heads, tiles, tile_heads, scale_log2, out_dev, static_cast<char*>(workspace));
}

}  // namespace rpg
