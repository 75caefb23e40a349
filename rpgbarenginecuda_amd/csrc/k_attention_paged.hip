// Attention of one new token per row over the paged KV cache.
//
// For row r, query head h of kv head h / G, over the positions j < lens[r]:
//   s_j = (q . k_j) / sqrt(D),  out = sum_j exp(s_j - max s) v_j / sum_j exp(s_j - max s)
// in one pass over the cache, with the running maximum m and sum l: on a new
// maximum the sum and the accumulated output are scaled by exp(m_old - m_new).
// Exponentials are taken as powers of two, with log2(e) in the scores' scale.
//
// What bounds it: the cache is read once, 2 D (+ 4) bytes of keys and values a
// position and kv head, and 4 D G operations are done on them. Both products run on
// the matrix cores, where the G query heads of a kv head are columns of a 16-column
// tile: rows of S = K Q^T are 16 keys, rows of O^T = V^T P^T 16 elements, so that a
// lane ends the first with the weights of the keys that it holds in the second.
//
// fp16 cache (16x16x32, fp32 sums): keys and values enter as they are kept, queries
// and weights, which are fp32, as two fp16 terms of 11 bits, hi + lo, in columns n
// and n + 8 of one tile. A query row is first scaled by a power of two to a largest
// magnitude in [2^14, 2^15), weights by 2^14, so that what fp16's low end loses is
// below 2^-38 of the largest. hi is cut off from slightly below the value, so that
// both terms have its sign and neither is zero: infinities in the cache then give
// what the one product would (weights below 2^-23 of the largest excepted, which may
// turn an infinite value into NaN).
//
// 8-bit cache (16x16x64, int32 sums): the codes enter as they are kept and a step's sums are exact. Queries are taken to
// whole numbers below 2^30, relative to a row's largest. What the codes of values are multiplied by is weight times their
// row's scale, p_j c_j: whole numbers of 2^-29 of the power of two at or below the largest of the head's 64 of this step.
// That is what counts in the step, so a row of a large scale and no weight costs the others nothing; each is off by at
// most 2^-30 of a term that is there. Either enters as four signed digits of 8 bits, in columns n, n + 4, n + 8, n + 12. A
// step's sums are then taken to fp32, where the output's have a power of two of their own, moved only where a step's
// largest passes it by 2^64: codes times scales of any size there is have room. (int32 sums kept from step to step, which
// need one power of two for all of them, were no faster: 128 x 8192 positions 188.5 us against 189.5, 1 x 32768 20.8
// against 20.2, 45 x 2000 25.3 against 25.8.) The maximum that weights are relative to moves only where a score exceeds it
// by 3 (log2). Of the four lanes that have a score's digits each does a part of the softmax.
//
// Keys and values come straight to LDS in whole 128-byte lines, the next step's as
// soon as this step has read what they replace; the transposition of values is the
// LDS read's. The pieces of 16 bytes of a row lie permuted by the row's number, which
// spreads the reads over the banks.
//
// Sharing out: work is counted in units of 32 or 64 positions of one (row, kv head,
// tile of up to 8 heads). Every wave adds up the rows' units by itself from lens and
// takes an equal, contiguous share of them, so that ragged batches and single long
// rows fill the card alike and nothing about the lengths is needed on the host. A
// wave writes what it holds whole; where a (row, tile) is split over waves of one
// workgroup they join in LDS, and where it is split over workgroups each leaves its
// part in the workspace and the last to arrive joins them, in order.
//
// Measured (the kernel between events that its dispatch carries, as every time in this
// file): 32 rows of up to 4096 positions in fp16, 16 / 8 heads, 269 MB: 50.3 us,
// 5.3 TB/s; 128 rows of up to 8192 in 8 bits, 32 / 8 heads, 1152 MB: 189.5 us, 6.1
// TB/s (fp16, 2230 MB: 355 us, 6.3 TB/s); 16 rows of 4000 in 8 bits, 64 / 8 heads, two
// column tiles, 136 MB: 35.0 us, 3.9 TB/s; where a pure read of as much reaches 7.0. While all workgroups run the reads come at about that
// rate; the rest is the end, where every other XCD is a tenth slower and of a compute
// unit's two workgroups the one whose loads come behind a fifth. Shares to match gained
// a few percent on ragged batches and lost as much where equal shares split no row
// (64 x 4096 positions from 93 to 100 us), and dealing the last fifth out late, in
// shares of their own, cost what it gained.
// 1 x 500 positions, 9 us, and 1 x 60, 7.0 us, are the chain of round trips: lengths
// 0.5, the search for the share 0.7, page table 0.2, keys 1.5, products and weights
// 1.9, join in LDS 0.6 and, where a pair is split, store and count 1.3 and the last
// one's read and join 1.5. One row of 32768 positions in 8 bits, 8 kv heads, 69 MB:
// 20.5 us, that chain with a join of 32 parts at its end and 10.7 us of reading in its
// middle (each further 32768 positions take 10.7 us, 6.5 TB/s, up to 262144: 95 us).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attention_dev.h"
#include "dev_util.h"
#include "kernels_gpu.h"
#include "launch.h"
#include "paged_kv.h"

namespace rpg {
namespace {

using namespace attn;
using dev::PagedView;

// Four waves of up to 17 KB of keys and values each: two workgroups to a compute unit. (Eight waves and one workgroup
// were slower on short calls, 1 x 500 positions by 15%, and alike on long ones; four waves and one workgroup with two
// steps under way each were slower on long ones.)
constexpr int kWaves = 4;
constexpr int kTileHeads = 8;
// Workgroups at most; a workspace has two part slots and a counter for each.
constexpr int kMaxGroups = 512;
// Bytes between two counters: on lines of their own, as the decode attention's.
constexpr size_t kCounterBytes = 256;
// Stores of a part to the workspace: device scope. With the streaming hint too their
// acknowledgement comes later (1 x 32768 positions in fp16 of one kv head 17.8 against 16.6 us).
constexpr int kPartPolicy = 16;

constexpr int PartFloats(int d) { return d + 4; }  // in LDS: o[d], m, l, and two to keep rows 16-byte aligned
constexpr uint32_t kLine = 128;
// In the workspace: o[heads][d], and a line of (m, l)
__host__ __device__ constexpr uint32_t SlotBytes(int32_t d, int32_t heads) {
  return static_cast<uint32_t>(heads * d) * 4u + kLine;
}

// ---------------------------------------------------------------- conversions

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

// Signed digit `at` (selector bytes: at, 4 + at) of four whole numbers given with
// 0x80808080 added: x = sum of digit_i 256^i with digit_i = byte i - 128 there.
__device__ __forceinline__ int Digit4(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t selector) {
  const uint32_t lo = __builtin_amdgcn_perm(b, a, selector), hi = __builtin_amdgcn_perm(d, c, selector);
  return static_cast<int>(__builtin_amdgcn_perm(hi, lo, 0x05040100u) ^ 0x80808080u);
}

// ---------------------------------------------------------------- sharing out

// How a pair's units are cut into items, of which a workgroup takes whole ones. From kManyUnits in the batch on an item is
// a unit, so that all workgroups get alike. With fewer, joining what two workgroups hold of a pair (a round trip to memory
// to store, one to count, one to read) costs more than some units more in turn: a pair of up to kWholeUnits is one item, a
// longer one is cut evenly into items of at most 2^step, about what each workgroup then gets.
// (One row of 250 positions, 8 units for each of 8 kv heads: 8.1 us whole, 9.1 in two items each; of 500, 16 units: 10.3
// whole, 9.6 in four items each.)
constexpr uint32_t kManyUnits = 8192;
constexpr uint32_t kWholeUnits = 8;
constexpr uint32_t kLeastStep = 2;

struct Cut {
  bool units;
  uint32_t step;

  // for a batch of `all` units
  __device__ __forceinline__ explicit Cut(uint32_t all) {
    units = all >= kManyUnits;
    step = kLeastStep + (all <= 4 * kMaxGroups ? 0 : all <= 8 * kMaxGroups ? 1 : 2);
  }
  __device__ __forceinline__ uint32_t Items(uint32_t n) const {
    return units ? n : n <= kWholeUnits ? min(n, 1u) : (n + (1u << step) - 1u) >> step;
  }
};

struct Rows {
  const int32_t* seq_ids;
  const int32_t* lens;
  int32_t n_seqs;
  int32_t capacity;  // positions that a table row has pages for, at most the largest int32
  int32_t n_rows;
  int32_t pairs;       // (kv head, tile) pairs of a row
  int32_t unit_shift;  // log2 of a unit's positions

  __device__ __forceinline__ int32_t Seq(int32_t r) const { return seq_ids != nullptr ? seq_ids[r] : r; }
  __device__ __forceinline__ bool Fine(int32_t seq, int32_t len) const {
    return seq >= 0 && seq < n_seqs && len >= 0 && len <= capacity;
  }
  // Units of one pair of row r; none for a row that is padding, empty or out of range.
  __device__ __forceinline__ uint32_t UnitsOf(int32_t seq, int32_t len) const {
    return Fine(seq, len) ? (static_cast<uint32_t>(len) + (1u << unit_shift) - 1u) >> unit_shift : 0u;
  }
  __device__ __forceinline__ uint32_t UnitsOf(int32_t r) const { return UnitsOf(Seq(r), lens[r]); }
  // for an r that is the same in every lane
  __device__ __forceinline__ int32_t ScalarSeq(int32_t r) const {
    return seq_ids != nullptr ? ScalarLoad(seq_ids + r) : r;
  }
  __device__ __forceinline__ uint32_t ScalarUnitsOf(int32_t r) const {
    return UnitsOf(ScalarSeq(r), ScalarLoad(lens + r));
  }
};

// No part of a batch's rows is shared.
struct NotShared {
  static constexpr bool kOn = false;
  __device__ __forceinline__ int32_t PagesOfLane(const Rows&, int32_t, int32_t, int32_t) const { return 0; }
  __device__ __forceinline__ int32_t PagesOf(const Rows&, int32_t, int32_t, int32_t) const { return 0; }
};

// Groups of rows that begin with the same pages (dev::SharedGroups): what a row has of them is attended to elsewhere, and
// here only what is behind. (32 rows of 1 to 1024 positions behind 2816 shared ones, fp16: 21.6 us, where the same positions
// alone in their tables take 19.5: groups are looked up for each row.)
struct Shared {
  static constexpr bool kOn = true;
  dev::SharedGroups groups;
  int32_t page_shift;

  // whole pages of row r before what is its own; r is the lane's
  __device__ __forceinline__ int32_t PagesOfLane(const Rows& rows, int32_t r, int32_t seq, int32_t len) const {
    return Taken(rows, groups.PagesOfLane(r), seq, len);
  }
  // r the same in every lane
  __device__ __forceinline__ int32_t PagesOf(const Rows& rows, int32_t r, int32_t seq, int32_t len) const {
    return Taken(rows, groups.PagesOf(r), seq, len);
  }
  __device__ __forceinline__ int32_t Taken(const Rows& rows, int32_t pages, int32_t seq, int32_t len) const {
    return rows.Fine(seq, len) && dev::TakesPart(pages, page_shift, len) ? pages : 0;
  }
};

// Unit c of `units` of `pair` of `row`.
struct Place {
  int32_t row, pair;
  uint32_t c, units;
};

// The batch as a wave sees it: rows are taken `each` to a lane, with the units and the items before them. (A short call's
// start is bound by fetching its instructions, so what is needed in several places is written in one.)
template <class S>
struct Batch {
  const Rows& rows;
  const S& shared;
  Cut cut{0};
  int lane;
  int32_t each;
  uint32_t units, items;
  uint32_t units_before, items_before;
  int32_t own_len = 0, own_seq = -1, own_pages = 0;  // where each is 1: of row `lane`
  uint32_t own_units = 0;

  __device__ __forceinline__ Batch(const Rows& r, const S& s, int l) : rows(r), shared(s), lane(l) {
    each = (rows.n_rows + 63) / 64;
    if (__builtin_expect(each == 1, 1)) {
      if (lane < rows.n_rows) {
        own_len = rows.lens[lane];
        own_seq = rows.Seq(lane);
        if constexpr (!S::kOn) own_units = rows.UnitsOf(own_seq, own_len);
      }
      if constexpr (S::kOn) {
        own_pages = shared.PagesOfLane(rows, lane, own_seq, own_len);
        own_len -= own_pages << PageShift();
        own_units = rows.UnitsOf(own_seq, own_len);
      }
    }
    units_before = Before(0, rows.n_rows, each, false, &units);
    cut = Cut(units);
    items = units;
    items_before = units_before;
    if (!cut.units) items_before = Before(0, rows.n_rows, each, true, &items);
  }

  // Of rows [lo, hi), taken `some` to a lane: the units, or items, before this lane's.
  __device__ __forceinline__ uint32_t Before(int32_t lo, int32_t hi, int32_t some, bool of_items, uint32_t* total) const {
    uint32_t own = 0;
    if (__builtin_expect(each == 1, 1)) {
      own = of_items ? cut.Items(own_units) : own_units;
    } else {
      const int64_t first = lo + static_cast<int64_t>(lane) * some;
      if constexpr (S::kOn) {  // groups are looked up by all lanes, those behind the last row too
#pragma unroll 1
        for (int32_t i = 0; i < some; ++i) {
          const uint32_t n = LaneUnitsOf(static_cast<int32_t>(min(first + i, static_cast<int64_t>(hi) - 1)));
          if (first + i < hi) own += of_items ? cut.Items(n) : n;
        }
      } else {
#pragma unroll 2
        for (int32_t i = 0; i < some; ++i) {
          if (first + i < hi) {
            const uint32_t n = LaneUnitsOf(static_cast<int32_t>(first + i));
            own += of_items ? cut.Items(n) : n;
          }
        }
      }
    }
    own *= static_cast<uint32_t>(rows.pairs);
    const uint32_t sum = ScanAdd(own);
    *total = __builtin_amdgcn_readlane(sum, 63);
    return sum - own;
  }

  // log2 of a page's positions
  __device__ __forceinline__ int32_t PageShift() const {
    if constexpr (S::kOn) return shared.page_shift;
    return 0;
  }
  __device__ __forceinline__ uint32_t LaneUnitsOf(int32_t r) const {
    if constexpr (!S::kOn) return rows.UnitsOf(r);
    const int32_t seq = rows.Seq(r), len = rows.lens[r];
    return rows.UnitsOf(seq, len - (shared.PagesOfLane(rows, r, seq, len) << PageShift()));
  }

  // Of one row, the same in every lane: pages that are not its own, units and positions behind them
  __device__ __forceinline__ int32_t PagesOf(int32_t r) const {
    if constexpr (!S::kOn) return 0;
    return __builtin_expect(each == 1, 1) ? __builtin_amdgcn_readlane(own_pages, r)
                                          : shared.PagesOf(rows, r, rows.ScalarSeq(r), ScalarLoad(rows.lens + r));
  }
  __device__ __forceinline__ uint32_t UnitsOf(int32_t r) const {
    if (__builtin_expect(each == 1, 1)) return __builtin_amdgcn_readlane(own_units, r);
    if constexpr (!S::kOn) return rows.ScalarUnitsOf(r);
    return rows.UnitsOf(rows.ScalarSeq(r), LenOf(r));
  }
  __device__ __forceinline__ int32_t LenOf(int32_t r) const {
    if (__builtin_expect(each == 1, 1)) return __builtin_amdgcn_readlane(own_len, r);
    return ScalarLoad(rows.lens + r) - (PagesOf(r) << PageShift());
  }
  __device__ __forceinline__ int64_t SeqOf(int32_t r) const {
    return __builtin_expect(each == 1, 1) ? __builtin_amdgcn_readlane(own_seq, r) : rows.ScalarSeq(r);
  }

  // Where item x (unit x, unless by_items) begins: its place, its number among the units, and in *past that of the first
  // unit behind it.
  __device__ __forceinline__ uint32_t Locate(uint32_t x, bool by_items, Place* p, uint32_t* past) const {
    int32_t lo = 0, hi = rows.n_rows, some = each;
    uint32_t ub = units_before, ib = items_before, before = 0;
#pragma unroll 1
    while (true) {
      // the counts do not fall from lane to lane, and the last lane at or below x does not stand for empty rows
      const uint32_t b = by_items ? ib : ub;
      const int at = static_cast<int>(__builtin_popcountll(__ballot(b <= x))) - 1;
      x -= __builtin_amdgcn_readlane(b, at);
      before += __builtin_amdgcn_readlane(ub, at);
      lo += at * some;
      if (__builtin_expect(some == 1, 1)) break;
      hi = min(lo + some, hi);
      some = (hi - lo + 63) / 64;
      uint32_t unused;
#pragma unroll 1
      for (int pass = 0; pass < 2; ++pass) {
        ub = ib;
        ib = Before(lo, hi, some, pass == 1, &unused);
      }
    }
    p->row = lo;
    p->units = UnitsOf(lo);
    const uint32_t k = by_items ? cut.Items(p->units) : p->units;
    uint32_t pair = 0;
    if (x >= k) pair = Scalar(x / k);
    const uint32_t i = x - pair * k;
    p->pair = static_cast<int32_t>(pair);
    const uint32_t first = before + pair * p->units;
    if (!by_items) {
      p->c = i;
      *past = first + i + 1;
    } else if (k == 1) {
      p->c = 0;
      *past = first + p->units;
    } else {  // k items of q units, and one more in the first r of them
      const uint32_t q = Scalar(p->units / k), r = p->units - q * k;
      p->c = i * q + min(i, r);
      *past = first + p->c + q + (i < r ? 1 : 0);
    }
    return first + p->c;
  }

  // The first item of a pair of n units, whose first unit is `first`.
  __device__ __forceinline__ uint32_t ItemOfPair(uint32_t first, int32_t row, int32_t pair, uint32_t n) const {
    if (cut.units) return first;
    const int32_t at = each == 1 ? row : static_cast<int32_t>(Scalar(static_cast<uint32_t>(row) / static_cast<uint32_t>(each)));
    uint32_t items_of_rows = 0;
#pragma unroll 1
    for (int32_t r = at * each; r < row; ++r) items_of_rows += cut.Items(UnitsOf(r));
    return __builtin_amdgcn_readlane(items_before, at) + items_of_rows * static_cast<uint32_t>(rows.pairs) +
           static_cast<uint32_t>(pair) * cut.Items(n);
  }
};

// ---------------------------------------------------------------- the kernel

// What a wave or workgroup holds of a (row, pair): its units [c0, c1) of n.
struct Piece {
  uint32_t first;  // number of the pair's first unit
  uint32_t c0, c1, n;
  int32_t row, pair;
};

// One tile is the rule, and a division takes as long as twenty other instructions.
__device__ __forceinline__ int32_t KvHeadOf(int32_t pair, int32_t tiles) { return tiles == 1 ? pair : pair / tiles; }

// The query heads of a piece.
struct HeadsOf {
  int32_t heads;
  int64_t head_row;  // row of the first in q and out

  __device__ __forceinline__ HeadsOf(const Piece& p, int32_t n_heads, int32_t group, int32_t tiles, int32_t tile_heads) {
    const int32_t kh = KvHeadOf(p.pair, tiles);
    const int32_t h0 = (p.pair - kh * tiles) * tile_heads;
    heads = min(tile_heads, group - h0);
    head_row = static_cast<int64_t>(p.row) * n_heads + kh * group + h0;
  }
};

// A pair of up to kJoinAtOnce parts is joined in one step; of more in two, each kFan parts in the first. (In one step, 256
// parts of 1 x 32768 positions of one kv head make 49.5 us of 16.6, 128 of 1 x 65536 of two 26.9 of 20.4; at 64 parts
// they were alike.)
constexpr uint32_t kJoinAtOnce = 32;
constexpr uint32_t kFan = 16;

// The workgroups wa, wa + 1, ... that hold parts of a piece's pair, and workgroup me's place among them.
struct Parts {
  uint32_t wa = 0, parts = 0, blocks = 0, block = 0, block_parts = 0;
  bool leads = false;  // the pair's first part is the first thing that workgroup wa holds

  __device__ __forceinline__ Parts() {}
  template <class S>
  __device__ __forceinline__ Parts(const Piece& p, const Batch<S>& batch, const Share& share, uint32_t me) {
    const uint32_t item = batch.ItemOfPair(p.first, p.row, p.pair, p.n);
    wa = share.Holder(item);
    leads = share.Begin(wa) == item;
    parts = share.Holder(item + batch.cut.Items(p.n) - 1) - wa + 1;
    blocks = parts <= kJoinAtOnce ? 1 : (parts + kFan - 1) / kFan;
    block = blocks == 1 ? 0 : (me - wa) / kFan;
    block_parts = blocks == 1 ? parts : min(kFan, parts - block * kFan);
  }
  // Counters, in words of the workspace. A workgroup is the first holder of one split pair at most, and a later block's
  // first holder of one at most.
  __device__ __forceinline__ uint32_t PairCounter() const { return wa * (kCounterBytes / 4); }
  __device__ __forceinline__ uint32_t BlockCounter() const {
    return (wa + block * kFan) * (kCounterBytes / 4) + (block == 0 ? 1 : 2);
  }
};

// One argument: a launch takes longer for every pointer among its arguments (0.06 us of host time).
struct AttentionArgs {
  PagedView view;
  Rows rows;
  const float* q;
  float* out;
  char* workspace;
  int32_t n_heads;
  int32_t group;  // query heads of a kv head
  int32_t tiles;
  int32_t tile_heads;
  float scale_log2;
};

// The same for rows that share their beginnings: what is behind these, and where (m, l) of each row and head go.
struct SharedAttentionArgs : AttentionArgs {
  const int32_t* group_rows;
  const int32_t* group_pages;
  int32_t n_groups;
  int64_t least;
  float* ml;
};

__device__ __forceinline__ void StoreMl(const SharedAttentionArgs& args, int64_t row_head, float m, float l) {
  *reinterpret_cast<float2*>(args.ml + 2 * row_head) = make_float2(m, l);
}

// kTiles: 8-bit caches, column tiles of up to 4 heads (1 or 2); else 1, of up to 8.
template <int D, bool kQ8, int kTiles, class Args>
__global__ __launch_bounds__(64 * kWaves, 2) void PagedAttentionKernel(const Args args) {
  constexpr bool kShared = std::is_same_v<Args, SharedAttentionArgs>;
  const PagedView& view = args.view;
  const Rows& rows = args.rows;
  const float* __restrict__ q = args.q;
  float* __restrict__ out = args.out;
  char* __restrict__ workspace = args.workspace;
  const int32_t n_heads = args.n_heads, group = args.group, tiles = args.tiles, tile_heads = args.tile_heads;
  const float scale_log2 = args.scale_log2;
  constexpr int kSub = D == 128 && !kQ8 ? 2 : 4;  // 16-key tiles of a step, which is a unit
  constexpr int kStep = 16 * kSub;
  constexpr int kRow = D * (kQ8 ? 1 : 2);  // bytes of a cached row
  constexpr int kPieces = kRow / 16;       // of 16 bytes
  constexpr int kLoads = kRow / 64;        // loads of 64 pieces for 16 keys
  constexpr int kSteps = kRow / 64;        // matrix products of 16 keys
  constexpr int kE = D / 16;               // tiles of 16 elements of a value row
  constexpr int kPart = PartFloats(D);
  constexpr int kCopies = kQ8 ? 4 : 2;     // columns of a head, that is lanes that have its final sums
  constexpr int kHeadCols = 16 / kCopies;
  constexpr int kOwn = kE / kCopies;       // tiles of 16 elements that each of them writes

  // a wave's step of keys and values, each row's scale behind them
  constexpr int kStage = kStep * kRow + (kQ8 ? kStep * 4 : 0);
  constexpr int kStageLoads = kSub * kLoads + (kQ8 ? 1 : 0);
  __shared__ __attribute__((aligned(16))) char k_lds[kWaves][kStage];
  __shared__ __attribute__((aligned(16))) char v_lds[kWaves][kStage];
  static_assert(kTileHeads * kPart * 4 <= kStep * kRow, "a part fits where keys or values were");
  struct Join {
    float4 o;
    float m, l;
  };
  __shared__ Join joins[64 * kWaves];
  __shared__ Piece pieces[kWaves][2];
  __shared__ int held[kWaves];
  __shared__ int flags[2];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int n = lane & 15;
  const int g = lane >> 4;
  const int head_col = n % kHeadCols;
  const int copy = n / kHeadCols;

  // the batch's units, and this wave's share
  const auto shared = [&] {
    if constexpr (kShared) {
      return Shared{dev::SharedGroups(args.group_rows, args.group_pages, args.n_groups, args.least, rows.n_rows, view.max_pages, lane),
                    view.page_shift};
    } else {
      return NotShared{};
    }
  }();
  using S = std::conditional_t<kShared, Shared, NotShared>;
  const Batch<S> batch(rows, shared, lane);
  const uint32_t groups = min(gridDim.x, batch.cut.units ? (batch.units + 3) / 4 : batch.items);
  const Share share(batch.items, max(groups, 1u));
  const uint32_t me = blockIdx.x;
  Place first;  // where the workgroup's share begins, and then the wave's
  uint32_t begin = 0, end = 0, u = 0, u_end = 0;
  if (me < groups) {
    const uint32_t next = share.Begin(me + 1);
    uint32_t x = share.Begin(me), past = 0;
    bool by_items = !batch.cut.units;
    int query = 0;
#pragma unroll 1
    while (true) {
      Place p;
      const uint32_t found = batch.Locate(x, by_items, &p, &past);
      if (query != 1) first = p;
      if (query == 2) break;
      if (query == 0) {
        begin = found;
        end = next == batch.items ? batch.units : by_items ? past : next;
        if (by_items && next != batch.items && next != x + 1) {
          x = next;
          query = 1;
          continue;
        }
      } else {
        end = found;
      }
      u = begin + (((end - begin) * wave) >> 2);
      u_end = begin + (((end - begin) * (wave + 1)) >> 2);
      static_assert(kWaves == 4, "a wave's share of its workgroup's");
      if (u == u_end || first.c + (u - begin) < first.units) {
        first.c += u - begin;
        break;
      }
      x = u;
      by_items = false;
      query = 2;
    }
  }

  int my_held = 0;  // bit 0: the first piece, bit 1: the last
  if (u < u_end) {
    char* const k_mine = k_lds[wave];
    char* const v_mine = v_lds[wave];
    // Loads: lane i takes piece i % kPieces of row i / kPieces of each load's rows, and puts there what belongs there:
    // piece p of key row r lies at p ^ k_swap(r), of value row r at p ^ v_swap(r).
    const int lrow = lane / kPieces, lpiece = lane % kPieces;
    constexpr int kLoadRows = 64 / kPieces;
    const auto k_swap = [](int r) { return kPieces == 16 ? r & 15 : kPieces == 8 ? r & 7 : (r >> 1) & 3; };
    const auto v_swap = [](int r, int odd) {  // odd: of an odd-numbered tile of 16 keys
      return !kQ8 ? 2 * (r & 3) : kPieces == 8 ? (r & 3) | (odd << 2) : ((r >> 1) & 1) | (odd << 1);
    };
    constexpr int kKeyOffs = kPieces == 16 ? 4 : 1;  // with 16 pieces the rows of a load are permuted as its number says
    uint32_t k_from[kKeyOffs], v_from[2][1];
#pragma unroll
    for (int i = 0; i < kKeyOffs; ++i) {
      k_from[i] = static_cast<uint32_t>(lrow * kRow + 16 * (lpiece ^ k_swap(i * kLoadRows + lrow)));
    }
#pragma unroll
    for (int odd = 0; odd < 2; ++odd) {
      v_from[odd][0] = static_cast<uint32_t>(lrow * kRow + 16 * (lpiece ^ v_swap(lrow, odd)));
    }
    // Reads: the key operand's pieces g, 4 + g, ... of row n; the value operand's rows as its keys have weights here
    const uint32_t k_at = static_cast<uint32_t>(n * kRow + 16 * (g ^ k_swap(n)));
    uint32_t v_at;
    if constexpr (kQ8) {
      const int i = n >> 1;  // key 4 g + i % 4 of tile i / 4, and of tile 2 + i / 4
      v_at = static_cast<uint32_t>(((i >> 2) * 16 + 4 * g + (i & 3)) * kRow + 16 * v_swap(i & 3, i >> 2) + 8 * (n & 1));
    } else {
      const int i = n >> 2;  // key 4 g + i of each tile
      v_at = static_cast<uint32_t>((4 * g + i) * kRow + 16 * (((n & 3) >> 1) ^ v_swap(i, 0)) + 8 * (n & 1));
    }

    // where the wave is: unit c of `units` of `pair` of `row`
    int32_t row = first.row, pair = first.pair;
    uint32_t c = first.c, units = first.units;
    int32_t len = batch.LenOf(row);
    const int32_t* table = view.pages + batch.SeqOf(row) * view.max_pages + batch.PagesOf(row);

    // Rows of the pool that the 16-key tiles of unit c start at; a tile past the end repeats the unit's first, a page
    // out of range is read as page 0 and its tile marked.
    int64_t at[kSub];
    int bad = 0;
    const auto find = [&]() {
      bad = 0;
      const int32_t pos = static_cast<int32_t>(c) * kStep;
      const int32_t left = len - pos;  // no sum of positions here or below may pass the largest int32
      const int32_t kh = KvHeadOf(pair, tiles);
      int32_t pages[kSub];
#pragma unroll
      for (int j = 0; j < kSub; ++j) {
        pages[j] = ScalarLoad(table + ((16 * j < left ? pos + 16 * j : pos) >> view.page_shift));
      }
#pragma unroll
      for (int j = 0; j < kSub; ++j) {
        const int32_t p = 16 * j < left ? pos + 16 * j : pos;
        const bool fine = static_cast<uint32_t>(pages[j]) < static_cast<uint32_t>(view.n_pages);
        const int32_t page = fine ? pages[j] : 0;
        bad |= fine ? 0 : 1 << j;
        at[j] = ((static_cast<int64_t>(page) * view.n_kv + kh) << view.page_shift) + (p & ((1 << view.page_shift) - 1));
      }
    };
    // the address of this lane's position's scale, of tile g (by masks: from a choice among them the compiler makes an
    // array in memory)
    uint32_t is_tile[kSub];
#pragma unroll
    for (int j = 0; j < kSub; ++j) is_tile[j] = g == j ? ~0u : 0u;
    const auto scale_of = [&](const float* scales) {
      uint32_t lo = 0, hi = 0;
#pragma unroll
      for (int j = 0; j < kSub; ++j) {
        lo |= static_cast<uint32_t>(at[j]) & is_tile[j];
        hi |= static_cast<uint32_t>(at[j] >> 32) & is_tile[j];
      }
      return scales + static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo) + n;
    };
    const uint32_t k_to = LdsAddress(k_mine), v_to = LdsAddress(v_mine);
    const auto load_k = [&]() {
      WaitLdsReads();
#pragma unroll
      for (int j = 0; j < kSub; ++j) {
        const Resource rs = RowsResource(static_cast<const char*>(view.k) + at[j] * kRow, 16 * kRow);
        LoadToLds<kLoads>(rs, k_from, k_to + j * kLoads * 1024);
      }
      if constexpr (kQ8) LoadWordToLds(scale_of(view.k_scale), k_to + kStep * kRow);
    };
    const auto load_v = [&]() {
      WaitLdsReads();
#pragma unroll
      for (int j = 0; j < kSub; ++j) {
        const Resource rs = RowsResource(static_cast<const char*>(view.v) + at[j] * kRow, 16 * kRow);
        LoadToLds<kLoads>(rs, v_from[j & 1], v_to + j * kLoads * 1024);
      }
      if constexpr (kQ8) LoadWordToLds(scale_of(view.v_scale), v_to + kStep * kRow);
    };

    // of a compute unit's two workgroups the second waits behind the first wherever both have something to issue: going
    // first there, it ends sooner (128 x 8192 positions in 8 bits 195.2 -> 190.4 us; other calls within a percent)
    if (me >= gridDim.x / 2) __builtin_amdgcn_s_setprio(1);
    find();
    load_k();
    load_v();

    // 8-bit caches: of the four lanes that have the copies of a column, each takes a part of the softmax and not all the
    // whole of it. Where there are two column tiles, odd copies take the second, even ones the first, and of the step's
    // tiles of 16 keys copies 2 and 3 the upper half; with one column tile odd copies take the upper half.
    constexpr int kMine = kQ8 ? kSub / 2 : kSub;  // tiles of 16 keys for a lane
    const bool upper = kQ8 && (kTiles > 1 ? copy >= 2 : (copy & 1) != 0);
    const int mine_at = upper ? kMine : 0;
    // the lane of the same column tile that has the other half
    const auto other_half = [](float x) { return kTiles > 1 ? Ror<8>(x) : Ror<4>(x); };
    // x of column tile t in every lane
    const bool second = kTiles > 1 && (copy & 1) != 0;
    const auto of_tile = [&](int t, float x) {
      if constexpr (kTiles == 1) return x;
      const float other = Ror<4>(x);  // by all lanes
      return second == (t == 1) ? x : other;
    };

    // per piece: the queries' terms or digits, and the running state
    Half8 qh[kQ8 ? 1 : kSteps];
    I32x4 qi[kQ8 ? kTiles : 1][kQ8 ? kSteps : 1];
    float to_score[kTiles], m, l;
    int key_exp = 0;  // 8-bit keys: the power of two that their scales are multiplied by, for the lane's tile
    // 8-bit values: the power of two (times what m moved by since) that acc holds them multiplied by; infinity where that
    // is nothing yet
    float shrink = INFINITY;
    F32x4 acc[kTiles][kE];
    // the digit that this lane's column stands for, and its weight
    const uint32_t digit = static_cast<uint32_t>(copy) * 0x0101u + 0x0400u;
    const float digit_by = __int_as_float((127 + 8 * copy) << 23);
    int64_t head_row = 0;
    int32_t heads = 0;
    const auto begin_piece = [&]() {
      const int32_t kh = KvHeadOf(pair, tiles);
      const int32_t h0 = (pair - kh * tiles) * tile_heads;
      heads = min(tile_heads, group - h0);
      head_row = static_cast<int64_t>(row) * n_heads + kh * group + h0;
      shrink = INFINITY;
      m = -INFINITY;
      l = 0.0f;
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        const int h = t * kHeadCols + head_col;
        const bool there = h < heads;
        const float* qr = q + (head_row + (there ? h : 0)) * D;
#pragma unroll
        for (int i = 0; i < kE; ++i) acc[t][i] = F32x4{0.0f, 0.0f, 0.0f, 0.0f};
        constexpr int kAt = kQ8 ? 16 : 8;  // elements of a lane for one product
        float x[kSteps][kAt];
        float top = 0.0f, odd = 0.0f;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
#pragma unroll
          for (int i = 0; i < kAt; i += 4) {
            const float4 a = dev::Load4(qr + (4 * s + g) * kAt + i);
            const float e[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              x[s][i + k] = there ? e[k] : 0.0f;
              top = fmaxf(top, fabsf(x[s][i + k]));
              if constexpr (kQ8) odd += x[s][i + k] * 0.0f;  // NaN if one of them is no finite number
            }
          }
        }
        top = MaxAcrossRows(top);
        if constexpr (kQ8) {
          // the power of two that brings top to [2^29, 2^30), taken back with the products where these stay in fp32's range
          // (below 2^43 before it), and what is left of it for queries far from 1 with the keys' scales
          const int by = 30 - __builtin_amdgcn_frexp_expf(top);
          const int back = min(max(-by, -80), 80);
          if (kTiles == 1 || second == (t == 1)) key_exp = -by - back;
          to_score[t] = ldexpf(scale_log2 * digit_by, back) + SumAcrossRows(odd);
#pragma unroll
          for (int s = 0; s < kSteps; ++s) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t w[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                w[k] = static_cast<uint32_t>(static_cast<int>(__builtin_rintf(ldexpf(x[s][4 * i + k], by)))) + 0x80808080u;
              }
              qi[t][s][i] = Digit4(w[0], w[1], w[2], w[3], digit);
            }
          }
        } else {
          const int e = min(max(268 - (__float_as_int(top) >> 23), 1), 254);  // brings top to [2^14, 2^15)
          const float up = __int_as_float(e << 23);
          to_score[t] = ldexpf(scale_log2, 127 - e);
#pragma unroll
          for (int s = 0; s < kSteps; ++s) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = Term2(x[s][2 * i] * up, x[s][2 * i + 1] * up, copy != 0);
            qh[s] = AsHalf8(w[0], w[1], w[2], w[3]);
          }
        }
      }
    };
    // the scales of keys 4 g .. 4 g + 3 of tile j
    const auto scales_at = [&](const char* stage, int j) {
      return *reinterpret_cast<const float4*>(stage + kStep * kRow + 64 * j + 16 * g);
    };

    uint32_t c_first = c;
    bool turned = true;  // the unit at hand is its piece's first
    F32x4 kept[kTiles][kOwn];
    float kept_m[kTiles], kept_l[kTiles];

    while (true) {
      if (turned) {
        begin_piece();
        turned = false;
      }
      const int32_t pos = static_cast<int32_t>(c) * kStep;
      const int32_t left = len - pos;  // positions from here
      const bool tail = left < kStep;
      const int this_bad = bad;
      // ---- scores, once the keys are there: the values' loads are younger
      WaitLoads<kStageLoads>();
      float s[kMine][4];
      I32x4 raw[kQ8 ? kTiles : 1][kSub];
      if constexpr (kQ8) {
#pragma unroll
        for (int j = 0; j < kSub; ++j) {
#pragma unroll
          for (int t = 0; t < kTiles; ++t) raw[t][j] = I32x4{0, 0, 0, 0};
#pragma unroll
          for (int i = 0; i < kSteps; ++i) {
            const I32x4 a = *reinterpret_cast<const I32x4*>(k_mine + j * 16 * kRow + (k_at ^ (64u * i)));
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
              raw[t][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, qi[t][i], raw[t][j], 0, 0, 0);
            }
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < kSub; ++j) {
          F32x4 sums = F32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int i = 0; i < kSteps; ++i) {
            const Half8 a = *reinterpret_cast<const Half8*>(k_mine + j * 16 * kRow + (k_at ^ (64u * i)));
            sums = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qh[i], sums, 0, 0, 0);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) s[j][i] = (sums[i] + Ror<8>(sums[i])) * to_score[0];
        }
      }
      // ---- the next unit, and its keys
      ++u;
      const bool more = u < u_end;
      const uint32_t c_end = c + 1;
      const uint32_t piece_units = units;
      const int32_t piece_row = row, piece_pair = pair;
      bool turn = !more;  // this unit is its piece's last
      float4 ks[kMine], vs[kMine];
      if constexpr (kQ8) {
#pragma unroll
        for (int j = 0; j < kMine; ++j) ks[j] = scales_at(k_mine, mine_at + j);
      }
      // The products of queries' and keys' codes as scores: sums over the digits' columns, each of the half of the keys and
      // the tile that are the lane's. With one column tile two lanes have the same score: the sums' order gives them the
      // same bits, since each takes another digit of the weight that comes of it.
      const auto scale_scores = [&]() {
        float x[kSub][4];
#pragma unroll
        for (int j = 0; j < kSub; ++j) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float first = static_cast<float>(raw[0][j][i]) * to_score[0];
            if constexpr (kTiles == 1) {
              x[j][i] = first + Ror<8>(first);
            } else {
              const float last = static_cast<float>(raw[kTiles - 1][j][i]) * to_score[kTiles - 1];
              const float send = second ? first : last;
              x[j][i] = (second ? last : first) + Ror<4>(send);
            }
          }
        }
#pragma unroll
        for (int j = 0; j < kMine; ++j) {
          const float by[4] = {ldexpf(ks[j].x, key_exp), ldexpf(ks[j].y, key_exp), ldexpf(ks[j].z, key_exp),
                               ldexpf(ks[j].w, key_exp)};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float lo = x[j][i], hi = x[kSub - kMine + j][i];
            const float send = upper ? lo : hi;
            s[j][i] = ((upper ? hi : lo) + other_half(send)) * by[i];
          }
        }
      };
      if constexpr (kTiles > 1) scale_scores();  // before the loads and not, as below, while they run: registers
      __builtin_amdgcn_sched_barrier(0);
      if (more) {
        ++c;
        if (c == units) {
          turn = true;
          c = 0;
          if (++pair == rows.pairs) {
            pair = 0;
            do {
              ++row;
              units = row < rows.n_rows ? batch.UnitsOf(row) : 1;
            } while (units == 0);
            row = min(row, rows.n_rows - 1);  // past the last only if the lengths change while this runs
            len = batch.LenOf(row);
            table = view.pages + batch.SeqOf(row) * view.max_pages + batch.PagesOf(row);
          }
        }
        find();
        load_k();
      }
      __builtin_amdgcn_sched_barrier(0);
      // ---- weights
      if constexpr (kQ8 && kTiles == 1) scale_scores();
      if (__builtin_expect(tail || this_bad != 0, 0)) {
#pragma unroll
        for (int j = 0; j < kMine; ++j) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (this_bad >> (mine_at + j) & 1) s[j][i] = NAN;
            if (16 * (mine_at + j) + 4 * g + i >= left) s[j][i] = -INFINITY;
          }
        }
      }
      float top = m;
#pragma unroll
      for (int j = 0; j < kMine; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, s[j][i]);
      }
      if constexpr (kQ8) top = fmaxf(top, other_half(top));
      top = MaxAcrossRows(top);
      if constexpr (kQ8) {
        if (__any(top > m + 3.0f)) {  // acc stays: what it holds, relative to a larger m, is less, and so multiplied by more
          const float to = top > m + 3.0f ? top : m;
          const float safe = to == -INFINITY ? 0.0f : to;
          l *= __builtin_amdgcn_exp2f(m - safe);
          shrink *= __builtin_amdgcn_exp2f(safe - m);
          m = to;
        }
        const float safe = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int j = 0; j < kMine; ++j) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[j][i] = __builtin_amdgcn_exp2f(s[j][i] - safe);
            l += s[j][i];
          }
        }
      }
      // the values are there: the next keys' loads, if any, are younger
      if (more) {
        WaitLoads<kStageLoads>();
      } else {
        WaitLoads<0>();
      }
      // ---- the output's sums
      if constexpr (kQ8) {
#pragma unroll
        for (int j = 0; j < kMine; ++j) vs[j] = scales_at(v_mine, mine_at + j);
        if (tail) {
#pragma unroll
          for (int j = 0; j < kMine; ++j) {
            const int32_t p = 16 * (mine_at + j) + 4 * g;
            vs[j].x = p < left ? vs[j].x : 0.0f;
            vs[j].y = p + 1 < left ? vs[j].y : 0.0f;
            vs[j].z = p + 2 < left ? vs[j].z : 0.0f;
            vs[j].w = p + 3 < left ? vs[j].w : 0.0f;
          }
        }
        // weights times scales, and the head's largest of the step (as whole numbers, where a NaN is larger than any number)
        uint32_t big = 0;
#pragma unroll
        for (int j = 0; j < kMine; ++j) {
          const float by[4] = {vs[j].x, vs[j].y, vs[j].z, vs[j].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[j][i] *= by[i];
            big = max(big, __float_as_uint(s[j][i]));
          }
        }
        const auto larger = [](float a, float b) { return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b))); };
        big = __float_as_uint(AcrossRows(larger(__uint_as_float(big), other_half(__uint_as_float(big))), larger));
        l = big >= 0x7F800000u ? NAN : l;
        const float largest = __uint_as_float(big);
        // the largest is in [2^e, 2^(e + 1)): the step's are whole numbers of 2^(e - 29), less than 2^30 of them
        const uint32_t biased = min(max(big >> 23, 1u), 253u);
        const float up = __uint_as_float((254u - biased) << 23), down = __uint_as_float(biased << 23);
        if (__any(largest * shrink > 0x1p64f)) {
          const bool grew = largest * shrink > 0x1p64f;
          const float back = grew ? up * __builtin_amdgcn_rcpf(shrink) : 1.0f;
          shrink = grew ? up : shrink;
#pragma unroll
          for (int t = 0; t < kTiles; ++t) {
            const float by = of_tile(t, back);
#pragma unroll
            for (int i = 0; i < kE; ++i) acc[t][i] *= by;
          }
        }
        // a whole number of this lane's digit, in acc
        const float unit = largest > 0.0f ? down * shrink : 0.0f;
        float units[kTiles];
#pragma unroll
        for (int t = 0; t < kTiles; ++t) units[t] = of_tile(t, unit) * (digit_by * 0x1p-29f);
        I32x4 w[kTiles];  // tile j of 16 keys: bytes 4 j ..
#pragma unroll
        for (int j = 0; j < kMine; ++j) {
          float d[4];  // whole numbers, and so below
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            d[i] = __uint_as_float(static_cast<uint32_t>(static_cast<int>(fmaf(s[j][i] * up, 0x1p29f, 0.5f))) + 0x80808080u);
          }
          // this lane's digit of its own four weights, and of those of the lanes that have the others
          const auto digits = [&](auto of) {
            return Digit4(__float_as_uint(of(d[0])), __float_as_uint(of(d[1])), __float_as_uint(of(d[2])),
                          __float_as_uint(of(d[3])), digit);
          };
          const int own = digits([](float x) { return x; });
          const int half = digits(other_half);
          const int lo = upper ? half : own, hi = upper ? own : half;
          if constexpr (kTiles == 1) {
            w[0][j] = lo;
            w[0][kSub - kMine + j] = hi;
          } else {
            // of the other tile: the next copy has its lower half for copies 0 and 3, the one before for 1 and 2
            const int next = digits([](float x) { return Ror<12>(x); });
            const int last = digits([](float x) { return Ror<4>(x); });
            const int lo2 = second != upper ? last : next, hi2 = second != upper ? next : last;
            w[0][j] = second ? lo2 : lo;
            w[0][kSub - kMine + j] = second ? hi2 : hi;
            w[1][j] = second ? lo : lo2;
            w[1][kSub - kMine + j] = second ? hi : hi2;
          }
        }
        I32x2 a[kE][2];
#pragma unroll
        for (int i = 0; i < kE; ++i) {
          const char* from = v_mine + (v_at ^ (16u * i));
          a[i][0] = ReadBytesAcross(from);
          a[i][1] = ReadBytesAcross(from + 32 * kRow);
        }
#pragma unroll
        for (int i = 0; i < kE; ++i) {
          const I32x4 v = I32x4{a[i][0][0], a[i][0][1], a[i][1][0], a[i][1][1]};
#pragma unroll
          for (int t = 0; t < kTiles; ++t) {
            const I32x4 x = __builtin_amdgcn_mfma_i32_16x16x64_i8(v, w[t], I32x4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[t][i][r] = fmaf(static_cast<float>(x[r]), units[t], acc[t][i][r]);
          }
        }
      } else {
        if (tail) {  // what stands behind the last position may not even be a number
#pragma unroll
          for (int i = 0; i < kStep * kRow / 1024; ++i) {
            const int to = 1024 * i + 16 * lane;
            if (to / kRow >= left) *reinterpret_cast<uint4*>(v_mine + to) = make_uint4(0u, 0u, 0u, 0u);
          }
        }
        const float safe = top == -INFINITY ? 0.0f : top;
        const float back = __builtin_amdgcn_exp2f(m - safe);
        m = top;
        l *= back;
        if (__any(back != 1.0f)) {
#pragma unroll
          for (int i = 0; i < kE; ++i) acc[0][i] *= back;
        }
        constexpr float up = 0x1p14f;
        uint32_t pt[kSub][2];
#pragma unroll
        for (int j = 0; j < kSub; ++j) {
          float w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            w[i] = __builtin_amdgcn_exp2f(s[j][i] - safe);
            l += w[i];
          }
          pt[j][0] = Term2(w[0] * up, w[1] * up, copy != 0);
          pt[j][1] = Term2(w[2] * up, w[3] * up, copy != 0);
        }
#pragma unroll
        for (int t = 0; t < kSub / 2; ++t) {
          const Half8 b = AsHalf8(pt[2 * t][0], pt[2 * t][1], pt[2 * t + 1][0], pt[2 * t + 1][1]);
          uint2 a[kE][2];
#pragma unroll
          for (int i = 0; i < kE; ++i) {
            const char* from = v_mine + t * 32 * kRow + (v_at ^ (32u * i));
            a[i][0] = ReadHalvesAcross(from);
            a[i][1] = ReadHalvesAcross(from + 16 * kRow);
          }
#pragma unroll
          for (int i = 0; i < kE; ++i) {
            acc[0][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                AsHalf8(a[i][0].x, a[i][0].y, a[i][1].x, a[i][1].y), b, acc[0][i], 0, 0, 0);
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      if (more) load_v();
      if (!turn) continue;

      // ---- the piece's (m, l, o): out, or kept where it is not the whole of its pair
      const bool whole = c_first == 0 && c_end == piece_units;
      if (!whole) {
        const int which = more ? 0 : 1;
        if (lane == 0) pieces[wave][which] = Piece{u - c_end, c_first, c_end, piece_units, piece_row, piece_pair};
        my_held |= 1 << which;
      }
      if constexpr (kQ8) l += other_half(l);
      l = SumAcrossRows(l);
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        const float total = of_tile(t, l), top = of_tile(t, m);
        // 8-bit values: one factor after the other, since their product may be too small a number
        const float unit = kQ8 ? 1.0f / of_tile(t, shrink) : 1.0f;
        const float by = (kQ8 ? 1.0f : 0x1p-14f) / (whole ? total : 1.0f);
        const int h = t * kHeadCols + head_col;
        F32x4 own[kOwn];
#pragma unroll
        for (int i = 0; i < kE; ++i) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float x = acc[t][i][r];
            x += Ror<8>(x);
            if constexpr (kQ8) x += Ror<4>(x);
            x *= by;
            if constexpr (kQ8) x *= unit;
            own[i % kOwn][r] = i < kOwn || copy == i / kOwn ? x : own[i % kOwn][r];
          }
        }
        if (!whole && more) {
#pragma unroll
          for (int i = 0; i < kOwn; ++i) kept[t][i] = own[i];
          kept_m[t] = top;
          kept_l[t] = total;
        } else if (h < heads) {
          float* to = whole ? out + (head_row + h) * D : reinterpret_cast<float*>(v_mine) + h * kPart;
#pragma unroll
          for (int i = 0; i < kOwn; ++i) *reinterpret_cast<F32x4*>(to + 16 * (copy * kOwn + i) + 4 * g) = own[i];
          if (!whole && copy == 0 && g == 0) {
            to[D] = top;
            to[D + 1] = total;
          }
          if constexpr (kShared) {
            if (whole && copy == 0 && g == 0) StoreMl(args, head_row + h, top, total);
          }
        }
      }
      if (!more) break;
      c_first = c;
      turned = true;
    }
    // the first piece, now that its keys' place is free
    if (my_held & 1) {
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        const int h = t * kHeadCols + head_col;
        if (h < tile_heads) {  // what lies past the piece's heads is not read
          float* to = reinterpret_cast<float*>(k_mine) + h * kPart;
#pragma unroll
          for (int i = 0; i < kOwn; ++i) *reinterpret_cast<F32x4*>(to + 16 * (copy * kOwn + i) + 4 * g) = kept[t][i];
          if (copy == 0 && g == 0) {
            to[D] = kept_m[t];
            to[D + 1] = kept_l[t];
          }
        }
      }
    }
  }
  if (lane == 0) held[wave] = my_held;
  __syncthreads();

  // The workgroup's pieces in order, neighbours of one pair joined: to out where that is the whole of a pair, else (the
  // workgroup's first and last at most) to its slots in the workspace, of the outputs and then a line of (m, l).
  const auto part = [&](int i) { return reinterpret_cast<const float*>(i & 1 ? v_lds[i >> 1] : k_lds[i >> 1]); };
  const uint32_t slot_bytes = SlotBytes(D, tile_heads);
  char* const slots = workspace + kMaxGroups * kCounterBytes;
  Piece open[2];
  int n_open = 0;
  const int of_lane = lane < 2 * kWaves ? lane : 0;  // lane i has piece i % 2 of wave i / 2
  const Piece mine = pieces[of_lane >> 1][of_lane & 1];
  const bool there = lane < 2 * kWaves && (held[of_lane >> 1] >> (of_lane & 1) & 1) != 0;
  uint64_t open_lanes = __ballot(there);
  while (open_lanes != 0) {
    const int from = __builtin_ctzll(open_lanes);
    const auto field = [&](uint32_t x, int i) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(x, i)); };
    Piece run;
    run.first = field(mine.first, from);
    const uint64_t same = __ballot(there && mine.first == run.first);  // one behind the other
    run.c0 = field(mine.c0, from);
    run.c1 = field(mine.c1, 63 - __builtin_clzll(same));
    run.n = field(mine.n, from);
    run.row = static_cast<int32_t>(field(static_cast<uint32_t>(mine.row), from));
    run.pair = static_cast<int32_t>(field(static_cast<uint32_t>(mine.pair), from));
    const int list = static_cast<int>(same);
    open_lanes &= ~same;
    const HeadsOf of(run, n_heads, group, tiles, tile_heads);
    const bool whole = run.c0 == 0 && run.c1 == run.n;
    const bool leads = run.first + run.c0 == begin;  // the workgroup's first piece
    const __amdgpu_buffer_rsrc_t rs =
        dev::OutResource(slots + (2 * static_cast<int64_t>(me) + (leads ? 0 : 1)) * slot_bytes, slot_bytes);
    for (int i = threadIdx.x; i < of.heads * (D / 4); i += 64 * kWaves) {
      const int h = i / (D / 4), d = 4 * (i % (D / 4));
      float4 x[2 * kWaves];
#pragma unroll
      for (int k = 0; k < 2 * kWaves; ++k) x[k] = *reinterpret_cast<const float4*>(part(k) + h * kPart + d);
      // what the pieces in the list count for under their common maximum; none of a piece that is not in the list, whose
      // place holds anything
      float2 ml[2 * kWaves];
#pragma unroll
      for (int k = 0; k < 2 * kWaves; ++k) ml[k] = *reinterpret_cast<const float2*>(part(k) + h * kPart + D);
      float top = -INFINITY, l = 0.0f;
#pragma unroll
      for (int k = 0; k < 2 * kWaves; ++k) {
        ml[k].x = list >> k & 1 ? ml[k].x : -INFINITY;
        top = fmaxf(top, ml[k].x);
      }
      const float safe = top == -INFINITY ? 0.0f : top;
      float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int k = 0; k < 2 * kWaves; ++k) {
        if (list >> k & 1) {  // the same in every lane
          const float f = __builtin_amdgcn_exp2f(ml[k].x - safe);
          l = fmaf(ml[k].y, f, l);
          o = make_float4(fmaf(x[k].x, f, o.x), fmaf(x[k].y, f, o.y), fmaf(x[k].z, f, o.z), fmaf(x[k].w, f, o.w));
        }
      }
      if (whole) {
        if constexpr (kShared) {
          if (d == 0) StoreMl(args, of.head_row + h, top, l);
        }
        const float inv = 1.0f / l;
        dev::Store4(out + (of.head_row + h) * D + d, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
      } else {
        dev::StoreBuf4<kPartPolicy>(rs, 16u * static_cast<uint32_t>(i), o);
        if (d == 0) {
          dev::StoreBufU2<kPartPolicy>(rs, slot_bytes - kLine + 8u * h,
                                       make_uint2(__float_as_uint(top), __float_as_uint(l)));
        }
      }
    }
    if (whole) continue;
    open[n_open == 0 ? 0 : 1] = run;
    ++n_open;
  }

  // Device-scope write-through stores, acknowledged before the count: what the last workgroup of a pair to arrive then
  // reads, with device-coherent loads, is all there. No workgroup waits for another. Where a pair has more parts than
  // kJoinAtOnce, the last of each kFan joins those and counts for them.
  if (n_open > 0) {
    // which parts of their pairs they are, while the stores are under way
    Parts of_first, of_last;
#pragma unroll 1
    for (int i = 0; i < n_open; ++i) {
      const Parts of(open[i == 0 ? 0 : 1], batch, share, me);
      if (i == 0) of_first = of;
      of_last = of;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x < n_open) {  // both at once
      const Parts& of = threadIdx.x == 0 ? of_first : of_last;
      flags[threadIdx.x] = Count(workspace, of.blocks > 1 ? of.BlockCounter() : of.PairCounter(), of.block_parts);
    }
    __syncthreads();
#pragma unroll 1
    for (int i = 0; i < n_open; ++i) {
      if (!__builtin_amdgcn_readfirstlane(flags[i])) continue;
      const Piece run = open[i == 0 ? 0 : 1];
      const Parts of = i == 0 ? of_first : of_last;
      const HeadsOf heads(run, n_heads, group, tiles, tile_heads);
      const uint32_t first_leads = of.leads ? 0u : 1u;
      const __amdgpu_buffer_rsrc_t all = dev::OutResource(slots + 2 * static_cast<int64_t>(of.wa) * slot_bytes,
                                                          (2 * of.parts) * slot_bytes);
      // wa's part is in its first slot only if the pair starts where its share does
      const auto slot_of = [&](uint32_t p) { return (2u * p + (p == 0 ? first_leads : 0u)) * slot_bytes; };
      // Four elements of a head to a thread, and as many sets of threads as there are, each taking every sets-th part,
      // kBatch of them requested at a time: a round trip past the L2 costs more than the arithmetic.
      constexpr int kBatch = 8;
      const int columns = heads.heads * (D / 4);
      // whole quotients of small numbers, a half away from where the reciprocal's error would show
      const float per_set = __builtin_amdgcn_rcpf(static_cast<float>(heads.heads));
      const int sets = static_cast<int>((64 * kWaves / (D / 4) + 0.5f) * per_set);
      const int set = static_cast<int>((static_cast<float>(threadIdx.x / (D / 4)) + 0.5f) * per_set);
      const int column = static_cast<int>(threadIdx.x) - set * columns;
      const int h = column / (D / 4);
      float top, l;
      float4 o;
      const auto join = [&](float m2, float l2, float4 o2) {
        const float to = fmaxf(top, m2);
        const float safe = to == -INFINITY ? 0.0f : to;
        const float f = __builtin_amdgcn_exp2f(top - safe), f2 = __builtin_amdgcn_exp2f(m2 - safe);
        top = to;
        l = fmaf(l2, f2, l * f);
        o = make_float4(fmaf(o2.x, f2, o.x * f), fmaf(o2.y, f2, o.y * f), fmaf(o2.z, f2, o.z * f),
                        fmaf(o2.w, f2, o.w * f));
      };
      // parts p0, p0 + step, ...: the sum is in set 0
      uint32_t p0 = of.block * kFan, step = 1;
      int count = static_cast<int>(of.block_parts);
      bool done = of.blocks == 1;
#pragma unroll 1
      while (true) {
        top = -INFINITY, l = 0.0f;
        o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (set < sets) {
#pragma unroll 1
          for (int w = set; w < count; w += kBatch * sets) {
            uint2 ml[kBatch];
            float4 x[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
              if (w + k * sets < count) {
                const uint32_t at = slot_of(p0 + static_cast<uint32_t>(w + k * sets) * step);
                ml[k] = dev::LoadBufU2<dev::kLoadDevicePolicy>(all, at + slot_bytes - kLine + 8u * h);
                x[k] = dev::LoadBuf4<dev::kLoadDevicePolicy>(all, at + 16u * column);
              }
            }
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
              if (w + k * sets < count) join(__uint_as_float(ml[k].x), __uint_as_float(ml[k].y), x[k]);
            }
          }
          joins[threadIdx.x] = Join{o, top, l};
        }
        __syncthreads();
        if (set == 0) {
#pragma unroll 1
          for (int k = 1; k < min(sets, count); ++k) {
            const Join& j = joins[k * columns + column];
            join(j.m, j.l, j.o);
          }
        }
        __syncthreads();  // joins may be written again
        if (done) break;
        // a block's sum takes its first part's place, and counts
        if (set == 0) {
          const uint32_t at = slot_of(p0);
          dev::StoreBuf4<kPartPolicy>(all, at + 16u * column, o);
          if (column % (D / 4) == 0) {
            dev::StoreBufU2<kPartPolicy>(all, at + slot_bytes - kLine + 8u * h,
                                         make_uint2(__float_as_uint(top), __float_as_uint(l)));
          }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (threadIdx.x == 0) flags[i] = Count(workspace, of.PairCounter(), of.blocks);
        __syncthreads();
        if (!__builtin_amdgcn_readfirstlane(flags[i])) break;
        p0 = 0;
        step = kFan;
        count = static_cast<int>(of.blocks);
        done = true;
      }
      if (!done) continue;
      if (set == 0) {
        if constexpr (kShared) {
          if (4 * column == h * D) StoreMl(args, heads.head_row + h, top, l);
        }
        const float inv = 1.0f / l;
        dev::Store4(out + heads.head_row * D + 4 * column, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
      }
    }
  }

  // rows with nothing to attend to: zeros, or NaN where the row is out of range
  for (int64_t r = me; r < rows.n_rows; r += gridDim.x) {
    const int32_t seq = static_cast<int32_t>(batch.SeqOf(static_cast<int32_t>(r)));
    const int32_t len = batch.LenOf(static_cast<int32_t>(r));
    if (seq < 0) continue;
    const bool fine = rows.Fine(seq, len);
    if (fine && len > 0) continue;
    if constexpr (kShared) {  // a row of nothing but what it shares has zeros of no weight
      for (int32_t h = threadIdx.x; h < n_heads; h += 64 * kWaves) StoreMl(args, r * n_heads + h, -INFINITY, 0.0f);
    }
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

template <class Args>
auto* KernelFor(const GpuPagedKv& kv, int32_t tile_heads) {
  if (kv.type != kKvQ8) {
    return kv.head_dim == 128 ? PagedAttentionKernel<128, false, 1, Args> : PagedAttentionKernel<64, false, 1, Args>;
  }
  if (tile_heads > 4) {
    return kv.head_dim == 128 ? PagedAttentionKernel<128, true, 2, Args> : PagedAttentionKernel<64, true, 2, Args>;
  }
  return kv.head_dim == 128 ? PagedAttentionKernel<128, true, 1, Args> : PagedAttentionKernel<64, true, 1, Args>;
}

}  // namespace

size_t GpuAttentionPagedWorkspaceBytes(int32_t n_heads, int32_t n_kv_heads, int32_t head_dim) {
  CheckHeads("AttentionPagedWorkspace", n_heads, n_kv_heads, head_dim);
  int32_t tiles, tile_heads;
  TilesOf(n_heads / n_kv_heads, &tiles, &tile_heads);
  return kMaxGroups * (kCounterBytes + 2 * static_cast<size_t>(SlotBytes(head_dim, tile_heads)));
}

void GpuAttentionPagedWorkspaceInit(void* workspace, size_t bytes) {
  RPG_CHECK(workspace != nullptr && bytes > 0 && bytes % 16 == 0 && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0,
            "AttentionPagedWorkspaceInit: a workspace is 256-byte aligned and a multiple of 16 bytes");
  GpuStreamFill(workspace, static_cast<int64_t>(bytes), 0);
}

void AttendPaged(const GpuPagedKv& kv, const GpuPageTable& table, const int32_t* seq_ids, const int32_t* lens,
                 const float* q_dev, int32_t n_heads, int64_t n_rows, float* out_dev, void* workspace,
                 size_t workspace_bytes, PagedPrefix* prefix) {
  const char* what = prefix == nullptr ? "AttentionPaged" : "AttentionPagedShared";
  CheckPagedKv(what, kv, table);
  CheckHeads(what, n_heads, kv.n_kv_heads, kv.head_dim);
  RPG_CHECK(n_rows >= 0 && n_rows <= 0x7FFFFFFF, "%s: %lld rows", what, static_cast<long long>(n_rows));
  if (n_rows == 0) return;
  RPG_CHECK(lens != nullptr && q_dev != nullptr && out_dev != nullptr && workspace != nullptr, "%s got a null pointer",
            what);
  RPG_CHECK(seq_ids != nullptr || n_rows <= table.n_seqs, "%s: %lld rows without seq_ids, but %lld sequences", what,
            static_cast<long long>(n_rows), static_cast<long long>(table.n_seqs));
  RPG_CHECK(((reinterpret_cast<uintptr_t>(q_dev) | reinterpret_cast<uintptr_t>(out_dev)) & 15) == 0,
            "%s: q and out have to be 16-byte aligned", what);
  RPG_CHECK(((reinterpret_cast<uintptr_t>(seq_ids) | reinterpret_cast<uintptr_t>(lens)) & 3) == 0,
            "%s: seq_ids and lens have to be 4-byte aligned", what);
  const int64_t q_bytes = n_rows * n_heads * kv.head_dim * 4;
  RPG_CHECK(!Overlap(q_dev, q_bytes, out_dev, q_bytes), "%s: out must not overlap q", what);
  const size_t own = GpuAttentionPagedWorkspaceBytes(n_heads, kv.n_kv_heads, kv.head_dim);
  const size_t need = prefix == nullptr
                          ? own
                          : GpuAttentionPagedSharedWorkspaceBytes(n_heads, kv.n_kv_heads, kv.head_dim, n_rows);
  RPG_CHECK((reinterpret_cast<uintptr_t>(workspace) & 255) == 0 && workspace_bytes >= need,
            "%s: a workspace of %zu bytes, 256-byte aligned, is needed (%zu given)", what, need, workspace_bytes);
  RPG_CHECK(!Overlap(out_dev, q_bytes, workspace, static_cast<int64_t>(need)) &&
                !Overlap(q_dev, q_bytes, workspace, static_cast<int64_t>(need)),
            "%s: the workspace must not overlap q or out", what);
  int32_t tiles, tile_heads;
  TilesOf(n_heads / kv.n_kv_heads, &tiles, &tile_heads);
  const Rows rows{seq_ids, lens, static_cast<int32_t>(table.n_seqs),
                  static_cast<int32_t>(std::min<int64_t>(table.max_pages * kv.page_size, 0x7FFFFFFF)),
                  static_cast<int32_t>(n_rows), kv.n_kv_heads * tiles, kv.head_dim == 128 && kv.type == kKvF16 ? 5 : 6};
  const int64_t most = (static_cast<int64_t>(rows.capacity) >> rows.unit_shift) + 1;
  RPG_CHECK(n_rows <= 0x7FFFFFFF / most / rows.pairs,
            "%s: %lld rows of up to %lld positions and %d heads are too many for one call", what,
            static_cast<long long>(n_rows), static_cast<long long>(rows.capacity), rows.pairs);
  // no more workgroups than the longest possible rows would give work to; for a few pairs one to a compute unit, since more
  // parts of a pair cost more to join than the card gives for them, also at great lengths. With two to a compute unit instead, 8 pairs of one row in 8 bits: of 32768 positions 21.8 us against 20.5, of 131072 54.2
  // against 52.5, of 262144 97.5 against 95.1 (fp16 173 against 170); one pair of 262144 23.9 against 21.8; 15 of 32768
  // 31.2 against 29.3 (fp16 49.2 against 50.0)
  const int64_t all_pairs = n_rows * rows.pairs;
  const int64_t at_once = all_pairs * kJoinAtOnce < kMaxGroups ? kMaxGroups / 2 : kMaxGroups;
  const int64_t groups = std::min<int64_t>(at_once, all_pairs * ((most + (1 << kLeastStep) - 1) >> kLeastStep));
  const float scale_log2 =
      static_cast<float>(1.4426950408889634 / std::sqrt(static_cast<double>(kv.head_dim)));
  const AttentionArgs args{dev::ViewOf(kv, table), rows, q_dev, out_dev, static_cast<char*>(workspace), n_heads,
                           n_heads / kv.n_kv_heads, tiles, tile_heads, scale_log2};
  const dim3 grid(static_cast<unsigned>(groups)), block(64 * kWaves);
  // what a group of all rows with all of their pages would save, at the most
  if (prefix == nullptr || prefix->n_groups == 0 || (n_rows - 1) * std::min<int64_t>(table.max_pages, 0x7FFFFFFF) < prefix->least) {
    Launch("PagedAttentionKernel", KernelFor<AttentionArgs>(kv, tile_heads), grid, block, args);
    return;
  }
  CheckPrefix(kv, table, n_heads, n_rows, static_cast<char*>(workspace) + own, prefix);
  SharedAttentionArgs shared;
  static_cast<AttentionArgs&>(shared) = args;
  shared.group_rows = prefix->group_rows;
  shared.group_pages = prefix->group_pages;
  shared.n_groups = prefix->n_groups;
  shared.least = prefix->least;
  shared.ml = prefix->ml;
  Launch("PagedAttentionKernel", KernelFor<SharedAttentionArgs>(kv, tile_heads), grid, block, shared);
  AttendPrefix(kv, table, seq_ids, lens, q_dev, n_heads, n_rows, out_dev, *prefix);
}

void GpuAttentionPaged(const GpuPagedKv& kv, const GpuPageTable& table, const int32_t* seq_ids, const int32_t* lens,
                       const float* q_dev, int32_t n_heads, int64_t n_rows, float* out_dev, void* workspace,
                       size_t workspace_bytes) {
  AttendPaged(kv, table, seq_ids, lens, q_dev, n_heads, n_rows, out_dev, workspace, workspace_bytes, nullptr);
}

}  // namespace rpg
