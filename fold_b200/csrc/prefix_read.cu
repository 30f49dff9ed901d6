// Attention of a batch of sequences that share a prefix (fold_prefix_read), on tcgen05 with
// accumulators in tensor memory (TMEM), keys and values staged by TMA from the paged cache.
//
// Mathematics. Row (token t of sequence i, query head h) sees the prefix's keys and its own; with
// x_j = scale * q.k_j the result is sum_j 2^(y_j) v_j / sum_j 2^(y_j), y = x log2(e). Any split of
// the keys into ranges gives partials (o, lse) that a log-sum-exp merge joins exactly, so the
// prefix is read for the rows of ALL sequences together, each sequence's own keys for its rows.
//
// Work. The rows of one KV head and one part (the prefix with all tokens, or one sequence's own
// keys with its tokens) are packed token by token, the group's heads side by side, into row tiles
// of at most ROWS (256; 128 at head size 256) rows. An item is (row tile, KV head); its keys are
// tiles of 128. All items, prefix first, lie on one line of cost units (a constant a key tile, a
// constant an item); each of the launch's CTAs takes an equal piece of that line, so a piece may
// begin and end inside an item at a tile border (a segment). The lengths are read on the device:
// every CTA computes the same line. A segment that starts its item writes its partial to the
// rows' own places, any other to the CTA's one continuation buffer (only a CTA's first segment can
// continue an item); the item's first CTA notes which CTAs follow, and the merge kernel joins.
//
// One CTA per SM, warps with fixed roles:
//   softmax warps (one or two warpgroups): a thread owns one row; S from TMEM, mask, running
//     maximum raised lazily, P = 2^(y - m) rounded to the input type and stored over S in TMEM,
//     O in TMEM rescaled when a maximum rose; at a segment's end O / l and lse go to memory;
//   TMA warp: K and V tiles, each lane one chunk of a page, into a ring of units;
//   MMA warp: S = Q K^T and O += P V (P from TMEM), issued by one lane;
//   scheduler warp: walks the items, publishes segments in a small ring;
//   Q warp: the segments' queries, by TMA or row by row.
// Two S buffers and two O accumulators ("slots") keep the tensor cores busy while a warpgroup is
// in its softmax: a wide row tile's slots are its two halves and share each K and V tile; otherwise
// they take the key tiles in turn and are joined at the end of the segment. At head size 256 one
// accumulator fills the columns that S leaves, so one warpgroup serves both S buffers. Segments of a
// few rows go another way (FewRows) and come last on the line.
//
// Rounding. Logits, maxima, sums, O and the partials are float32; P is rounded once to the type of
// V (the MMA takes operands of one type), the sums are of the unrounded P, the result is rounded
// once. Against 64 bits that is 0.0023 (bf16) or 0.00029 (fp16) of the outputs' norm, where rounding
// the outputs alone is 0.0017 and 0.00021. In bf16, P as a high and a low part (two MMAs a tile)
// brings 0.0023 to 0.0017 and costs a quarter: 256 sequences over 32K keys 220 us for 174, 64 over 16K
// 71 for 58, prompts at head size 256 455 for 365. With value channels of eight times the size the
// largest error is 0.0013 for 0.0007 where a row's weights lie on many of 128K keys, and that of the
// result's own rounding (0.06) where they lie on few. So P stays one bf16; for more, keep the cache in
// fp16.
//
// Measured (bf16, head size 128, 32 query and 8 KV heads, pages of 16; the GPU's time of a captured
// call, the best of 15 samples of ten):
//   256 sequences of one token, 32K shared and up to 256 own keys: 175 us (788 TFLOP/s; in the long
//     run over the prefix 1160, 0.70 of the measured peak; 188 us at the clocks of a long run);
//   3 sequences of 8 tokens, 128K shared: 107 us (5.0 TB/s, 0.77 of the measured copy rate; 6 TB/s
//     behind the first 10 us);
//   64 sequences of one token, 16K shared and up to 1024 own keys: 58 us, of which the start of the
//     pipeline (lengths, line, first page, first tile) takes 8 and the merge 4.
// What bounds the wide case: with the exponentials left out it takes as long, with most of the MMAs
// left out 0.8 and without both 0.75 of the time: the K and V tiles' way from L2 into shared memory
// and the MMAs share the SM's bandwidth, and the hand-over between softmax and MMA is a chain of
// waits. Tried and dropped: exponentials by polynomial beside the special unit, P handed over in two
// halves, the tile's maximum found beside the exponentials, a second MMA warp (one a slot).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "far_read.cuh"
#include "host_common.h"
#include "tcgen05.cuh"

namespace fold {
namespace {
using namespace tc;

constexpr int TK = 128;  // keys per tile

// A row's maximum only moves when a logit passes it by more than this (log2 units); P then stays
// below 2^8 (2^15 with the fp16 shift).
constexpr float kRowRaise = 8.f;

struct PrefixParams {
  const void* q;
  int64_t q_st, q_sh;
  const int* qsl;
  const int* own_lens;
  const int* prefix_len;
  int b;
  const int* prefix_table;
  const int* tables;
  int64_t table_stride;
  int prefix_cap, own_cap;  // positions the tables can hold
  int64_t num_blocks;
  int block_size, chunk;  // chunk: rows of one TMA load, the largest power of two <= 128 dividing block_size
  int mul_b, mul_h, oob;  // plane index of (block, head) = block * mul_b + head * mul_h; oob: past the last
  int causal;
  float scale_log2;
  void* out;
  int64_t o_st, o_sh;
  float* lse;
  int n, hq, hkv, group;
  int item_cost;  // kItemCost, by head size
  int half_toks;  // tokens whose rows fill a half of a wide row tile: 128 / group
  int ctas;
  // workspace
  int4* plan;       // [2][n][hkv]: first CTA, number of CTAs, first token of the row tile
  float* o_prim;    // [2][n][hq][hd]
  float* lse_prim;  // [2][n][hq]
  float* o_cont;    // [ctas][ROWS][hd]
  float* lse_cont;  // [ctas][ROWS]
  int* err;
};

template <int HD_, class T_>
struct Cfg {
  using T = T_;
  static constexpr int HD = HD_;
  static constexpr int NWG = HD == 256 ? 1 : 2;  // softmax warpgroups = O accumulators
  static constexpr int NSW = NWG * 4;
  static constexpr int NTHREADS = (NSW + 4) * 32;  // + TMA, MMA, scheduler, Q
  static constexpr int ROWS = NWG * 128;
  static constexpr int UC = HD < 128 ? HD : 128;  // columns of a unit
  static constexpr int KU = HD / UC;              // units of a K (or V) tile
  static constexpr int NCG = UC / 64;             // 64-column groups of a unit
  static constexpr int UNIT = TK * UC * 2;
  static constexpr int Q_CG = 128 * 128;  // one 64-column group of a Q tile
  static constexpr int Q_TILE = 128 * HD * 2;
  static constexpr int QB = HD == 256 ? 1 : 2;
  static constexpr int MISC = 1024 + 2048;  // barriers, segments, scan; row statistics
  static constexpr int FIT = (kSmemLimit - MISC - QB * Q_TILE) / UNIT;
  static constexpr int NU = FIT > 12 ? 12 : FIT;
  // A wait for a unit goes by its phase's parity, so the unit NU places before it must be known to have
  // landed: else the wait may take that one's older phase for its own. A softmax warp that holds S of
  // tile j knows K up to j and V up to j - 2 landed (S of j is issued behind P V of j - 2), so of the
  // places before V of j (units from (2j + 2) KU on) only those of V of j - 1 (from 2j KU on) are open.
  // A ring of three tiles or more does not reach back to them; at head size 256 (5 units, KU 2) it
  // does, and every softmax warp waits for V of every tile.
  static constexpr bool ALL_WAIT_V = NU < 3 * KU;
  static constexpr int OFF_Q = NU * UNIT;
  static constexpr int OFF_BAR = OFF_Q + QB * Q_TILE;
  static constexpr int OFF_STAT = OFF_BAR + 1024;
  static constexpr int SMEM = OFF_BAR + MISC;
  static constexpr int TMEM_S = 0, TMEM_O = 256, TMEM_COLS = 512;
  static constexpr bool F16 = sizeof(T) == 2 && !std::is_same<T, __nv_bfloat16>::value;
  // fp16 keeps P in [2^-24, 2^15): scaled up by 2^7 so that small weights stay above its smallest step
  static constexpr float SHIFT = F16 ? 7.f : 0.f;
  static_assert(NU >= 4 && SMEM <= kSmemLimit, "shared memory");
};

// Cost units of the line, from the CTAs' finishing times at decode, prompt and draft shapes: about
// 0.3 us, an eighth of a key tile of a wide row tile. A tile of up to 128 rows takes 6, of few rows 4;
// an item costs its Q, its first keys' way through the pipeline and its partial besides (at head size
// 256, where one Q tile and one accumulator hold nothing ready, more: prompts of 90 to 700 tokens behind
// 8K keys took 416 us with 12, 391 with 16, 354 with 20, 364 with 24; of few rows, where two are under
// way at a time, less: with 6 for 3 the 256 sequences over 32K keys took 184 us, with 2 183, with 3 174).
// Head size 64 takes the same 12 as 128: drafted blocks 29.3, 29.6, 29.7, 30.3 us with 8, 12, 18, 24, those
// prompts 259, 249, 246, 248, 96 single rows over 3000 keys 33.3, 31.4, 31.0, 31.2.
constexpr int kWideTileCost = 8, kTileCost = 6, kFewTileCost = 4;
constexpr int kItemCost = 12, kItemCost256 = 20, kFewItemCost = 3;

struct Seg {
  int part;  // 0: prefix, 1: own keys, -1: no more work
  int seq, head, tok0, ntok;
  int kb, ke;   // key tiles [kb, ke)
  int limit;    // keys any row of the item sees
  int lim0, lim_step;  // row of token tok0 + x sees min(limit, lim0 + x * lim_step) keys
  int pad[2];
};
constexpr int kSegs = 4;

// Registers a thread of a block with two softmax warpgroups: at launch (384 threads; the build checks
// it), then of the softmax warps and of the others.
constexpr int kLaunchRegs = 168, kSoftmaxRegs = 208, kOtherRegs = 88;
static_assert(2 * kSoftmaxRegs + kOtherRegs <= 3 * kLaunchRegs, "a share that is not there is waited for");

// The line may be cut where the few rows begin if either side has this many CTAs.
constexpr int kCutCtas = 16;
// No piece is shorter, nor, by a rounded number of CTAs on a side of that cut, shorter than the
// longest tile: then no CTA between an item's first and last is without a tile of it, and its
// partials are those of consecutive CTAs. Eight sequences' own keys alone (64 items): 16.8 us, with
// pieces of 18 units at least 18.7.
constexpr int kMinPiece = 10;
static_assert(kMinPiece * (kCutCtas - 1) / kCutCtas >= kWideTileCost, "a tile a piece");
// Segments of up to this many rows are read by the softmax warps themselves (FewRows).
constexpr int kFewRows = 16;

// Q of up to this many rows is copied row by row (cp.async), of more as one TMA box of the half tile,
// which always moves all of its rows: 32 KB at head size 128, for 4 rows of a decode step half as much
// again as a short sequence's keys. Row by row a warp copies two rows a round.
constexpr int kFewQRows = 32;

struct Bars {
  uint64_t full[12], empty[12];
  uint64_t s_full[2], p_full[2], pv_done;
  uint64_t q_full[2], q_empty[2];
  uint64_t seg_full[kSegs], seg_empty[kSegs];
  uint64_t seg_done[2], o_free[2], stat_full, stat_free, drained, meet, few_meet[2], few_turn;
  uint32_t tmem;
  int start_seq[2];
  int64_t start_base[2];
  int64_t scan[2][12];
  Seg seg[kSegs];
};
static_assert(sizeof(Bars) <= 1024, "barriers fit their place");

// ---------------------------------------------------------------- the line of work
__device__ __forceinline__ int capped(int len, int cap, int* err) {
  if (len > cap) {
    set_error(err, FOLD_DEVERR_CAPACITY);
    len = cap;
  }
  return max(len, 0);
}

__device__ __forceinline__ int tile_cost(const PrefixParams& p, int ntok) {
  return ntok * p.group <= kFewRows ? kFewTileCost : ntok > p.half_toks ? kWideTileCost : kTileCost;
}

// Query rows of sequence s, [first, last), kept inside [0, n] whatever qsl holds.
__device__ __forceinline__ void seq_rows(const PrefixParams& p, int s, int& first, int& last) {
  first = min(max(__ldg(p.qsl + s), 0), p.n);
  last = min(max(__ldg(p.qsl + s + 1), first), p.n);
}

// The own-keys item of tokens [tok0, tok0 + ntok) of a sequence (rows [first, last), m own keys).
__device__ __forceinline__ void own_limits(const PrefixParams& p, int first, int last, int m, int tok0, int ntok,
                                           int& limit, int& lim0) {
  lim0 = p.causal ? m - (last - tok0) + 1 : m;
  limit = p.causal ? max(min(m, lim0 + ntok - 1), 0) : m;
}

// Division of non-negative values, in 32 bits where they fit.
__device__ __forceinline__ int64_t quot(int64_t a, int64_t b) {
  return ((a | b) >> 32) == 0 ? static_cast<uint32_t>(a) / static_cast<uint32_t>(b) : a / b;
}

__device__ __forceinline__ int start_cost(const PrefixParams& p, int ntok) {
  return ntok * p.group <= kFewRows ? kFewItemCost : p.item_cost;
}
__device__ __forceinline__ int64_t item_cost(const PrefixParams& p, int tiles, int ntok) {
  return tiles == 0 ? 2 : start_cost(p, ntok) + static_cast<int64_t>(tiles) * tile_cost(p, ntok);
}

// Cost of the own items of sequence s and one KV head: of many rows, and of few.
template <class C>
__device__ __forceinline__ void seq_cost(const PrefixParams& p, int s, int per_tile, int64_t (&cost)[2]) {
  int first, last;
  seq_rows(p, s, first, last);
  const int m = capped(__ldg(p.own_lens + s), p.own_cap, p.err);
  cost[0] = cost[1] = 0;
  for (int t0 = first; t0 < last; t0 += per_tile) {
    const int nt = min(per_tile, last - t0);
    int limit, lim0;
    own_limits(p, first, last, m, t0, nt, limit, lim0);
    cost[nt * p.group <= kFewRows] += item_cost(p, (limit + TK - 1) / TK, nt);
  }
}

// ---------------------------------------------------------------- loads, stores and conversions of this kernel
// Eight floats to a 32-byte boundary, one whole sector.
__device__ __forceinline__ void store8(float* dst, const float* v) {
  asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst), "f"(v[0]), "f"(v[1]), "f"(v[2]),
               "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}
__device__ __forceinline__ void tma_load_5d(void* dst, const CUtensorMap* map, uint64_t* bar, int c2, int c3, int c4) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %3, %4, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(0), "r"(c2), "r"(c3), "r"(c4)
      : "memory");
}
template <class T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  return pack_bf16(lo, hi);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  return pack_f16_sat(lo, hi);
}

// Ring position (in tiles' K or V) of K and V of the CTA's tile j, counted over all its segments:
// K runs one tile ahead, K0 K1 V0 K2 V1 ..., the order in which the MMAs first need them.
__device__ __forceinline__ uint32_t k_pos(uint32_t j) { return j == 0 ? 0 : 2 * j - 1; }
__device__ __forceinline__ uint32_t v_pos(uint32_t j) { return 2 * j + 2; }

// ---------------------------------------------------------------- segments of few rows
// A row tile of at most kFewRows rows (a decode step's, whose keys are read once for a handful of
// rows) would leave most of the 128 lanes of S idle and pay for the way through the MMA warp. The
// softmax warps take such segments themselves with mma.sync, a warpgroup every other one: each of its
// four warps owns 32 keys of every tile and keeps rows x keys and rows x hd fragments in registers
// (S = Q K^T, its C fragments are the A fragments of P V), with a maximum, sum and O of its own, so
// that no warp waits for another until the segment's end, where the warps' partials are joined
// through the Q tile. A short segment is a chain of latencies (Q, K, V, two meetings of the warps, the
// partial), which the other group's segment fills: 2048 segments of 4 rows and 1 to 256 keys take 52 us,
// by both groups together 58, by the MMA warp's way 82. Memory bound: the ring's units are all in
// flight (one row over 200K keys: 137 us, 6.0 TB/s). 17 to 32 rows took 2.5 us a tile here against 1.7;
// the joining deferred behind the next segment's first tile was slower.
template <class C>
struct FewRows {
  static constexpr int HD = C::HD, GW = 4, KW = TK / GW;  // warps of a group, keys of a tile a warp owns
  using T = typename C::T;
  const PrefixParams& p;
  const Seg& s;
  Bars& B;
  unsigned char* smem;
  float2* stats;
  const int group, warp, lane, cta;  // warp: of the group
  const uint32_t tile0, qu;
  uint32_t meets;    // of this group's warps so far
  const uint32_t index;  // of the segment among those of few rows

  // The group's warps, with a bounded wait.
  __device__ __forceinline__ bool meet() {
    __syncwarp();
    if (lane == 0) mbar_arrive(&B.few_meet[group]);
    return warp_wait(&B.few_meet[group], meets++ & 1);
  }
  __device__ __forceinline__ static void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (C::F16) mma_f16(d, a[0], a[1], a[2], a[3], b0, b1);
    else mma_bf16(d, a[0], a[1], a[2], a[3], b0, b1);
  }

  __device__ __forceinline__ bool run() {
    constexpr int MT = kFewRows / 16;
    const int ntile = s.ke - s.kb, rows = s.ntok * p.group;
    const int g = lane >> 2, t4 = lane & 3, mi = lane >> 3, mr = lane & 7;  // fragment row, column; ldmatrix
    const uint32_t qslot = qu % C::QB;
    // the other group has the last tile of the segment before: every earlier unit of the ring has
    // landed, so that a wait for this segment's units cannot take an older phase for theirs
    if (C::NWG == 2 && index > 0 && !warp_wait(&B.few_turn, (index - 1) & 1)) return false;
    if (!warp_wait(&B.q_full[qslot], (qu / C::QB) & 1)) return false;
    const uint32_t base = smem_u32(smem), qt = base + C::OFF_Q + qslot * C::Q_TILE;
    auto q_frag = [&](int mt, int kk, uint32_t (&a)[4]) {
      const int r = mt * 16 + (mi & 1) * 8 + mr, c = 2 * kk + (mi >> 1);
      ldsm_x4(qt + (c >> 3) * C::Q_CG + r * 128 + (((c & 7) ^ mr) << 4), a[0], a[1], a[2], a[3]);
    };
    constexpr bool HOLD = MT == 1 && HD <= 128;  // Q stays in registers
    uint32_t qf[HOLD ? HD / 16 : 1][4];
    if constexpr (HOLD) {
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk) q_frag(0, kk, qf[kk]);
    }
    float o[MT][HD / 8][4], m[MT][2], l[MT][2];
    int lim[MT][2];
    bool in[MT][2];
    int low = 0x7fffffff;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = mt * 16 + e * 8 + g;
        in[mt][e] = r < rows;
        lim[mt][e] = in[mt][e] ? min(s.limit, s.lim0 + (r / p.group) * s.lim_step) : 0;
        if (in[mt][e]) low = min(low, lim[mt][e]);
        m[mt][e] = -INFINITY, l[mt][e] = 0.f;
      }
    low = __reduce_min_sync(0xffffffffu, low);  // keys that every row sees
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int c = 0; c < HD / 8; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[mt][c][e] = 0.f;

    for (int j = 0; j < ntile; ++j) {
      const int key0 = (s.kb + j) * TK;
      const uint32_t ku = k_pos(tile0 + j) * C::KU, vu = v_pos(tile0 + j) * C::KU;
#pragma unroll
      for (int w = 0; w < C::KU; ++w)
        if (!warp_wait(&B.full[(ku + w) % C::NU], ((ku + w) / C::NU) & 1)) return false;
      constexpr int KG = KW / 16;  // groups of 16 keys
      const int row0 = warp * KW;  // this warp's first key of the tile
      const bool any = key0 + row0 < s.limit;
      uint32_t pa[KG][MT][4];
      if (any) {
        float x[KG][MT][2][4];
#pragma unroll
        for (int i = 0; i < KG * MT * 8; ++i) (&x[0][0][0][0])[i] = 0.f;
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          const uint32_t unit = base + ((ku + kk * 16 / C::UC) % C::NU) * C::UNIT;
          const int c = (2 * kk + (mi & 1)) % (C::UC / 8);
          uint32_t a[MT][4];
          if constexpr (!HOLD) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) q_frag(mt, kk, a[mt]);
          }
#pragma unroll
          for (int kg = 0; kg < KG; ++kg) {
            uint32_t b[4];
            ldsm_x4(unit + (((row0 + kg * 16) >> 3) + (mi >> 1)) * C::NCG * 1024 + (c >> 3) * 1024 + mr * 128 +
                        (((c & 7) ^ mr) << 4),
                    b[0], b[1], b[2], b[3]);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              mma(x[kg][mt][0], HOLD ? qf[HOLD ? kk : 0] : a[mt], b[0], b[1]);
              mma(x[kg][mt][1], HOLD ? qf[HOLD ? kk : 0] : a[mt], b[2], b[3]);
            }
          }
        }
        if (key0 + row0 + KW > low) {
#pragma unroll
          for (int kg = 0; kg < KG; ++kg)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (key0 + row0 + kg * 16 + (e >> 2) * 8 + 2 * t4 + (e & 1) >= lim[mt][(e >> 1) & 1])
                  x[kg][mt][e >> 2][e & 3] = -INFINITY;
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          float f[2] = {1.f, 1.f};
          bool up = false;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float top = -INFINITY;
#pragma unroll
            for (int kg = 0; kg < KG; ++kg)
#pragma unroll
              for (int n = 0; n < 2; ++n) top = fmax3(top, x[kg][mt][n][2 * e], x[kg][mt][n][2 * e + 1]);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2)) * p.scale_log2;
            const bool raise = in[mt][e] && (top > m[mt][e] + kRowRaise || (m[mt][e] == -INFINITY && top > m[mt][e]));
            if (raise) f[e] = fast_exp2(m[mt][e] - top), m[mt][e] = top;
            up |= raise;
          }
          if (__any_sync(0xffffffffu, up)) {
            l[mt][0] *= f[0], l[mt][1] *= f[1];
#pragma unroll
            for (int c = 0; c < HD / 8; ++c) o[mt][c][0] *= f[0], o[mt][c][1] *= f[0], o[mt][c][2] *= f[1], o[mt][c][3] *= f[1];
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float neg = m[mt][e] == -INFINITY ? 0.f : C::SHIFT - m[mt][e];
#pragma unroll
            for (int kg = 0; kg < KG; ++kg)
#pragma unroll
              for (int n = 0; n < 2; ++n) {
                const float a = fast_exp2(fmaf(x[kg][mt][n][2 * e], p.scale_log2, neg));
                const float d = fast_exp2(fmaf(x[kg][mt][n][2 * e + 1], p.scale_log2, neg));
                l[mt][e] += a + d;
                pa[kg][mt][2 * n + e] = pack2<T>(a, d);
              }
          }
        }
      }
      __syncwarp();
      if (lane == 0) {  // K goes back before V is waited for: the ring need not hold both
#pragma unroll
        for (int w = 0; w < C::KU; ++w) mbar_arrive_n(&B.empty[(ku + w) % C::NU], C::NWG);
      }
#pragma unroll
      for (int w = 0; w < C::KU; ++w)
        if (!warp_wait(&B.full[(vu + w) % C::NU], ((vu + w) / C::NU) & 1)) return false;
      if (j + 1 == ntile) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&B.few_turn);
      }
      if (any) {
        // slots past the limit may hold anything (NaN included): this warp's rows of them become zeros
        const int seen = s.limit - key0 - row0;
        if (seen < KW) {
#pragma unroll
          for (int w = 0; w < C::KU; ++w) {
            unsigned char* vt = smem + ((vu + w) % C::NU) * C::UNIT;
            for (int e = lane; e < (KW - seen) * C::NCG * 8; e += 32) {
              const int r = row0 + seen + e / (C::NCG * 8), c = e % (C::NCG * 8);
              *reinterpret_cast<uint4*>(vt + (r >> 3) * C::NCG * 1024 + (c >> 3) * 1024 + (r & 7) * 128 + (c & 7) * 16) =
                  make_uint4(0, 0, 0, 0);
            }
          }
          fence_proxy_async();  // the unit is loaded again by TMA
          __syncwarp();
        }
#pragma unroll
        for (int c = 0; c < HD / 16; ++c) {
          const uint32_t unit = base + ((vu + c * 16 / C::UC) % C::NU) * C::UNIT;
          const int cc = (2 * c + (mi >> 1)) % (C::UC / 8);
#pragma unroll
          for (int kg = 0; kg < KG; ++kg) {
            uint32_t b[4];
            ldsm_x4_t(unit + (((row0 + kg * 16) >> 3) + (mi & 1)) * C::NCG * 1024 + (cc >> 3) * 1024 + mr * 128 +
                          (((cc & 7) ^ mr) << 4),
                      b[0], b[1], b[2], b[3]);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              mma(o[mt][2 * c], pa[kg][mt], b[0], b[1]);
              mma(o[mt][2 * c + 1], pa[kg][mt], b[2], b[3]);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) {
#pragma unroll
        for (int w = 0; w < C::KU; ++w) mbar_arrive_n(&B.empty[(vu + w) % C::NU], C::NWG);
      }
    }

    // ---- the warps' partials joined, eight rows at a time, in the Q tile's memory
    float* scratch = reinterpret_cast<float*>(smem + C::OFF_Q + qslot * C::Q_TILE);  // [warp][8 rows][HD]
#pragma unroll
    for (int h = 0; h < 2 * MT; ++h) {
      if (h * 8 >= rows) break;
      const int mt = h >> 1, e = h & 1, nr = min(8, rows - h * 8);
      if (!meet()) return false;  // Q, or the last eight rows, have been read
      float ls = l[mt][e];
      ls += __shfl_xor_sync(0xffffffffu, ls, 1);
      ls += __shfl_xor_sync(0xffffffffu, ls, 2);
      if (t4 == 0) stats[(group * GW + warp) * 8 + g] = make_float2(m[mt][e], ls);
      if (g < nr) {
#pragma unroll
        for (int c = 0; c < HD / 8; ++c)
          *reinterpret_cast<float2*>(scratch + (warp * 8 + g) * HD + c * 8 + 2 * t4) =
              make_float2(o[mt][c][2 * e], o[mt][c][2 * e + 1]);
      }
      if (!meet()) return false;
      for (int r = warp; r < nr; r += GW) {
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < GW; ++w) top = fmaxf(top, stats[(group * GW + w) * 8 + r].x);
        const float mz = top == -INFINITY ? 0.f : top;
        float f[GW], sum = 0.f;
#pragma unroll
        for (int w = 0; w < GW; ++w) {
          const float2 a = stats[(group * GW + w) * 8 + r];
          f[w] = fast_exp2(a.x - mz), sum += f[w] * a.y;
        }
        const bool some = sum > 0.f;
        const float inv = some ? 1.f / sum : 0.f;
        const int row = h * 8 + r, x = row / p.group;
        const int64_t prim = (static_cast<int64_t>(s.part) * p.n + s.tok0 + x) * p.hq + s.head * p.group + row - x * p.group;
        const int64_t cont = static_cast<int64_t>(cta) * C::ROWS + row;
        float* od = s.kb == 0 ? p.o_prim + prim * HD : p.o_cont + cont * HD;
        for (int c = lane * 4; c < HD; c += 128) {
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < GW; ++w) {
            const float4 v = *reinterpret_cast<const float4*>(scratch + (w * 8 + r) * HD + c);
            acc.x += f[w] * v.x, acc.y += f[w] * v.y, acc.z += f[w] * v.z, acc.w += f[w] * v.w;
          }
          // no key: 0; a NaN sum reaches the output
          *reinterpret_cast<float4*>(od + c) = some ? make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv)
                                                    : make_float4(sum, sum, sum, sum);
        }
        if (lane == 0)
          (s.kb == 0 ? p.lse_prim + prim : p.lse_cont + cont)[0] =
              some ? (top - C::SHIFT + __log2f(sum)) * kLn2 : (sum == 0.f ? -INFINITY : sum);
      }
    }
    fence_proxy_async();  // the Q tile may be loaded by TMA next
    __syncwarp();
    if (lane == 0) mbar_arrive_n(&B.q_empty[qslot], C::NWG);
    return true;
  }
};

// ---------------------------------------------------------------- the kernel
template <class C>
__global__ void __launch_bounds__(C::NTHREADS, 1)
    prefix_read_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                       const __grid_constant__ CUtensorMap vmap, const PrefixParams p) {
  constexpr int HD = C::HD, KU = C::KU, NU = C::NU, NWG = C::NWG, NSW = C::NSW, QB = C::QB;
  using T = typename C::T;
  extern __shared__ __align__(1024) unsigned char smem[];
  Bars& B = *reinterpret_cast<Bars*>(smem + C::OFF_BAR);
  float2* stats = reinterpret_cast<float2*>(smem + C::OFF_STAT);  // [slot][row]: maximum, sum
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int per_tile = NWG * p.half_toks;  // tokens of a full row tile

  if (warp == NSW) {
    if (lane == 0) {
      for (int i = 0; i < NU; ++i) mbar_init(&B.full[i], 1), mbar_init(&B.empty[i], NSW);
      for (int i = 0; i < 2; ++i) {
        mbar_init(&B.s_full[i], 1), mbar_init(&B.p_full[i], 4);
        mbar_init(&B.q_full[i], 1), mbar_init(&B.q_empty[i], NSW);
        mbar_init(&B.seg_done[i], 1), mbar_init(&B.o_free[i], NSW);
      }
      for (int i = 0; i < kSegs; ++i) mbar_init(&B.seg_full[i], 1), mbar_init(&B.seg_empty[i], 3 + NSW);
      mbar_init(&B.pv_done, 1), mbar_init(&B.stat_full, NSW), mbar_init(&B.stat_free, NSW);
      mbar_init(&B.drained, 1), mbar_init(&B.meet, NSW);
      mbar_init(&B.few_meet[0], 4), mbar_init(&B.few_meet[1], 4), mbar_init(&B.few_turn, 4);
      fence_mbar_init();
    }
    __syncwarp();
  } else if (warp == NSW + 1) {
    tmem_alloc(&B.tmem, C::TMEM_COLS);
    tmem_relinquish();
  }
  wait_for_producer();

  // ---- the line: items of many rows, then items of few; of each the prefix's before the sequences'
  const int tok_lo = min(max(__ldg(p.qsl), 0), p.n), tok_hi = min(max(__ldg(p.qsl + p.b), tok_lo), p.n);
  const int plen = capped(__ldg(p.prefix_len), p.prefix_cap, p.err);
  const int ptiles = (plen + TK - 1) / TK;
  const int prow_tiles = plen > 0 ? (tok_hi - tok_lo + per_tile - 1) / per_tile : 0;
  const int last_tok = prow_tiles ? tok_hi - tok_lo - (prow_tiles - 1) * per_tile : 0;
  const int64_t pc_full = item_cost(p, ptiles, per_tile), pc_last = item_cost(p, ptiles, last_tok);
  const bool last_few = last_tok * p.group <= kFewRows;  // only the last row tile can be of few rows
  const int64_t pfull = prow_tiles ? (prow_tiles - 1) * pc_full * p.hkv : 0, plast = prow_tiles ? pc_last * p.hkv : 0;
  const int per_thread = (p.b + C::NTHREADS - 1) / C::NTHREADS;
  const int s_lo = min(tid * per_thread, p.b), s_hi = min(s_lo + per_thread, p.b);
  int64_t mine[2] = {0, 0}, incl[2];
  for (int s = s_lo; s < s_hi; ++s) {
    int64_t c[2];
    seq_cost<C>(p, s, per_tile, c);
    mine[0] += c[0] * p.hkv, mine[1] += c[1] * p.hkv;
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    incl[k] = mine[k];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, incl[k], o);
      if (lane >= o) incl[k] += y;
    }
    if (lane == 31) B.scan[k][warp] = incl[k];
  }
  tc_fence_before();
  __syncthreads();  // barriers, TMEM address and warp sums are visible
  tc_fence_after();
  int64_t own_total[2] = {0, 0}, excl[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    excl[k] = incl[k] - mine[k];
#pragma unroll
    for (int w = 0; w < C::NTHREADS / 32; ++w) {
      if (w < warp) excl[k] += B.scan[k][w];
      own_total[k] += B.scan[k][w];
    }
  }
  // where on the line the prefix's and the sequences' items of either kind begin
  const int64_t from_own[2] = {pfull + (last_few ? 0 : plast),
                               pfull + plast + own_total[0]};
  const int64_t from_last = last_few ? pfull + own_total[0] : pfull;
  const int64_t total = from_own[1] + own_total[1];
  const int ctas = static_cast<int>(max64(1, min64(p.ctas, total / kMinPiece)));
  // CTAs 2i and 2i+1 run on neighbouring SMs, and one that reads few rows beside one with many slows
  // both (the wide one's key tiles by a third, and the call waited for it: 183 us against 174 at 256
  // sequences over 32K keys). So where both kinds have CTAs enough for it to cost little, the line is
  // cut where the few rows begin, with an even number of CTAs before the cut.
  const int64_t many = last_few ? from_last : from_own[1];
  int before = (static_cast<int>(quot(many * ctas, max64(total, 1))) + 1) & ~1;
  if (before < kCutCtas || ctas - before < kCutCtas) before = 0;
  const int64_t cut_x = before ? many : 0;
  const int64_t each[2] = {before ? quot(cut_x, before) : 0, quot(total - cut_x, ctas - before)};
  const uint32_t rest[2] = {static_cast<uint32_t>(cut_x - each[0] * before),
                            static_cast<uint32_t>(total - cut_x - each[1] * (ctas - before))};
  auto cut = [&](int c) {  // where CTA c's piece begins
    if (c < before) return each[0] * c + rest[0] * static_cast<uint32_t>(c) / static_cast<uint32_t>(before);
    const uint32_t x = c - before;
    return cut_x + each[1] * x + rest[1] * x / static_cast<uint32_t>(ctas - before);
  };
  const int cta = blockIdx.x;
  const int64_t x0 = cta < ctas ? cut(cta) : total, x1 = cta < ctas ? cut(cta + 1) : total;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int64_t own_x = max64(x0 - from_own[k], 0);  // where this CTA's piece of them starts
    if (mine[k] > 0 && own_x >= excl[k] && own_x < excl[k] + mine[k]) {
      int64_t at = excl[k];
      int s = s_lo;
      for (; s + 1 < s_hi; ++s) {  // the thread's last one needs no look
        int64_t c[2];
        seq_cost<C>(p, s, per_tile, c);
        if (own_x < at + c[k] * p.hkv) break;
        at += c[k] * p.hkv;
      }
      B.start_seq[k] = s, B.start_base[k] = at;
    }
  }
  __syncthreads();
  const uint32_t tmem = B.tmem;
  release_dependents();  // the merge may be scheduled; it waits for this grid to complete

  // Every role walks the segments in the scheduler's order.
  auto few_rows = [&](const Seg& s) { return s.ntok * p.group <= kFewRows; };
  auto next_seg = [&](int sg, Seg& s) {
    if (!warp_wait(&B.seg_full[sg % kSegs], (sg / kSegs) & 1)) return false;
    s = B.seg[sg % kSegs];
    __syncwarp();
    if (lane == 0) mbar_arrive(&B.seg_empty[sg % kSegs]);
    return true;
  };

  // With two softmax warpgroups the launch's registers are dealt out again: a softmax thread holds a row
  // of S (128 values).
  if (warp < NSW) {
    if constexpr (NWG == 2) regs_up<kSoftmaxRegs>();
    // ------------------------------------------------------------ softmax warps
    const int wg = warp >> 2, row = (warp & 3) * 32 + lane;  // row of the slot = TMEM lane
    const uint32_t lane_addr = static_cast<uint32_t>((warp & 3) * 32) << 16;
    uint32_t scnt[2] = {0, 0};  // S tiles read per buffer
    uint32_t step0 = 0, tile0 = 0;  // steps and tiles of the CTA's earlier segments
    uint32_t done = 0;          // segments this warpgroup had steps of
    uint32_t qu = 0;            // Q tiles of earlier segments
    int few_from = -1;          // the first segment of few rows
    Seg few_seg{};
    uint32_t joins = 0;         // segments whose two slots were joined
    bool ok = true;
    for (int sg = 0; ok; ++sg) {
      Seg s;
      ok = next_seg(sg, s);
      if (!ok || s.part < 0) break;
      if (few_rows(s)) {
        few_from = sg, few_seg = s;
        break;
      }
      const int ntile = s.ke - s.kb;
      const bool wide = s.ntok > p.half_toks;
      const bool joined = NWG == 2 && !wide && ntile > 1;  // both slots hold every row's keys
      // this warpgroup's first step of the segment: its row half, or its first tile
      const int mine0 = NWG == 2 ? (wg ^ step0) & 1 : 0;
      const int half = wide ? mine0 : 0;
      const int tok_first = half * p.half_toks;  // first token of this warpgroup's rows
      const bool live = row < min(s.ntok - tok_first, p.half_toks) * p.group;
      const int xr = row / p.group, x = live ? tok_first + xr : 0;
      const int lim = live ? min(s.limit, s.lim0 + x * s.lim_step) : 0;
      const bool warp_live = __any_sync(0xffffffffu, live);
      const int warp_lim = __reduce_min_sync(0xffffffffu, live ? lim : 0x7fffffff);
      float m = -INFINITY, l = 0.f;
      bool empty_o = true;
      for (int j = (NWG == 2 && !wide) ? mine0 : 0; j < ntile; j += (NWG == 2 && !wide) ? 2 : 1) {
        const int b = NWG == 2 ? wg : (step0 + j) & 1;
        ok = warp_wait(&B.s_full[b], scnt[b] & 1);
        ++scnt[b];
        if (!ok) break;
        tc_fence_after();
        const uint32_t sa = tmem + C::TMEM_S + b * TK + lane_addr;
        const int key0 = (s.kb + j) * TK;
        if (warp_live) {
          float v[TK];
#pragma unroll
          for (int c = 0; c < TK; c += 32) tmem_ld32(sa + c, v + c);
          tmem_wait_ld();
          if (key0 + TK > warp_lim) {
            const int seen = lim - key0;
#pragma unroll
            for (int c = 0; c < TK; ++c) v[c] = c < seen ? v[c] : -INFINITY;
          }
          float mx[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
          for (int c = 4; c < TK; c += 8) {
#pragma unroll
            for (int k = 0; k < 4; ++k) mx[k] = c + 4 + k < TK ? fmax3(mx[k], v[c + k], v[c + 4 + k]) : fmaxf(mx[k], v[c + k]);
          }
          const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale_log2;
          const bool raise = top > m + kRowRaise || (m == -INFINITY && top > m);
          if (__any_sync(0xffffffffu, raise)) {
            const float mn = raise ? top : m;
            const float f = raise ? fast_exp2(m - mn) : 1.f;  // 0 for the first keys
            l *= f, m = mn;
            if (!empty_o) {
              // the accumulator holds the products up to the slot's last tile; with one
              // accumulator the last tile's may still be running (those before it are complete with S
              // of this tile, so the parity can stand for the last tile's phase only)
              if (NWG == 1) ok = warp_wait(&B.pv_done, (tile0 + j - 1) & 1);
              if (!ok) break;
              tc_fence_after();
              const uint32_t oa = tmem + C::TMEM_O + (NWG == 2 ? wg * HD : 0) + lane_addr;
#pragma unroll 1
              for (int c = 0; c < HD; c += 16) {
                float o[16];
                tmem_ld16(oa + c, o);
#pragma unroll
                for (int k = 0; k < 16; ++k) o[k] *= f;
                tmem_st16(oa + c, reinterpret_cast<const uint32_t*>(o));
              }
            }
          }
          const float neg = m == -INFINITY ? 0.f : C::SHIFT - m;
          float l0 = 0.f, l1 = 0.f;
#pragma unroll
          for (int c = 0; c < TK; c += 32) {
            uint32_t w[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              float a = v[c + 2 * k], d = v[c + 2 * k + 1];
              ffma2(a, d, p.scale_log2, neg, neg);
              a = fast_exp2(a), d = fast_exp2(d);
              fadd2(l0, l1, l0, l1, a, d);
              w[k] = pack2<T>(a, d);
            }
            tmem_st16(sa + c / 2, w);
          }
          l += l0 + l1;
          tmem_wait_st();
        }
        empty_o = false;
        // slots of the last page past the limit may hold anything (NaN included): their V rows
        // become zeros before the tensor cores read them
        const int vk = s.limit - key0;
        const bool rest = vk < TK && vk % p.chunk != 0 && (!wide || mine0 == 0);
        if (C::ALL_WAIT_V || rest || (warp & 3) == 0) {  // V has landed when the MMA warp gets P
          const uint32_t u = v_pos(tile0 + j) * KU;
#pragma unroll
          for (int w = 0; w < KU; ++w) ok = ok && warp_wait(&B.full[(u + w) % NU], ((u + w) / NU) & 1);
          if (!ok) break;
        }
        if (rest) {
          const int vend = (vk / p.chunk + 1) * p.chunk;
          const uint32_t u = v_pos(tile0 + j) * KU;
#pragma unroll
          for (int w = 0; w < KU; ++w) {
            unsigned char* vt = smem + ((u + w) % NU) * C::UNIT;
            for (int e = row; e < (vend - vk) * C::NCG * 8; e += 128) {
              const int vr = vk + e / (C::NCG * 8), c = e % (C::NCG * 8);
              *reinterpret_cast<uint4*>(vt + (vr >> 3) * C::NCG * 1024 + (c >> 3) * 1024 + (vr & 7) * 128 +
                                        (c & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
          }
          fence_proxy_async();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&B.p_full[b]);
      }
      if (!ok) break;
      tile0 += ntile, step0 += wide ? 2 * ntile : ntile, qu += wide ? 2 : 1;
      if (NWG == 2 && !wide && ntile == 1 && mine0 == 1) continue;  // the other slot's segment

      // ---- the segment's partial: O / l and lse
      ok = warp_wait(&B.seg_done[NWG == 2 ? wg : 0], done++ & 1);
      if (!ok) break;
      tc_fence_after();
      float ws[2] = {1.f, 0.f};
      if (joined) {
        if (joins > 0) ok = warp_wait(&B.stat_free, (joins - 1) & 1);
        if (!ok) break;
        stats[wg * 128 + row] = make_float2(m, l);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&B.stat_full);
        ok = warp_wait(&B.stat_full, joins & 1);  // and both accumulators are complete
        if (!ok) break;
        tc_fence_after();
        const float2 a = stats[row], c = stats[128 + row];
        __syncwarp();
        if (lane == 0) mbar_arrive(&B.stat_free);
        ++joins;
        m = fmaxf(a.x, c.x);
        const float mz = m == -INFINITY ? 0.f : m;
        ws[0] = fast_exp2(a.x - mz), ws[1] = fast_exp2(c.x - mz);
        l = a.y * ws[0] + c.y * ws[1];
      }
      const bool some = l > 0.f;
      const float inv = some ? 1.f / l : 0.f;
      ws[0] *= inv, ws[1] *= inv;
      const int tok = s.tok0 + x, hqi = s.head * p.group + row - xr * p.group;
      const int64_t prim = (static_cast<int64_t>(s.part) * p.n + tok) * p.hq + hqi;
      const int64_t cont = static_cast<int64_t>(cta) * C::ROWS + half * 128 + row;
      float* od = s.kb == 0 ? p.o_prim + prim * HD : p.o_cont + cont * HD;
      if (live && (!joined || wg == 0))
        (s.kb == 0 ? p.lse_prim + prim : p.lse_cont + cont)[0] =
            some ? (m - C::SHIFT + __log2f(l)) * kLn2 : (l == 0.f ? -INFINITY : l);
      if (warp_live) {
        // joined slots: each warpgroup writes half of the columns of both accumulators' sum
        const int c_lo = joined ? wg * (HD / 2) : 0, c_hi = joined ? c_lo + HD / 2 : HD;
        const uint32_t oa = tmem + C::TMEM_O + ((NWG == 2 && !joined) ? wg * HD : 0) + lane_addr;
#pragma unroll 1
        for (int c = c_lo; c < c_hi; c += 32) {
          float o[32];
          tmem_ld32(oa + c, o);
          if (joined) {
            float o2[32];
            tmem_ld32(oa + HD + c, o2);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = some ? o[k] * ws[0] + o2[k] * ws[1] : l;
          } else {
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = some ? o[k] * ws[0] : l;  // l: 0, or the NaN of the row
          }
          if (live) {
#pragma unroll
            for (int k = 0; k < 32; k += 8) store8(od + c + k, o + k);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        // an accumulator is free when all warps that read it are through (joined: both groups')
        if (joined) mbar_arrive(&B.o_free[0]), mbar_arrive(&B.o_free[1]);
        else mbar_arrive_n(&B.o_free[NWG == 2 ? wg : 0], NSW / 4);
      }
    }
    // ---- the segments of few rows, which come last
    if (ok && few_from >= 0) {
      // every warpgroup is through with the earlier segments, and their tiles with the ring
      __syncwarp();
      if (lane == 0) mbar_arrive(&B.meet);
      ok = warp_wait(&B.meet, 0);
      uint32_t meets = 0, index = 0;
      Seg s = few_seg;
      for (int sg = few_from; ok && s.part >= 0; ++index) {
        if (NWG == 1 || (index & 1) == static_cast<uint32_t>(wg)) {
          FewRows<C> f{p, s, B, smem, stats, wg, warp & 3, lane, cta, tile0, qu, meets, index};
          ok = f.run();
          meets = f.meets;
        }
        tile0 += s.ke - s.kb, ++qu;
        ok = ok && next_seg(++sg, s);
      }
    }
    if (!ok && lane == 0) set_error(p.err, FOLD_DEVERR_TIMEOUT);
  } else {
    if constexpr (NWG == 2) regs_down<kOtherRegs>();
    if (warp == NSW) {
      // ------------------------------------------------------------ TMA producer
      const int nch = TK / p.chunk;
      uint32_t u = 0;  // ring position
      bool ok = true;
      prefetch_tensormap(&kmap);
      prefetch_tensormap(&vmap);
      // one K or V tile at this lane's chunk's place
      auto load_tile = [&](const CUtensorMap* map, int c3, int id) {
#pragma unroll
        for (int w = 0; w < KU; ++w, ++u) {
          const int slot = u % NU;
          if (u >= NU) ok = warp_wait(&B.empty[slot], ((u / NU) - 1) & 1);
          if (!ok) return;
          if (lane == 0) mbar_arrive_expect_tx(&B.full[slot], C::UNIT);
          __syncwarp();
          if (lane < nch)
            tma_load_5d(smem + slot * C::UNIT + lane * p.chunk * (C::UC * 2), map, &B.full[slot], w * C::NCG, c3, id);
        }
      };
      bool owed = false;  // the V tile of the last K tile is still to come
      int v_c3 = 0, v_id = 0;
      for (int sg = 0; ok; ++sg) {
        Seg s;
        ok = next_seg(sg, s);
        if (!ok || s.part < 0) break;
        const int* table = s.part == 0 ? p.prefix_table : p.tables + s.seq * p.table_stride;
        // plane index of this lane's chunk of key tile j (chunks past the limit, and blocks that
        // do not exist, lie past the map and load as zeros)
        auto page = [&](int j) {
          const int p0 = j * TK + lane * p.chunk;
          if (lane >= nch || j >= s.ke || p0 >= s.limit) return p.oob;
          const int blk = __ldg(table + p0 / p.block_size);
          if (blk < 0 || blk >= p.num_blocks) {
            set_error(p.err, FOLD_DEVERR_BLOCK_TABLE);
            return p.oob;
          }
          return blk * p.mul_b + s.head * p.mul_h;
        };
        int next = page(s.kb);
        for (int j = s.kb; ok && j < s.ke; ++j) {
          const int id = next, c3 = ((j * TK + lane * p.chunk) % p.block_size) / 8;
          next = page(j + 1);  // looked up one tile ahead
          load_tile(&kmap, c3, id);
          if (ok && owed) load_tile(&vmap, v_c3, v_id);
          owed = true, v_c3 = c3, v_id = id;
        }
      }
      uint32_t gap = 0;
      if (ok && owed) {
        gap = u, u += KU;  // the last V keeps its place (v_pos); the K that would run ahead of it is left out
        load_tile(&vmap, v_c3, v_id);
      }
      if (!ok && lane == 0) set_error(p.err, FOLD_DEVERR_TIMEOUT);
      // copies in flight land before exit
      for (uint32_t w = u > NU ? u - NU : 0; w < u; ++w)
        if (gap == 0 || w - gap >= KU) warp_wait(&B.full[w % NU], (w / NU) & 1);
    } else if (warp == NSW + 1) {
      // ------------------------------------------------------------ MMA issuer
      // Steps over all segments, alternating the S buffers: QK of step g+2 is issued behind PV of
      // step g, across segments' borders. The whole warp walks; one lane issues.
      constexpr uint32_t idesc_s = idesc_of(C::F16, TK, 0);
      constexpr uint32_t idesc_o = idesc_of(C::F16, C::UC, 1);
      constexpr uint32_t hi_q = desc_hi(1024), hi_kv = desc_hi(C::NCG * 1024);
      const uint32_t base = uniform(smem_u32(smem)), q_base = base + C::OFF_Q, tm = uniform(tmem);
      // The issue of MMAs lasts about as long as they run, so all else in a step comes where it hides
      // behind the last ones issued: the next K behind PV, the next P behind QK. V is waited for by
      // the softmax warps, before they hand over P.
      struct Place {  // of a unit in the ring, walked (K0 K1 V0 K2 V1 ...) rather than divided out
        uint32_t slot, parity;
        __device__ __forceinline__ void move(uint32_t n) {
          slot += n;
          if (slot >= NU) slot -= NU, parity ^= 1;
        }
        __device__ __forceinline__ Place unit(int w) const {
          Place x = *this;
          if (w) x.move(w);
          return x;
        }
      };
      struct Step {
        Place v;
        uint32_t v_lo[KU], fresh;
        bool valid, first, last, free_kv;
      } st0, st1;
      bool ok = true, more = true, ended = false, wide = false;
      int sg = 0, i = 0, steps = 0;  // next segment; next step of the current one
      uint32_t qu = 0;               // Q tiles used before the current segment
      uint32_t pcnt[2] = {0, 0}, ocnt[2] = {0, 0};
      Place k_at{0, 0}, v_at{2 * KU, 0}, k_now{0, 0}, v_now{0, 0};  // of the next tile, of this one
      uint32_t k_step = KU, k_lo[KU], v_lo[KU];
      auto qk = [&](Step& st, const int b) {  // the next step, into S buffer b
        st.valid = false;
        if (i == steps) {
          if (!more) return;
          if (steps) qu += wide ? 2 : 1;
          Seg s;
          ok = next_seg(sg, s);
          if (!ok) return;
          ++sg;
          if (s.part < 0 || few_rows(s)) {  // all that follow are the softmax warps' own
            more = false, ended = s.part < 0, i = steps = 0;
            return;
          }
          wide = s.ntok > p.half_toks;  // the steps of a tile are its row halves
          steps = (s.ke - s.kb) * (wide ? 2 : 1), i = 0;
        }
        const int half = wide ? i & 1 : 0;
        const uint32_t quse = qu + half, qslot = quse % QB;
        const uint32_t a = uniform(desc_lo(q_base + qslot * C::Q_TILE, 16));
        if (half == 0) {
          k_now = k_at, v_now = v_at;
          k_at.move(k_step), v_at.move(2 * KU);
          k_step = 2 * KU;
#pragma unroll
          for (int w = 0; w < KU; ++w) {
            k_lo[w] = uniform(desc_lo(base + k_now.unit(w).slot * C::UNIT, 16));
            ok = ok && mbar_wait(&B.full[k_now.unit(w).slot], k_now.unit(w).parity);
          }
        }
        if (i == half) ok = ok && mbar_wait(&B.q_full[qslot], (quse / QB) & 1);  // the first use of this Q tile
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) return;
        const bool free_kv = !wide || half == 1;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int w = 0; w < KU; ++w) {
#pragma unroll
            for (int kk = 0; kk < C::UC / 16; ++kk)
              mma_ss(tm + C::TMEM_S + b * TK, a + ((w * C::NCG + (kk >> 2)) * C::Q_CG + (kk & 3) * 32) / 16, hi_q,
                     k_lo[w] + ((kk >> 2) * 1024 + (kk & 3) * 32) / 16, hi_kv, idesc_s, w > 0 || kk > 0);
            if (w == KU - 1) tc_commit(&B.s_full[b]);
            if (free_kv) commit_for<NSW>(&B.empty[k_now.unit(w).slot]);
          }
          if (i + (wide ? 2 : 1) >= steps) commit_for<NSW>(&B.q_empty[qslot]);
        }
        __syncwarp();
        st.valid = true, st.first = NWG == 2 ? i < 2 : i == 0, st.last = i + NWG >= steps, st.free_kv = free_kv;
        st.v = v_now, st.fresh = uniform(st.first ? 0 : 1);
#pragma unroll
        for (int w = 0; w < KU; ++w) {
          if (half == 0) v_lo[w] = uniform(desc_lo(base + v_now.unit(w).slot * C::UNIT, 1024));
          st.v_lo[w] = v_lo[w];
        }
        ++i;
      };
      auto pv = [&](Step& st, const int b) {
        const int acc = NWG == 2 ? b : 0;
        if (st.first) {  // the accumulator's last segment has been read
          if (ocnt[acc] > 0) ok = mbar_wait(&B.o_free[acc], (ocnt[acc] - 1) & 1);
          ++ocnt[acc];
        }
        ok = ok && mbar_wait(&B.p_full[b], pcnt[b]++ & 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) return;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int w = 0; w < KU; ++w) {
#pragma unroll
            for (int ks = 0; ks < TK / 16; ++ks)
              mma_ts(tm + C::TMEM_O + acc * HD + w * C::UC, tm + C::TMEM_S + b * TK + ks * 8,
                     st.v_lo[w] + ks * 2 * C::NCG * 1024 / 16, hi_kv, idesc_o, ks > 0 ? 1 : st.fresh);
            if (st.free_kv) commit_for<NSW>(&B.empty[st.v.unit(w).slot]);
          }
          if (NWG == 1) tc_commit(&B.pv_done);
          if (st.last) tc_commit(&B.seg_done[acc]);
        }
        __syncwarp();
        qk(st, b);
      };
      qk(st0, 0);
      if (ok) qk(st1, 1);
      while (ok && st0.valid) {
        pv(st0, 0);
        if (!ok || !st1.valid) break;
        pv(st1, 1);
      }
      for (Seg s; ok && !ended; ended = s.part < 0) ok = next_seg(sg++, s);
      if (!ok) {  // let what was issued finish before TMEM goes
        if (elect_one()) {
          set_error(p.err, FOLD_DEVERR_TIMEOUT);
          tc_commit(&B.drained);
        }
        __syncwarp();
        warp_wait(&B.drained, 0);
      }
    } else if (warp == NSW + 3) {
      // ------------------------------------------------------------ Q loader
      uint32_t qu = 0;
      bool ok = true;
      for (int sg = 0; ok; ++sg) {
        Seg s;
        ok = next_seg(sg, s);
        if (!ok || s.part < 0) break;
        for (int t0 = 0; ok && t0 < s.ntok; t0 += p.half_toks, ++qu) {
          const uint32_t slot = qu % QB;
          if (qu >= QB) ok = warp_wait(&B.q_empty[slot], ((qu / QB) - 1) & 1);
          if (!ok) break;
          const int nt = min(p.half_toks, s.ntok - t0);
          unsigned char* dst = smem + C::OFF_Q + slot * C::Q_TILE;
          if (nt * p.group > kFewQRows) {
            // a box of half_toks tokens (those past nt give rows that nobody reads)
            if (lane == 0) {
              mbar_arrive_expect_tx(&B.q_full[slot], HD / 64 * p.half_toks * p.group * 128);
#pragma unroll
              for (int c = 0; c < HD / 64; ++c)
                tma_load_3d_plain(dst + c * C::Q_CG, &qmap, &B.q_full[slot], c * 64, s.head * p.group, s.tok0 + t0);
            }
            __syncwarp();
          } else {
            constexpr int CPR = HD / 8, RPI = 32 / CPR;  // 16-byte chunks of a row, rows a round
            const int c = lane % CPR;
            int r = lane / CPR, x = r / p.group, g = r - x * p.group;
            const uint32_t d = smem_u32(dst) + (c >> 3) * C::Q_CG;
            const T* src = static_cast<const T*>(p.q) + (s.tok0 + t0) * p.q_st + s.head * p.group * p.q_sh + c * 8;
            for (; x < nt; r += RPI, g += RPI) {
              while (g >= p.group) g -= p.group, ++x;
              if (x < nt) cp_async_16(d + r * 128 + (((c & 7) ^ (r & 7)) << 4), src + x * p.q_st + g * p.q_sh, 16);
            }
            cp_async_wait_all();
            fence_proxy_async();  // Q is read by the tensor cores
            __syncwarp();
            if (lane == 0) mbar_arrive(&B.q_full[slot]);
          }
        }
      }
      if (!ok && lane == 0) set_error(p.err, FOLD_DEVERR_TIMEOUT);
      // copies in flight land before exit (a read that gives up may leave the last tiles unread)
      for (uint32_t w = qu > QB ? qu - QB : 0; w < qu; ++w) warp_wait(&B.q_full[w % QB], (w / QB) & 1);
    } else if (warp == NSW + 2) {
      // ------------------------------------------------------------ scheduler
      int sg = 0;
      bool ok = true;
      auto publish = [&](const Seg& s) {
        if (sg >= kSegs) ok = warp_wait(&B.seg_empty[sg % kSegs], ((sg / kSegs) - 1) & 1);
        if (!ok) return;
        if (lane == 0) {
          B.seg[sg % kSegs] = s;
          mbar_arrive(&B.seg_full[sg % kSegs]);
        }
        __syncwarp();
        ++sg;
      };
      // one item: s without its tile range; at: its place on the line
      auto item = [&](Seg s, int64_t at) {
        const int tiles = (s.limit + TK - 1) / TK, w = tile_cost(p, s.ntok), start = start_cost(p, s.ntok);
        const int64_t end = at + item_cost(p, tiles, s.ntok);
        // key tiles of this item that lie before place x of the line
        auto tiles_before = [&](int64_t x) {
          if (x >= end) return tiles;
          const int64_t y = x - at - start + w / 2;
          return y <= 0 ? 0 : static_cast<int>(min64(quot(y, w), tiles));
        };
        s.kb = at >= x0 ? 0 : tiles_before(x0), s.ke = tiles_before(x1);
        if (s.kb < s.ke) publish(s);
        if (at >= x0) {  // the item starts here: note the CTAs that hold its tiles
          int c0 = cta, cnt = tiles > 0;
          if (s.ke < tiles) {
            int upto = s.ke;
            while (upto == 0) ++c0, upto = tiles_before(cut(c0 + 1));
            // a CTA at or past the item's end, then back
            const int k = end > cut_x;
            const int64_t past = (k ? before + quot(end - cut_x, each[1]) : quot(end, each[0])) + 1;
            int c1 = max(static_cast<int>(min64(ctas - 1, past)), c0);
            while (c1 > c0 && tiles_before(cut(c1)) >= tiles) --c1;
            cnt = c1 - c0 + 1;
          }
          for (int x = lane; x < s.ntok; x += 32)
            p.plan[(static_cast<int64_t>(s.part) * p.n + s.tok0 + x) * p.hkv + s.head] = make_int4(c0, cnt, s.tok0, 0);
        }
      };
      // items of row tiles [rt, rt_end) of the prefix, c each, the first at place `from`
      auto walk_prefix = [&](int rt, int rt_end, int64_t c, int64_t from) {
        const int64_t row_cost = c * p.hkv;
        if (rt >= rt_end || x1 <= from || x0 >= from + (rt_end - rt) * row_cost) return;
        Seg s{};
        s.limit = s.lim0 = plen;
        const int64_t in = max64(x0 - from, 0);
        const int skip = static_cast<int>(quot(in, row_cost));
        int64_t at = from + skip * row_cost;
        int h = static_cast<int>(quot(in - skip * row_cost, c));
        for (rt += skip; ok && rt < rt_end && at < x1; ++rt, h = 0, at += row_cost) {
          s.tok0 = tok_lo + rt * per_tile, s.ntok = min(per_tile, tok_hi - s.tok0);
          for (; ok && h < p.hkv && at + h * c < x1; ++h) {
            s.head = h;
            item(s, at + h * c);
          }
        }
      };
      // the sequences' own items of many (0) or few (1) rows
      auto walk_own = [&](int k) {
        if (own_total[k] == 0 || x1 <= from_own[k] || x0 >= from_own[k] + own_total[k]) return;
        Seg s{};
        s.part = 1, s.lim_step = p.causal ? 1 : 0;
        int64_t at = from_own[k] + B.start_base[k];
        for (int q = B.start_seq[k]; ok && q < p.b && at < x1; ++q) {
          int first, last;
          seq_rows(p, q, first, last);
          const int m = capped(__ldg(p.own_lens + q), p.own_cap, p.err);
          for (int t0 = first; ok && t0 < last && at < x1; t0 += per_tile) {
            s.seq = q, s.tok0 = t0, s.ntok = min(per_tile, last - t0);
            if (few_rows(s) != (k == 1)) continue;
            own_limits(p, first, last, m, t0, s.ntok, s.limit, s.lim0);
            const int64_t c = item_cost(p, (s.limit + TK - 1) / TK, s.ntok);
            int h = 0;
            if (at + c * p.hkv <= x0) h = p.hkv;  // wholly before this CTA's piece
            else if (x0 > at) h = static_cast<int>(quot(x0 - at, c));
            for (; ok && h < p.hkv && at + h * c < x1; ++h) {
              s.head = h;
              item(s, at + h * c);
            }
            at += c * p.hkv;
          }
        }
      };
      if (x0 < x1) {
        walk_prefix(0, prow_tiles - 1, pc_full, 0);
        if (!last_few) walk_prefix(prow_tiles - 1, prow_tiles, pc_last, from_last);
        walk_own(0);
        if (last_few && prow_tiles) walk_prefix(prow_tiles - 1, prow_tiles, pc_last, from_last);
        walk_own(1);
      }
      if (ok) {
        Seg s{};
        s.part = -1;
        publish(s);
      }
      if (!ok && lane == 0) set_error(p.err, FOLD_DEVERR_TIMEOUT);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == NSW + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

// Joins the partials of one row: its prefix item's and its own item's, one per CTA that held a part
// of the item. WPR warps a row take every WPR-th partial each; a lane reads the lse of one.
// Latency bound (a few partials of a row, from L2).
template <int HD, class T, int WPR>
__global__ void __launch_bounds__(128) prefix_merge_kernel(const PrefixParams p, int cont_rows) {
  constexpr int V = HD / 32, RPB = 4 / WPR;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = warp % WPR;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * RPB + warp / WPR;
  const int tok = static_cast<int>(row / p.hq), h = static_cast<int>(row - static_cast<int64_t>(tok) * p.hq);
  const int hk = h / p.group, g = h - hk * p.group;
  wait_for_producer();
  if (tok >= p.n || tok < p.qsl[0] || tok >= p.qsl[p.b]) return;  // with WPR 4 the whole block
  const bool prefix = p.prefix_len[0] > 0 && p.prefix_cap > 0;
  const int4 none = make_int4(0, 0, 0, 0);
  // a read that gave up (FOLD_DEVERR_TIMEOUT) may have left a plan unwritten
  auto sane = [&](int4 v) {
    const bool fine = v.x >= 0 && v.y >= 0 && v.y <= p.ctas && v.x <= p.ctas - v.y && v.z >= 0 && v.z <= tok &&
                      tok - v.z < (cont_rows / 128) * p.half_toks;
    return fine ? v : none;
  };
  const int4 pp = prefix ? sane(p.plan[static_cast<int64_t>(tok) * p.hkv + hk]) : none;
  const int4 po = sane(p.plan[(static_cast<int64_t>(p.n) + tok) * p.hkv + hk]);
  const int cnt = pp.y + po.y;
  float acc[V], m = -INFINITY, z = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.f;
  for (int base = 0; sub + WPR * base < cnt; base += 32) {
    const int i = sub + WPR * (base + lane);
    const float* o = nullptr;
    float lse = -INFINITY;
    if (i < cnt) {
      const bool own = i >= pp.y;
      const int4 plan = own ? po : pp;
      const int k = own ? i - pp.y : i;
      if (k == 0) {
        const int64_t at = (static_cast<int64_t>(own ? p.n : 0) + tok) * p.hq + h;
        lse = p.lse_prim[at], o = p.o_prim + at * HD;
      } else {
        const int x = tok - plan.z, half = x / p.half_toks;
        const int64_t at = static_cast<int64_t>(plan.x + k) * cont_rows + half * 128 + (x - half * p.half_toks) * p.group + g;
        lse = p.lse_cont[at], o = p.o_cont + at * HD;
      }
    }
    float top = lse;
#pragma unroll
    for (int s = 16; s; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
    top = fmaxf(top, m);
    const float mz = top == -INFINITY ? 0.f : top;
    const float w = i < cnt ? __expf(lse - mz) : 0.f, f = __expf(m - mz);
    m = top;
    float zs = w;
#pragma unroll
    for (int s = 16; s; s >>= 1) zs += __shfl_xor_sync(0xffffffffu, zs, s);
    z = z * f + zs;
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] *= f;
    const int nk = min(32, (cnt - sub + WPR - 1) / WPR - base);
#pragma unroll 4
    for (int k = 0; k < nk; ++k) {
      const float wk = __shfl_sync(0xffffffffu, w, k);
      const float* ok = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(o), k));
      if constexpr (V == 2) {
        const float2 a = reinterpret_cast<const float2*>(ok)[lane];
        acc[0] += wk * a.x, acc[1] += wk * a.y;
      } else {
#pragma unroll
        for (int j = 0; j < V; j += 4) {
          const float4 a = reinterpret_cast<const float4*>(ok)[lane * (V / 4) + j / 4];
          acc[j] += wk * a.x, acc[j + 1] += wk * a.y, acc[j + 2] += wk * a.z, acc[j + 3] += wk * a.w;
        }
      }
    }
  }
  if constexpr (WPR > 1) {
    __shared__ float sm[WPR], sz[WPR], so[WPR][HD];
    if (lane == 0) sm[sub] = m, sz[sub] = z;
#pragma unroll
    for (int j = 0; j < V; ++j) so[sub][lane * V + j] = acc[j];
    __syncthreads();
    if (sub) return;
    float top = sm[0];
#pragma unroll
    for (int w = 1; w < WPR; ++w) top = fmaxf(top, sm[w]);
    const float mz = top == -INFINITY ? 0.f : top;
    m = top, z = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] = 0.f;
#pragma unroll
    for (int w = 0; w < WPR; ++w) {
      const float f = __expf(sm[w] - mz);
      z += sz[w] * f;
#pragma unroll
      for (int j = 0; j < V; ++j) acc[j] += f * so[w][lane * V + j];
    }
  }
  const float inv = z > 0.f ? 1.f / z : (z == 0.f ? 0.f : z);  // a NaN reaches the output
  T* out = static_cast<T*>(p.out) + tok * p.o_st + h * p.o_sh + lane * V;
  uint32_t w[V / 2];
#pragma unroll
  for (int i = 0; i < V; i += 2) w[i / 2] = pack2<T>(acc[i] * inv, acc[i + 1] * inv);
  if constexpr (V == 2) *reinterpret_cast<uint32_t*>(out) = w[0];
  else if constexpr (V == 4) *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[1]);
  else *reinterpret_cast<uint4*>(out) = make_uint4(w[0], w[1], w[2], w[3]);
  if (lane == 0 && p.lse)
    p.lse[static_cast<int64_t>(h) * p.n + tok] = z > 0.f ? m + logf(z) : (z == 0.f ? -INFINITY : z);
}

// ---------------------------------------------------------------- host
// The places of a workspace, counted from its first 32-byte boundary: partials are stored 32 bytes at a
// time (store8), callers give 16-byte boundaries.
constexpr int kBaseAlign = 32;
struct Layout {
  int64_t plan, o_prim, lse_prim, o_cont, lse_cont, bytes;
};
Layout layout(int64_t n, int hq, int hkv, int hd, int ctas) {
  const int64_t rows = hd == 256 ? 128 : 256;
  auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
  Layout w;
  w.plan = 0;
  w.o_prim = up(2 * n * hkv * 16);
  w.lse_prim = w.o_prim + up(2 * n * hq * hd * 4);
  w.o_cont = w.lse_prim + up(2 * n * hq * 4);
  w.lse_cont = w.o_cont + up(ctas * rows * hd * 4);
  w.bytes = w.lse_cont + up(ctas * rows * 4) + kBaseAlign - 16;
  return w;
}

int ctas_of_device() {
  const int sms = device_sm_count();
  return sms > 0 ? sms : 148;
}

// 3-D map of q: columns, heads, tokens; a box is one 64-column group of a half row tile's rows.
int query_map(const PrefixParams& p, int hd, bool f16, CUtensorMap* out) {
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(hd), static_cast<cuuint64_t>(p.hq), static_cast<cuuint64_t>(p.n)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(p.q_sh) * 2, static_cast<cuuint64_t>(p.q_st) * 2};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(p.group), static_cast<cuuint32_t>(p.half_toks)};
  return tiled_map("prefix read", p.q, 3, dims, strides, box, f16, out);
}

// 5-D map of a K or V plane: 64 columns, 8 slots, 64-column groups, groups of 8 slots, and blocks
// and heads as one index (in units of the smaller of their strides). A box of `chunk` slots lands
// as [group of 8 slots][64-column group][8 rows of 128 bytes], 128-byte swizzled: consecutive
// chunks stack to a tile whose 8-row groups have one stride, whatever the page size.
int plane_map(const void* base, int hd, int box_cols, int block_size, int chunk, int64_t slot, int64_t unit,
              int64_t count, bool f16, CUtensorMap* out) {
  const cuuint64_t dims[5] = {64, 8, static_cast<cuuint64_t>(hd / 64), static_cast<cuuint64_t>(block_size / 8),
                              static_cast<cuuint64_t>(count)};
  const cuuint64_t strides[4] = {static_cast<cuuint64_t>(slot) * 2, 128, static_cast<cuuint64_t>(slot) * 16,
                                 static_cast<cuuint64_t>(unit) * 2};
  const cuuint32_t box[5] = {64, 8, static_cast<cuuint32_t>(box_cols / 64), static_cast<cuuint32_t>(chunk / 8), 1};
  return tiled_map("prefix read", base, 5, dims, strides, box, f16, out);
}

template <int HD, class T>
int launch_prefix(const PrefixParams& p, const void* k, const void* v, int64_t slot, int64_t unit, cudaStream_t stream) {
  using C = Cfg<HD, T>;
  CUtensorMap qmap, kmap, vmap;
  if (int s = query_map(p, HD, C::F16, &qmap)) return s;
  const int64_t count = p.oob;
  if (int s = plane_map(k, HD, C::UC, p.block_size, p.chunk, slot, unit, count, C::F16, &kmap)) return s;
  if (int s = plane_map(v, HD, C::UC, p.block_size, p.chunk, slot, unit, count, C::F16, &vmap)) return s;
  static std::atomic<uint64_t> configured{0};
  if (int s = allow_smem(prefix_read_kernel<C>, C::SMEM, configured, "cudaFuncSetAttribute(prefix_read)")) return s;
  if constexpr (C::NWG == 2) {
    // the register shares the warps take must add up to what a block is launched with
    static const int regs = [] {
      cudaFuncAttributes a{};
      return cudaFuncGetAttributes(&a, prefix_read_kernel<C>) == cudaSuccess ? a.numRegs : 0;
    }();
    if (regs != kLaunchRegs) return fail(FOLD_ERR_UNSUPPORTED, "prefix read: built with other register shares than launched");
  }
  if (int s = launch_behind(prefix_read_kernel<C>, dim3(p.ctas), C::NTHREADS, C::SMEM, stream, "prefix_read_kernel",
                            qmap, kmap, vmap, p))
    return s;
  const int64_t rows = static_cast<int64_t>(p.n) * p.hq;
  // few rows have many partials each, which four warps share: with four and with one warp a row the whole
  // call took 31.1 and 34.3 us at 256 rows over 16K keys, 68.5 and 71.5 at 1024 over 64K, 89.0 and 92.2 at
  // 1152 over 64K, 43.1 and 43.8 at 1536 over 16K, 46.6 and 46.0 at 2048, 71.9 and 66.2 at 4096
  if (rows <= 1536)
    return launch_behind(prefix_merge_kernel<HD, T, 4>, dim3(static_cast<unsigned>(rows)), 128, 0, stream,
                         "prefix_merge_kernel", p, C::ROWS);
  return launch_behind(prefix_merge_kernel<HD, T, 1>, dim3(static_cast<unsigned>((rows + 3) / 4)), 128, 0, stream,
                       "prefix_merge_kernel", p, C::ROWS);
}

}  // namespace
}  // namespace fold

extern "C" {

int64_t fold_prefix_read_workspace(int n, int hq, int hkv, int hd) {
  if (n < 0 || hq < 1 || hkv < 1 || hq % hkv || hq / hkv > 128 || (hd != 64 && hd != 128 && hd != 256)) return -1;
  return fold::layout(n, hq, hkv, hd, fold::ctas_of_device()).bytes;
}

int fold_prefix_read(const void* q, int64_t q_stride_tok, int64_t q_stride_head, const int* qsl, const int* own_lens,
                     const int* prefix_len, int b, const void* k_cache, const void* v_cache, int64_t num_blocks,
                     int block_size, int64_t cache_stride_block, int64_t cache_stride_head, int64_t cache_stride_slot,
                     const int* prefix_table, int prefix_table_len, const int* block_tables,
                     int64_t block_tables_stride, int block_tables_len, int causal, float softmax_scale, void* out,
                     int64_t o_stride_tok, int64_t o_stride_head, float* lse, void* workspace, int64_t workspace_bytes,
                     int n, int hq, int hkv, int hd, int dtype, int* err, void* stream) {
  using namespace fold;
  if (n < 0 || b < 0 || hq < 1 || hkv < 1 || hq % hkv || num_blocks < 1 || block_size < 16 || block_size % 16 ||
      prefix_table_len < 0 || block_tables_len < 0 || (dtype != FOLD_BF16 && dtype != FOLD_FP16))
    return fail(FOLD_ERR_INVALID_ARGUMENT, "prefix read: bad sizes or type");
  if (hd != 64 && hd != 128 && hd != 256) return fail(FOLD_ERR_UNSUPPORTED, "prefix read: head size 64, 128 or 256");
  if (hq / hkv > 128) return fail(FOLD_ERR_UNSUPPORTED, "prefix read: hq / hkv must be at most 128");
  if (!(softmax_scale > 0.f) || softmax_scale > 1e30f)
    return fail(FOLD_ERR_INVALID_ARGUMENT, "prefix read: softmax_scale must be positive and finite");
  if (n == 0 || b == 0) return FOLD_OK;
  if (!q || !qsl || !own_lens || !prefix_len || !k_cache || !v_cache || (prefix_table_len && !prefix_table) ||
      (block_tables_len && !block_tables) || !out)  // a table of no blocks may be null
    return fail(FOLD_ERR_INVALID_ARGUMENT, "prefix read: null pointer");
  auto overlap = [&](int64_t stride) { return stride < hd && stride > -hd; };  // of rows that are neighbours
  if ((n > 1 && overlap(o_stride_tok)) || (hq > 1 && overlap(o_stride_head)))
    return fail(FOLD_ERR_INVALID_ARGUMENT, "prefix read: the rows of out must not share memory");
  if (!aligned16(q) || !aligned16(out) || !aligned16(k_cache) || !aligned16(v_cache) || q_stride_tok % 8 ||
      q_stride_head % 8 || o_stride_tok % 8 || o_stride_head % 8 || cache_stride_block % 8 || cache_stride_head % 8 ||
      cache_stride_slot % 8)
    return fail(FOLD_ERR_ALIGNMENT, "prefix read: rows of q, out and the cache must start on 16-byte boundaries");
  if (n == 1) q_stride_tok = static_cast<int64_t>(hq) * hd;  // strides of a single row or head are free
  if (hq == 1) q_stride_head = hd;
  if (q_stride_tok < 1 || q_stride_head < 1 || q_stride_tok >= (int64_t(1) << 38) || q_stride_head >= (int64_t(1) << 38))
    return fail(FOLD_ERR_INVALID_ARGUMENT, "prefix read: q's strides must be positive");
  if (cache_stride_slot < hd || cache_stride_slot >= (int64_t(1) << 35))
    return fail(FOLD_ERR_INVALID_ARGUMENT, "prefix read: bad cache strides");
  // blocks and heads as one index of the plane
  int64_t unit, mul_b = 0, mul_h = 0;
  if (hkv == 1) unit = num_blocks == 1 ? hd : cache_stride_block, mul_b = 1;
  else if (num_blocks == 1) unit = cache_stride_head, mul_h = 1;
  else unit = cache_stride_block < cache_stride_head ? cache_stride_block : cache_stride_head;
  if (unit < 8 || unit >= (int64_t(1) << 38))
    return fail(FOLD_ERR_INVALID_ARGUMENT, "prefix read: bad cache strides");
  if (hkv > 1 && num_blocks > 1) {
    if (cache_stride_block % unit || cache_stride_head % unit)
      return fail(FOLD_ERR_INVALID_ARGUMENT, "prefix read: of the cache's block and head strides one must divide the other");
    mul_b = cache_stride_block / unit, mul_h = cache_stride_head / unit;
  }
  const int64_t most = 2147483000;
  if (num_blocks > most || mul_b > most || mul_h > most || (num_blocks - 1) > most / (mul_b > 0 ? mul_b : 1) ||
      (num_blocks - 1) * mul_b + (hkv - 1) * mul_h > most)
    return fail(FOLD_ERR_INVALID_ARGUMENT, "prefix read: the cache has too many blocks");
  if (static_cast<int64_t>(n) * hq > (int64_t(1) << 31))
    return fail(FOLD_ERR_INVALID_ARGUMENT, "prefix read: too many rows");
  const int ctas = ctas_of_device();
  const Layout w = layout(n, hq, hkv, hd, ctas);
  if (!workspace || workspace_bytes < w.bytes)
    return fail(FOLD_ERR_INVALID_ARGUMENT, "prefix read: the workspace holds fold_prefix_read_workspace bytes");
  if (!aligned16(workspace)) return fail(FOLD_ERR_ALIGNMENT, "prefix read: the workspace must be 16-byte aligned");
  PrefixParams p{};
  p.q = q, p.q_st = q_stride_tok, p.q_sh = q_stride_head, p.qsl = qsl, p.own_lens = own_lens;
  p.prefix_len = prefix_len, p.b = b, p.prefix_table = prefix_table, p.tables = block_tables;
  p.table_stride = block_tables_stride;
  auto positions = [&](int blocks) {
    const int64_t x = static_cast<int64_t>(blocks) * block_size;
    return static_cast<int>(x < most ? x : most / 128 * 128);
  };
  p.prefix_cap = positions(prefix_table_len), p.own_cap = positions(block_tables_len);
  p.num_blocks = num_blocks, p.block_size = block_size;
  p.chunk = 16;
  while (p.chunk < 128 && block_size % (2 * p.chunk) == 0) p.chunk *= 2;
  p.mul_b = static_cast<int>(mul_b), p.mul_h = static_cast<int>(mul_h);
  p.oob = static_cast<int>((num_blocks - 1) * mul_b + (hkv - 1) * mul_h + 1);
  p.causal = causal ? 1 : 0, p.scale_log2 = softmax_scale * kLog2e;
  p.out = out, p.o_st = o_stride_tok, p.o_sh = o_stride_head, p.lse = lse;
  p.n = n, p.hq = hq, p.hkv = hkv, p.group = hq / hkv, p.half_toks = 128 / p.group;
  p.item_cost = hd == 256 ? kItemCost256 : kItemCost, p.ctas = ctas, p.err = err;
  char* ws = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(workspace) + kBaseAlign - 1) & ~uintptr_t(kBaseAlign - 1));
  p.plan = reinterpret_cast<int4*>(ws + w.plan);
  p.o_prim = reinterpret_cast<float*>(ws + w.o_prim), p.lse_prim = reinterpret_cast<float*>(ws + w.lse_prim);
  p.o_cont = reinterpret_cast<float*>(ws + w.o_cont), p.lse_cont = reinterpret_cast<float*>(ws + w.lse_cont);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t slot = cache_stride_slot;
  if (dtype == FOLD_BF16) {
    if (hd == 64) return launch_prefix<64, __nv_bfloat16>(p, k_cache, v_cache, slot, unit, st);
    if (hd == 128) return launch_prefix<128, __nv_bfloat16>(p, k_cache, v_cache, slot, unit, st);
    return launch_prefix<256, __nv_bfloat16>(p, k_cache, v_cache, slot, unit, st);
  }
  if (hd == 64) return launch_prefix<64, __half>(p, k_cache, v_cache, slot, unit, st);
  if (hd == 128) return launch_prefix<128, __half>(p, k_cache, v_cache, slot, unit, st);
  return launch_prefix<256, __half>(p, k_cache, v_cache, slot, unit, st);
}

}  // extern "C"
