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
//   MMA warp: S = Q K^T and O += P V (P from TMEM), issued by one thread;
//   scheduler warp: walks the items, publishes segments in a small ring, loads Q by cp.async.
// Two S buffers and two O accumulators ("slots") keep the tensor cores busy while a warpgroup is
// in its softmax: above 128 rows the slots are the two halves of the row tile and share each K and
// V tile; otherwise they take the key tiles in turn and are joined at the end of the segment. At
// head size 256 one accumulator fills the columns that S leaves, so one warpgroup serves both S
// buffers.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cudaTypedefs.h>

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
  static constexpr int NTHREADS = (NSW + 4) * 32;  // + TMA, MMA, scheduler, one idle
  static constexpr int ROWS = NWG * 128;
  static constexpr int UC = HD < 128 ? HD : 128;  // columns of a unit
  static constexpr int KU = HD / UC;              // units of a K (or V) tile
  static constexpr int NCG = UC / 64;             // 64-column groups of a unit
  static constexpr int UNIT = TK * UC * 2;
  static constexpr int Q_CG = 128 * 128;  // one 64-column group of a Q tile
  static constexpr int Q_TILE = 128 * HD * 2;
  static constexpr int QB = HD == 256 ? 1 : 2;
  static constexpr int MISC = 768 + 2048;  // barriers, segments, scan; row statistics
  static constexpr int FIT = (kSmemLimit - MISC - QB * Q_TILE) / UNIT;
  static constexpr int NU = FIT > 12 ? 12 : FIT;
  static constexpr int OFF_Q = NU * UNIT;
  static constexpr int OFF_BAR = OFF_Q + QB * Q_TILE;
  static constexpr int OFF_STAT = OFF_BAR + 768;
  static constexpr int SMEM = OFF_BAR + MISC;
  static constexpr int TMEM_S = 0, TMEM_O = 256, TMEM_COLS = 512;
  static constexpr bool F16 = sizeof(T) == 2 && !std::is_same<T, __nv_bfloat16>::value;
  // fp16 keeps P in [2^-24, 2^15): scaled up by 2^7 so that small weights stay above its smallest step
  static constexpr float SHIFT = F16 ? 7.f : 0.f;
  static_assert(NU >= 4 && SMEM <= kSmemLimit, "shared memory");
};

// Cost units (a quarter of a key tile of a row tile of at most 128 rows).
constexpr int kTileCost = 4, kWideTileCost = 8, kItemCost = 4;

struct Seg {
  int part;  // 0: prefix, 1: own keys, -1: no more work
  int seq, head, tok0, rows;
  int kb, ke;   // key tiles [kb, ke)
  int limit;    // keys any row of the item sees
  int lim0, lim_step;  // row of token tok0 + x sees min(limit, lim0 + x * lim_step) keys
  int pad[2];
};
constexpr int kSegs = 4;

struct Bars {
  uint64_t full[12], empty[12];
  uint64_t s_full[2], p_full[2], pv_done;
  uint64_t q_full[2], q_empty[2];
  uint64_t seg_full[kSegs], seg_empty[kSegs];
  uint64_t seg_done, o_free, stat_full;
  uint32_t tmem;
  int start_seq;
  int64_t start_base;
  int64_t scan[16];
  Seg seg[kSegs];
};
static_assert(sizeof(Bars) <= 768, "barriers fit their place");

// ---------------------------------------------------------------- the line of work
__device__ __forceinline__ int capped(int len, int cap, int* err) {
  if (len > cap) {
    set_error(err, FOLD_DEVERR_CAPACITY);
    len = cap;
  }
  return max(len, 0);
}

__device__ __forceinline__ int tile_cost(int rows) { return rows > 128 ? kWideTileCost : kTileCost; }

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

__device__ __forceinline__ int64_t item_cost(int tiles, int rows) {
  return kItemCost + static_cast<int64_t>(tiles) * tile_cost(rows);
}

// Cost of all own items of sequence s and one KV head.
template <int ROWS>
__device__ __forceinline__ int64_t seq_cost(const PrefixParams& p, int s, int per_tile) {
  int first, last;
  seq_rows(p, s, first, last);
  const int m = capped(__ldg(p.own_lens + s), p.own_cap, p.err);
  int64_t c = 0;
  for (int t0 = first; t0 < last; t0 += per_tile) {
    const int nt = min(per_tile, last - t0);
    int limit, lim0;
    own_limits(p, first, last, m, t0, nt, limit, lim0);
    c += item_cost((limit + TK - 1) / TK, nt * p.group);
  }
  return c;
}

// ---------------------------------------------------------------- TMEM and MMA forms of this kernel
__device__ __forceinline__ void tmem_ld32(uint32_t a, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(a)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t a, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(a),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// D[tmem] (+)= A[tmem] x B[smem desc].
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u)
      : "memory");
}
// Instruction descriptor of kind::f16 for bf16 or f16 operands, f32 accumulation, M = 128.
constexpr uint32_t idesc_of(bool f16, int n, int b_mn) {
  const uint32_t fmt = f16 ? 0u : 1u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | (static_cast<uint32_t>(b_mn) << 16) |
         (static_cast<uint32_t>(n >> 3) << 17) | (8u << 24);
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
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity));
}

// Ring position (in tiles' K or V) of K(j) and V(j) of a segment of T tiles: K runs one tile
// ahead, K0 K1 V0 K2 V1 ... V(T-1), the order in which the MMAs first need them.
__device__ __forceinline__ int k_pos(int j) { return j == 0 ? 0 : 2 * j - 1; }
__device__ __forceinline__ int v_pos(int j, int T) { return min(2 * j + 2, 2 * T - 1); }

// ---------------------------------------------------------------- the kernel
template <class C>
__global__ void __launch_bounds__(C::NTHREADS, 1)
    prefix_read_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                       const PrefixParams p) {
  constexpr int HD = C::HD, KU = C::KU, NU = C::NU, NWG = C::NWG, NSW = C::NSW, QB = C::QB;
  using T = typename C::T;
  extern __shared__ __align__(1024) unsigned char smem[];
  Bars& B = *reinterpret_cast<Bars*>(smem + C::OFF_BAR);
  float2* stats = reinterpret_cast<float2*>(smem + C::OFF_STAT);  // [slot][row]: maximum, sum
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int per_tile = C::ROWS / p.group;  // tokens of a full row tile

  if (warp == NSW) {
    if (lane == 0) {
      for (int i = 0; i < NU; ++i) mbar_init(&B.full[i], 1), mbar_init(&B.empty[i], 1);
      for (int i = 0; i < 2; ++i) {
        mbar_init(&B.s_full[i], 1), mbar_init(&B.p_full[i], 4);
        mbar_init(&B.q_full[i], 1), mbar_init(&B.q_empty[i], 1);
      }
      for (int i = 0; i < kSegs; ++i) mbar_init(&B.seg_full[i], 1), mbar_init(&B.seg_empty[i], 2 + NSW);
      mbar_init(&B.pv_done, 1), mbar_init(&B.seg_done, 1), mbar_init(&B.o_free, NSW), mbar_init(&B.stat_full, NSW);
      fence_mbar_init();
    }
    __syncwarp();
  } else if (warp == NSW + 1) {
    tmem_alloc(&B.tmem, C::TMEM_COLS);
    tmem_relinquish();
  }
  wait_for_producer();

  // ---- the line: prefix items first, then every sequence's own items
  const int tok_lo = min(max(__ldg(p.qsl), 0), p.n), tok_hi = min(max(__ldg(p.qsl + p.b), tok_lo), p.n);
  const int plen = capped(__ldg(p.prefix_len), p.prefix_cap, p.err);
  const int ptiles = (plen + TK - 1) / TK;
  const int prow_tiles = plen > 0 ? (tok_hi - tok_lo + per_tile - 1) / per_tile : 0;
  const int last_tok = prow_tiles ? tok_hi - tok_lo - (prow_tiles - 1) * per_tile : 0;
  const int64_t pc_full = item_cost(ptiles, per_tile * p.group), pc_last = item_cost(ptiles, last_tok * p.group);
  const int64_t ptotal = prow_tiles ? ((prow_tiles - 1) * pc_full + pc_last) * p.hkv : 0;
  const int per_thread = (p.b + C::NTHREADS - 1) / C::NTHREADS;
  const int s_lo = min(tid * per_thread, p.b), s_hi = min(s_lo + per_thread, p.b);
  int64_t mine = 0;
  for (int s = s_lo; s < s_hi; ++s) mine += seq_cost<C::ROWS>(p, s, per_tile) * p.hkv;
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) B.scan[warp] = incl;
  tc_fence_before();
  __syncthreads();  // barriers, TMEM address and warp sums are visible
  tc_fence_after();
  int64_t before = 0, total = ptotal;
#pragma unroll
  for (int w = 0; w < C::NTHREADS / 32; ++w) {
    if (w < warp) before += B.scan[w];
    total += B.scan[w];
  }
  // no piece shorter than an item's start and one tile
  const int ctas = static_cast<int>(max64(1, min64(p.ctas, total / (kItemCost + kTileCost))));
  auto cut = [&](int c) { return total * c / ctas; };
  const int cta = blockIdx.x;
  const int64_t x0 = cta < ctas ? cut(cta) : total, x1 = cta < ctas ? cut(cta + 1) : total;
  const int64_t own_from = max64(x0 - ptotal, 0);  // where this CTA's own part starts
  const int64_t excl = before + incl - mine;
  if (mine > 0 && own_from >= excl && own_from < excl + mine) {
    int64_t at = excl;
    int s = s_lo;
    for (; s < s_hi; ++s) {
      const int64_t c = seq_cost<C::ROWS>(p, s, per_tile) * p.hkv;
      if (own_from < at + c) break;
      at += c;
    }
    B.start_seq = s, B.start_base = at;
  }
  __syncthreads();
  const uint32_t tmem = B.tmem;

  if (warp == NSW) {
    // ------------------------------------------------------------ TMA producer
    const int nch = TK / p.chunk;
    uint32_t u = 0;  // units issued
    bool ok = true;
    prefetch_tensormap(&kmap);
    for (int sg = 0; ok; ++sg) {
      ok = warp_wait(&B.seg_full[sg % kSegs], (sg / kSegs) & 1);
      if (!ok) break;
      const Seg s = B.seg[sg % kSegs];
      __syncwarp();
      if (lane == 0) mbar_arrive(&B.seg_empty[sg % kSegs]);
      if (s.part < 0) break;
      const int ntile = s.ke - s.kb;
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
      int ids[2] = {0, 0};
      int next = page(s.kb);
      for (int pos = 0; ok && pos < 2 * ntile; ++pos) {
        const bool is_v = pos != 0 && (pos == 2 * ntile - 1 || (pos & 1) == 0);
        const int j = pos == 0 ? 0 : pos == 2 * ntile - 1 ? ntile - 1 : is_v ? pos / 2 - 1 : (pos + 1) / 2;
        int id;
        if (is_v) {
          id = (j & 1) ? ids[1] : ids[0];
        } else {
          id = next;
          if (j & 1) ids[1] = id;
          else ids[0] = id;
          next = page(s.kb + j + 1);  // looked up one tile ahead
        }
        const int c3 = (((s.kb + j) * TK + lane * p.chunk) % p.block_size) / 8;
#pragma unroll
        for (int w = 0; w < KU; ++w, ++u) {
          const int slot = u % NU;
          if (u >= NU) ok = warp_wait(&B.empty[slot], ((u / NU) - 1) & 1);
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(&B.full[slot], C::UNIT);
          __syncwarp();
          if (lane < nch)
            tma_load_5d(smem + slot * C::UNIT + lane * p.chunk * (C::UC * 2), is_v ? &vmap : &kmap, &B.full[slot],
                        w * C::NCG, c3, id);
        }
      }
    }
    if (!ok && lane == 0) set_error(p.err, FOLD_DEVERR_TIMEOUT);
    // copies in flight land before exit
    for (uint32_t w = u > NU ? u - NU : 0; w < u; ++w) warp_wait(&B.full[w % NU], (w / NU) & 1);
  } else if (warp == NSW + 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      constexpr uint32_t idesc_s = idesc_of(C::F16, TK, 0);
      constexpr uint32_t idesc_o = idesc_of(C::F16, C::UC, 1);
      const uint32_t base = smem_u32(smem), q_base = base + C::OFF_Q;
      uint32_t u0 = 0, qu = 0;             // ring units and Q tiles of earlier segments
      uint32_t pcnt[2] = {0, 0};           // P tiles consumed per S buffer
      bool ok = true;
      int sg = 0;
      for (; ok; ++sg) {
        ok = mbar_wait(&B.seg_full[sg % kSegs], (sg / kSegs) & 1);
        if (!ok) break;
        const Seg s = B.seg[sg % kSegs];
        mbar_arrive(&B.seg_empty[sg % kSegs]);
        if (s.part < 0) break;
        const int ntile = s.ke - s.kb;
        const bool wide = s.rows > 128;  // the slots are row halves; else they alternate key tiles
        const int steps = wide ? 2 * ntile : ntile;
        auto qk = [&](int i) {
          const int b = i & 1, j = wide ? i >> 1 : i;
          const uint32_t quse = qu + (wide ? b : 0), qslot = quse % QB;
          if (wide ? i < 2 : i == 0) ok = ok && mbar_wait(&B.q_full[qslot], (quse / QB) & 1);
          const uint32_t u = u0 + k_pos(j) * KU;
          const uint32_t d = tmem + C::TMEM_S + b * TK;
#pragma unroll
          for (int w = 0; w < KU; ++w) {
            const uint32_t slot = (u + w) % NU;
            if (!wide || b == 0) ok = ok && mbar_wait(&B.full[slot], ((u + w) / NU) & 1);
            if (!ok) return;
            tc_fence_after();
#pragma unroll
            for (int kk = 0; kk < C::UC / 16; ++kk) {
              const uint32_t a = q_base + qslot * C::Q_TILE + (w * C::NCG + (kk >> 2)) * C::Q_CG + (kk & 3) * 32;
              const uint32_t kb = base + slot * C::UNIT + (kk >> 2) * 1024 + (kk & 3) * 32;
              tc_mma(d, smem_desc(a, 16, 1024, kSwizzle128), smem_desc(kb, 16, C::NCG * 1024, kSwizzle128), idesc_s,
                     w > 0 || kk > 0);
            }
          }
          tc_commit(&B.s_full[b]);
          if (!wide || b == 1)
            for (int w = 0; w < KU; ++w) tc_commit(&B.empty[(u + w) % NU]);
          if (i + (wide ? 2 : 1) >= steps) tc_commit(&B.q_empty[qslot]);
        };
        qk(0);
        if (ok && steps > 1) qk(1);
        for (int i = 0; ok && i < steps; ++i) {
          const int b = i & 1, j = wide ? i >> 1 : i;
          ok = mbar_wait(&B.p_full[b], pcnt[b] & 1);
          ++pcnt[b];
          // the accumulators of the last segment have been read
          if (ok && i == 0 && sg > 0) ok = mbar_wait(&B.o_free, (sg - 1) & 1);
          const uint32_t u = u0 + v_pos(j, ntile) * KU;
          const uint32_t a = tmem + C::TMEM_S + b * TK;
          const uint32_t o = tmem + C::TMEM_O + (NWG == 2 ? b * HD : 0);
          const bool first = NWG == 2 ? i < 2 : i == 0;
#pragma unroll
          for (int w = 0; w < KU; ++w) {
            const uint32_t slot = (u + w) % NU;
            if (!wide || b == 0) ok = ok && mbar_wait(&B.full[slot], ((u + w) / NU) & 1);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int ks = 0; ks < TK / 16; ++ks) {
              const uint32_t v = base + slot * C::UNIT + ks * 2 * C::NCG * 1024;
              tc_mma_ts(o + w * C::UC, a + ks * 8, smem_desc(v, 1024, C::NCG * 1024, kSwizzle128), idesc_o,
                        !first || ks > 0);
            }
          }
          if (!ok) break;
          if (NWG == 1) tc_commit(&B.pv_done);
          if (!wide || b == 1)
            for (int w = 0; w < KU; ++w) tc_commit(&B.empty[(u + w) % NU]);
          if (i + 2 < steps) qk(i + 2);
        }
        if (!ok) break;
        tc_commit(&B.seg_done);
        u0 += 2 * ntile * KU;
        qu += wide ? 2 : 1;
      }
      if (!ok) {  // let what was issued finish before TMEM goes
        set_error(p.err, FOLD_DEVERR_TIMEOUT);
        tc_commit(&B.seg_done);
        mbar_wait(&B.seg_done, sg & 1);
      }
    }
    __syncwarp();
  } else if (warp == NSW + 2) {
    // ------------------------------------------------------------ scheduler and Q loader
    uint32_t qu = 0;
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
      if (s.part < 0) return;
      for (int r0 = 0; r0 < s.rows; r0 += 128, ++qu) {
        const uint32_t slot = qu % QB;
        if (qu >= QB) ok = warp_wait(&B.q_empty[slot], ((qu / QB) - 1) & 1);
        if (!ok) return;
        const int nr = min(128, s.rows - r0);
        const uint32_t dst = smem_u32(smem + C::OFF_Q + slot * C::Q_TILE);
        for (int e = lane; e < nr * (HD / 8); e += 32) {
          const int r = e / (HD / 8), c = e - r * (HD / 8);
          const int x = (r0 + r) / p.group, g = r0 + r - x * p.group;
          const T* src = static_cast<const T*>(p.q) + (s.tok0 + x) * p.q_st + (s.head * p.group + g) * p.q_sh + c * 8;
          cp_async_16(dst + (c >> 3) * C::Q_CG + r * 128 + (((c & 7) ^ (r & 7)) << 4), src, 16);
        }
        cp_async_wait_all();
        fence_proxy_async();  // Q is read by the tensor cores
        __syncwarp();
        if (lane == 0) mbar_arrive(&B.q_full[slot]);
      }
    };
    // one item: s without its tile range; at: its place on the line
    auto item = [&](Seg s, int ntok, int64_t at) {
      const int tiles = (s.limit + TK - 1) / TK, w = tile_cost(s.rows);
      // key tiles of this item that lie before place x of the line
      auto tiles_before = [&](int64_t x) {
        const int64_t y = x - at - kItemCost + w / 2;
        return y <= 0 ? 0 : static_cast<int>(min64(y / w, tiles));
      };
      s.kb = tiles_before(x0), s.ke = cta + 1 == ctas ? tiles : tiles_before(x1);
      if (s.kb < s.ke) publish(s);
      if (at >= x0) {  // the item starts here: note the CTAs that hold its tiles
        int c0 = cta, cnt = 0;
        if (tiles > 0) {
          auto upto = [&](int c) { return c + 1 >= ctas ? tiles : tiles_before(cut(c + 1)); };
          while (upto(c0) == 0) ++c0;
          int c1 = static_cast<int>(min64(ctas - 1, (at + kItemCost + static_cast<int64_t>(tiles) * w) * ctas / total));
          c1 = max(c1, c0);
          while (c1 > c0 && tiles_before(cut(c1)) >= tiles) --c1;
          cnt = c1 - c0 + 1;
        }
        for (int x = lane; x < ntok; x += 32)
          p.plan[(static_cast<int64_t>(s.part) * p.n + s.tok0 + x) * p.hkv + s.head] = make_int4(c0, cnt, s.tok0, 0);
      }
    };
    if (x0 < x1) {
      Seg s{};
      if (x0 < ptotal) {
        const int64_t row_cost = pc_full * p.hkv;
        int rt = static_cast<int>(min64(x0 / row_cost, prow_tiles - 1));
        const int64_t in_row = x0 - rt * row_cost;
        int h = static_cast<int>(min64(in_row / (rt + 1 < prow_tiles ? pc_full : pc_last), p.hkv - 1));
        for (; ok && rt < prow_tiles; ++rt, h = 0) {
          const int ntok = rt + 1 < prow_tiles ? per_tile : last_tok;
          const int64_t c = rt + 1 < prow_tiles ? pc_full : pc_last;
          for (; ok && h < p.hkv; ++h) {
            const int64_t at = rt * row_cost + h * c;
            if (at >= x1) break;
            s.part = 0, s.seq = 0, s.head = h, s.tok0 = tok_lo + rt * per_tile, s.rows = ntok * p.group;
            s.limit = plen, s.lim0 = plen, s.lim_step = 0;
            item(s, ntok, at);
          }
          if (h < p.hkv) break;
        }
      }
      if (x1 > ptotal) {
        int64_t at = ptotal + B.start_base;
        for (int q = B.start_seq; ok && q < p.b && at < x1; ++q) {
          int first, last;
          seq_rows(p, q, first, last);
          const int m = capped(__ldg(p.own_lens + q), p.own_cap, p.err);
          for (int t0 = first; ok && t0 < last && at < x1; t0 += per_tile) {
            const int ntok = min(per_tile, last - t0);
            s.part = 1, s.seq = q, s.tok0 = t0, s.rows = ntok * p.group, s.lim_step = p.causal ? 1 : 0;
            own_limits(p, first, last, m, t0, ntok, s.limit, s.lim0);
            const int64_t c = item_cost((s.limit + TK - 1) / TK, s.rows);
            int h = 0;
            if (at + c * p.hkv <= x0) h = p.hkv;  // wholly before this CTA's piece
            else if (x0 > at) h = static_cast<int>((x0 - at) / c);
            for (; ok && h < p.hkv && at + h * c < x1; ++h) {
              s.head = h;
              item(s, ntok, at + h * c);
            }
            at += c * p.hkv;
          }
        }
      }
    }
    if (ok) {
      Seg s{};
      s.part = -1;
      publish(s);
    }
    if (!ok && lane == 0) set_error(p.err, FOLD_DEVERR_TIMEOUT);
  } else if (warp < NSW) {
    // ------------------------------------------------------------ softmax warps
    const int wg = warp >> 2, row = (warp & 3) * 32 + lane;  // row of the slot = TMEM lane
    const uint32_t lane_addr = static_cast<uint32_t>((warp & 3) * 32) << 16;
    uint32_t scnt[2] = {0, 0};  // S tiles read per buffer
    uint32_t u0 = 0, pv = 0;
    bool ok = true;
    for (int sg = 0; ok; ++sg) {
      ok = warp_wait(&B.seg_full[sg % kSegs], (sg / kSegs) & 1);
      if (!ok) break;
      const Seg s = B.seg[sg % kSegs];
      __syncwarp();
      if (lane == 0) mbar_arrive(&B.seg_empty[sg % kSegs]);
      if (s.part < 0) break;
      const int ntile = s.ke - s.kb;
      const bool wide = s.rows > 128;
      const int r = row + (wide ? wg * 128 : 0);
      const bool live = r < s.rows;
      const int x = live ? r / p.group : 0;
      const int lim = live ? min(s.limit, s.lim0 + x * s.lim_step) : 0;
      const bool warp_live = __any_sync(0xffffffffu, live);
      const int warp_lim = __reduce_min_sync(0xffffffffu, live ? lim : 0x7fffffff);
      float m = -INFINITY, l = 0.f;
      bool empty_o = true;
      for (int j = (NWG == 2 && !wide) ? wg : 0; j < ntile; j += (NWG == 2 && !wide) ? 2 : 1) {
        const int b = NWG == 2 ? wg : j & 1;
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
              // accumulator the last tile's may still be running
              if (NWG == 1) ok = warp_wait(&B.pv_done, (pv + j - 1) & 1);
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
        if (vk < TK && vk % p.chunk != 0 && (!wide || wg == 0)) {
          const int vend = (vk / p.chunk + 1) * p.chunk;
          const uint32_t u = u0 + v_pos(j, ntile) * KU;
#pragma unroll
          for (int w = 0; w < KU; ++w) {
            ok = ok && warp_wait(&B.full[(u + w) % NU], ((u + w) / NU) & 1);
            if (!ok) break;
            unsigned char* vt = smem + ((u + w) % NU) * C::UNIT;
            for (int e = row; e < (vend - vk) * C::NCG * 8; e += 128) {
              const int vr = vk + e / (C::NCG * 8), c = e % (C::NCG * 8);
              *reinterpret_cast<uint4*>(vt + (vr >> 3) * C::NCG * 1024 + (c >> 3) * 1024 + (vr & 7) * 128 +
                                        (c & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
          }
          if (!ok) break;
          fence_proxy_async();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&B.p_full[b]);
      }
      if (!ok) break;
      u0 += 2 * ntile * KU;
      pv += ntile;

      // ---- the segment's partial: O / l and lse
      ok = warp_wait(&B.seg_done, sg & 1);
      if (!ok) break;
      tc_fence_after();
      const bool joined = NWG == 2 && !wide;  // both slots hold every row's keys
      float ws[2] = {1.f, 0.f};
      if (joined) {
        stats[wg * 128 + row] = make_float2(m, l);
        __syncwarp();
        if (lane == 0) mbar_arrive(&B.stat_full);
        ok = warp_wait(&B.stat_full, sg & 1);
        if (!ok) break;
        const float2 a = stats[row], c = stats[128 + row];
        m = fmaxf(a.x, c.x);
        const float mz = m == -INFINITY ? 0.f : m;
        ws[0] = fast_exp2(a.x - mz), ws[1] = fast_exp2(c.x - mz);
        l = a.y * ws[0] + c.y * ws[1];
      } else if (NWG == 2) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&B.stat_full);  // keeps the barrier's phase with the segments'
      }
      const bool some = l > 0.f;
      const float inv = some ? 1.f / l : 0.f;
      ws[0] *= inv, ws[1] *= inv;
      const int tok = s.tok0 + x, hqi = s.head * p.group + r - x * p.group;
      const int64_t prim = (static_cast<int64_t>(s.part) * p.n + tok) * p.hq + hqi;
      const int64_t cont = static_cast<int64_t>(cta) * C::ROWS + r;
      float* od = s.kb == 0 ? p.o_prim + prim * HD : p.o_cont + cont * HD;
      if (live && (!joined || wg == 0))
        (s.kb == 0 ? p.lse_prim + prim : p.lse_cont + cont)[0] =
            some ? (m - C::SHIFT + __log2f(l)) * kLn2 : (l == 0.f ? -INFINITY : l);
      if (warp_live) {
        // joined slots: each warpgroup writes half of the columns of both accumulators' sum
        const int c_lo = joined ? wg * (HD / 2) : 0, c_hi = joined ? c_lo + HD / 2 : HD;
        const bool two = joined && ntile > 1;
        const uint32_t oa = tmem + C::TMEM_O + ((NWG == 2 && wide) ? wg * HD : 0) + lane_addr;
#pragma unroll 1
        for (int c = c_lo; c < c_hi; c += 16) {
          float o[16];
          tmem_ld16(oa + c, o);
#pragma unroll
          for (int k = 0; k < 16; ++k) o[k] = some ? o[k] * ws[0] : l;  // l: 0, or the NaN of the row
          if (two) {
            float o2[16];
            tmem_ld16(oa + HD + c, o2);
#pragma unroll
            for (int k = 0; k < 16; ++k) o[k] += some ? o2[k] * ws[1] : 0.f;
          }
          if (live) {
#pragma unroll
            for (int k = 0; k < 16; k += 4)
              *reinterpret_cast<float4*>(od + c + k) = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&B.o_free);
    }
    if (!ok && lane == 0) set_error(p.err, FOLD_DEVERR_TIMEOUT);
  }

  tc_fence_before();
  __syncthreads();
  if (warp == NSW + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

// Joins the partials of one row: its prefix item's and its own item's. One warp per (token, head).
template <int HD, class T, int ROWS>
__global__ void __launch_bounds__(128) prefix_merge_kernel(const PrefixParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t row = blockIdx.x * 4ll + (threadIdx.x >> 5);
  const int tok = static_cast<int>(row / p.hq), h = static_cast<int>(row - static_cast<int64_t>(tok) * p.hq);
  if (tok >= p.n || tok < p.qsl[0] || tok >= p.qsl[p.b]) return;
  wait_for_producer();
  constexpr int V = HD / 32;
  float acc[V], m = -INFINITY, z = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.f;
  auto add = [&](float lse, const float* o) {
    if (lse == -INFINITY) return;
    const float mn = fmaxf(m, lse), f = __expf(m - mn), w = __expf(lse - mn);
    m = mn, z = z * f + w;
    float x[V];
    if constexpr (V == 2) {
      const float2 a = reinterpret_cast<const float2*>(o)[lane];
      x[0] = a.x, x[1] = a.y;
    } else {
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        const float4 a = reinterpret_cast<const float4*>(o)[lane * (V / 4) + i / 4];
        x[i] = a.x, x[i + 1] = a.y, x[i + 2] = a.z, x[i + 3] = a.w;
      }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = acc[i] * f + w * x[i];
  };
  const int hk = h / p.group, g = h - hk * p.group;
#pragma unroll 1
  for (int part = (p.prefix_len[0] > 0 && p.prefix_cap > 0) ? 0 : 1; part < 2; ++part) {
    const int64_t tr = static_cast<int64_t>(part) * p.n + tok;
    const int4 plan = p.plan[tr * p.hkv + hk];
    if (plan.y < 1) continue;
    add(p.lse_prim[tr * p.hq + h], p.o_prim + (tr * p.hq + h) * HD);
    const int r = (tok - plan.z) * p.group + g;
    for (int c = plan.x + 1; c < plan.x + plan.y; ++c) {
      const int64_t at = static_cast<int64_t>(c) * ROWS + r;
      add(p.lse_cont[at], p.o_cont + at * HD);
    }
  }
  const float inv = z > 0.f ? 1.f / z : 0.f;
  T* out = static_cast<T*>(p.out) + tok * p.o_st + h * p.o_sh + lane * V;
  uint32_t w[V / 2];
#pragma unroll
  for (int i = 0; i < V; i += 2) w[i / 2] = pack2<T>(z == z ? acc[i] * inv : z, z == z ? acc[i + 1] * inv : z);
  if constexpr (V == 2) *reinterpret_cast<uint32_t*>(out) = w[0];
  else if constexpr (V == 4) *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[1]);
  else *reinterpret_cast<uint4*>(out) = make_uint4(w[0], w[1], w[2], w[3]);
  if (lane == 0 && p.lse)
    p.lse[static_cast<int64_t>(h) * p.n + tok] = z > 0.f ? m + logf(z) : (z == 0.f ? -INFINITY : z);
}

// ---------------------------------------------------------------- host
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
  w.bytes = w.lse_cont + up(ctas * rows * 4);
  return w;
}

int ctas_of_device() {
  const int sms = device_sm_count();
  return sms > 0 ? sms : 148;
}

// 5-D map of a K or V plane: 64 columns, 8 slots, 64-column groups, groups of 8 slots, and blocks
// and heads as one index (in units of the smaller of their strides). A box of `chunk` slots lands
// as [group of 8 slots][64-column group][8 rows of 128 bytes], 128-byte swizzled: consecutive
// chunks stack to a tile whose 8-row groups have one stride, whatever the page size.
int plane_map(const void* base, int hd, int box_cols, int block_size, int chunk, int64_t slot, int64_t unit,
              int64_t count, bool f16, CUtensorMap* out) {
  static const PFN_cuTensorMapEncodeTiled_v12000 encode = [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult r;
    const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &r);
    return e == cudaSuccess && r == cudaDriverEntryPointSuccess
               ? reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn)
               : nullptr;
  }();
  if (!encode) return fail(FOLD_ERR_TENSOR_MAP, "prefix read: cuTensorMapEncodeTiled is not available from the driver");
  const cuuint64_t dims[5] = {64, 8, static_cast<cuuint64_t>(hd / 64), static_cast<cuuint64_t>(block_size / 8),
                              static_cast<cuuint64_t>(count)};
  const cuuint64_t strides[4] = {static_cast<cuuint64_t>(slot) * 2, 128, static_cast<cuuint64_t>(slot) * 16,
                                 static_cast<cuuint64_t>(unit) * 2};
  const cuuint32_t box[5] = {64, 8, static_cast<cuuint32_t>(box_cols / 64), static_cast<cuuint32_t>(chunk / 8), 1};
  const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
  const CUresult r = encode(out, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5,
                            const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(FOLD_ERR_TENSOR_MAP, "prefix read: cuTensorMapEncodeTiled failed with CUresult " + std::to_string(r));
  return FOLD_OK;
}

template <int HD, class T>
int launch_prefix(const PrefixParams& p, const void* k, const void* v, int64_t slot, int64_t unit, cudaStream_t stream) {
  using C = Cfg<HD, T>;
  CUtensorMap kmap, vmap;
  const int64_t count = p.oob;
  if (int s = plane_map(k, HD, C::UC, p.block_size, p.chunk, slot, unit, count, C::F16, &kmap)) return s;
  if (int s = plane_map(v, HD, C::UC, p.block_size, p.chunk, slot, unit, count, C::F16, &vmap)) return s;
  static std::atomic<uint64_t> configured{0};
  if (int s = allow_smem(prefix_read_kernel<C>, C::SMEM, configured, "cudaFuncSetAttribute(prefix_read)")) return s;
  if (int s = launch_behind(prefix_read_kernel<C>, dim3(p.ctas), C::NTHREADS, C::SMEM, stream, "prefix_read_kernel",
                            kmap, vmap, p))
    return s;
  const int64_t rows = static_cast<int64_t>(p.n) * p.hq;
  return launch_behind(prefix_merge_kernel<HD, T, C::ROWS>, dim3(static_cast<unsigned>((rows + 3) / 4)), 128, 0, stream,
                       "prefix_merge_kernel", p);
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
  if (!q || !qsl || !own_lens || !prefix_len || !k_cache || !v_cache || !prefix_table || !block_tables || !out)
    return fail(FOLD_ERR_INVALID_ARGUMENT, "prefix read: null pointer");
  if (!aligned16(q) || !aligned16(out) || !aligned16(k_cache) || !aligned16(v_cache) || q_stride_tok % 8 ||
      q_stride_head % 8 || o_stride_tok % 8 || o_stride_head % 8 || cache_stride_block % 8 || cache_stride_head % 8 ||
      cache_stride_slot % 8)
    return fail(FOLD_ERR_ALIGNMENT, "prefix read: rows of q, out and the cache must start on 16-byte boundaries");
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
  p.n = n, p.hq = hq, p.hkv = hkv, p.group = hq / hkv, p.ctas = ctas, p.err = err;
  char* ws = static_cast<char*>(workspace);
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
