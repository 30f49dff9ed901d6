// Attention over whole prompts (fold_prompt_read): sequences of different lengths packed one behind the
// other, heads in groups that share keys and values, causal or with a window.
//
// Mathematics. With x_rj = scale q_r.k_j for the keys j in [r - left, r + right] of r's sequence,
// o_r = sum_j e^(x_rj - lse_r) v_j and lse_r = log sum_j e^(x_rj). One pass over the keys keeps a running
// maximum m and sum l of each row and rescales what was summed when the maximum rises.
//
// Rounding. Logits, maxima, sums and O are float32; P is rounded once to the type of V (the sums are of the
// unrounded P), the result once: 0.0020 (bf16) or 0.00026 (fp16) of the output's norm against 64 bits, where rounding
// the output alone is 0.0016 and 0.0002.
//
// Measured (bf16, head size 128, 32 query and 8 KV heads, causal; the GPU's time): one sequence of 16384 tokens
// 1.99 ms in a long run (1107 TFLOP/s, 0.79 of the measured sustained GEMM rate; the board is at its 1000 W), 1.74 ms
// a dozen times in a row, of 8192 tokens 475 us (1157 TFLOP/s), of 2048 52 us, of 512 15 us, of 40 9 us; 24 sequences
// of up to 2100 tokens 452 us. A tile's turn is a chain (softmax 1500-1600 cycles, P V and the next S 1024) which the other tile
// fills: 1840 cycles a tile for 1024 of products. Short sequences lose half of the diagonal tiles and some 4 us a
// block's tile for its start and its result. Exponentials by polynomial beside the special unit were slower (8192
// tokens 537 us for 474).
#include "prompt.cuh"
#include "tcgen05.cuh"

namespace fold {
namespace {
using namespace prompt;

struct ReadParams {
  Shape s;
  Rows q, k, v, out;
  float* lse;
  int* err;
};

// ---------------------------------------------------------------- mma.sync, head sizes from 136 to 256
// A CTA of eight warps takes 128 rows of one head, a warp 16 of them; keys in tiles of 64, two stages.
template <int DP, class T>
__global__ void __launch_bounds__(256) prompt_read_mma_kernel(const ReadParams p) {
  using Sm = SmemTile<DP>;
  // weights in fp16 are held 2^10 up: small ones of many keys stay above its smallest step
  constexpr float kShift = std::is_same<T, __half>::value ? 10.f : 0.f;
  extern __shared__ __align__(1024) unsigned char smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const uint32_t sq = smem_u32(smem), sk = sq + 2 * Sm::BYTES, sv = sk + 2 * Sm::BYTES;
  wait_for_producer();
  Tile t;
  if (!find_tile<128>(p.s, gridDim.x - 1 - blockIdx.x, t)) return;  // the last rows see most keys: first
  const int h = blockIdx.y, hk = h / p.s.group, hd = p.s.hd;
  int lo, hi;
  keys_of(p.s, t.len, t.row0, min(t.row0 + 128, t.len), lo, hi);
  const int kb = lo / 64, ke = (hi + 63) / 64;
  stage_rows<DP, 256, 128>(sq, p.q, t.first, t.len, t.row0, h, hd);
  stage_rows<DP, 256>(sk, p.k, t.first, t.len, kb * 64, hk, hd);
  stage_rows<DP, 256>(sv, p.v, t.first, t.len, kb * 64, hk, hd);
  cp_commit();
  float o[DP / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int c = 0; c < DP / 8; ++c)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[c][e] = 0.f;
  int klo[2], khi[2];  // the keys of this thread's two rows
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = t.row0 + warp * 16 + e * 8 + g;
    keys_of(p.s, t.len, r, r + 1, klo[e], khi[e]);
  }
  for (int j = kb; j < ke; ++j) {
    const int st = (j - kb) & 1;
    if (j + 1 < ke) {
      stage_rows<DP, 256>(sk + (st ^ 1) * Sm::BYTES, p.k, t.first, t.len, (j + 1) * 64, hk, hd);
      stage_rows<DP, 256>(sv + (st ^ 1) * Sm::BYTES, p.v, t.first, t.len, (j + 1) * 64, hk, hd);
    }
    cp_commit();
    cp_wait<1>();
    __syncthreads();
    float x[8][4];
#pragma unroll
    for (int i = 0; i < 32; ++i) (&x[0][0])[i] = 0.f;
    product_t<DP, T>(x, sq, warp * 16, sk + st * Sm::BYTES);
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = j * 64 + i * 8 + 2 * t4 + (e & 1);
        x[i][e] = key >= klo[e >> 1] && key < khi[e >> 1] ? x[i][e] * p.s.scale_log2 : -INFINITY;
        top[e >> 1] = fmaxf(top[e >> 1], x[i][e]);
      }
    uint32_t pa[4][4];
    float f[2], neg[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 1));
      top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 2));
      const float up = fmaxf(m[e], top[e]);
      f[e] = up == -INFINITY ? 1.f : fast_exp2(m[e] - up);
      m[e] = up, l[e] *= f[e], neg[e] = up == -INFINITY ? 0.f : kShift - up;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float a = fast_exp2(x[i][2 * e] + neg[e]), b = fast_exp2(x[i][2 * e + 1] + neg[e]);
        l[e] += a + b;
        pa[i >> 1][(i & 1) * 2 + e] = pack_pair<T>(a, b);  // one rounding of P to the type of V
      }
#pragma unroll
    for (int c = 0; c < DP / 8; ++c) o[c][0] *= f[0], o[c][1] *= f[0], o[c][2] *= f[1], o[c][3] *= f[1];
    product<DP, DP / 16, T>(o, pa, sv + st * Sm::BYTES, 0);
    __syncthreads();
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
    const int r = t.row0 + warp * 16 + e * 8 + g;
    if (r >= t.len) continue;
    const float inv = l[e] > 0.f ? 1.f / l[e] : (l[e] == 0.f ? 0.f : l[e]);  // a NaN reaches the output
    T* out = static_cast<T*>(p.out.ptr) + (t.first + r) * p.out.tok + h * p.out.head;
#pragma unroll
    for (int c = 0; c < DP / 8; ++c)
      if (c * 8 < hd) *reinterpret_cast<uint32_t*>(out + c * 8 + 2 * t4) = pack_pair<T>(o[c][2 * e] * inv, o[c][2 * e + 1] * inv);
    if (p.lse && t4 == 0)
      p.lse[static_cast<int64_t>(h) * p.s.n + t.first + r] =
          l[e] > 0.f ? (m[e] - kShift + __log2f(l[e])) * kLn2 : (l[e] == 0.f ? -INFINITY : l[e]);
  }
}

template <int DP, class T>
int launch_mma(const ReadParams& p, cudaStream_t stream) {
  constexpr int smem = 6 * SmemTile<DP>::BYTES;
  static std::atomic<uint64_t> configured{0};
  if (int s = allow_smem(prompt_read_mma_kernel<DP, T>, smem, configured, "cudaFuncSetAttribute(prompt_read)")) return s;
  return launch_behind(prompt_read_mma_kernel<DP, T>, dim3(tile_numbers(p.s.n, p.s.b, 128), p.s.hq), 256, smem, stream,
                       "prompt_read_mma_kernel", p);
}

// ---------------------------------------------------------------- tcgen05, head sizes up to 128
// Heads of other sizes than 64 and 128 are loaded with zeros behind them (outside of the maps).
// A CTA takes two tiles of 128 rows that read the same keys: two heads of a group, or, where a group has an
// odd number of heads, 256 rows of one. Warps with fixed roles:
//   two softmax warpgroups, one a tile: a thread owns a row; S from tensor memory, mask, maximum, P = 2^(y - m)
//     rounded to the type of V and stored over S; O in tensor memory rescaled when a maximum rose; at the end
//     O / l and lse go out;
//   K and V by TMA into a ring, Q by TMA, the MMAs (S = Q K^T and O += P V, P from tensor memory), and a
//   scheduler that asks for the next tile.
// While one tile is in its softmax the tensor cores work for the other: P V of its last keys, then S of its next.
template <int HD_, class T_>
struct ReadCfg {
  using T = T_;
  static constexpr int HD = HD_, NTHREADS = 384, NSW = 8;
  static constexpr int NCG = HD / 64;              // groups of 64 columns: a row of one is a swizzled 128 bytes
  static constexpr int CG = 128 * 128;             // bytes of a group of a 128-row tile
  static constexpr int UNIT = NCG * CG;            // a Q, K or V tile
  static constexpr int QB = HD == 64 ? 2 : 1;      // Q tiles a warpgroup: at 64 the next one loads early
  static constexpr int MISC = 1024;
  static constexpr int FIT = (232448 - MISC - 2 * QB * UNIT) / UNIT;
  static constexpr int NU = FIT > 8 ? 8 : FIT;     // K and V tiles in the ring
  static constexpr int OFF_Q = NU * UNIT, OFF_BAR = OFF_Q + 2 * QB * UNIT, SMEM = OFF_BAR + MISC;
  static constexpr int TMEM_S = 0, TMEM_O = 256;
  static constexpr bool F16 = std::is_same<T, __half>::value;
  // fp16 holds P up by 2^7, so that small weights stay above its smallest step; it stays below 2^15
  static constexpr float SHIFT = F16 ? 7.f : 0.f;
  static_assert(SMEM <= 232448 && NU >= 5, "shared memory");
};

// A row's maximum only moves when a logit passes it by more than this (log2 units).
constexpr float kRowRaise = 8.f;

// Registers a thread: at launch (the build checks it), then of the softmax warps and of the others.
constexpr int kLaunchRegs = 168, kSoftmaxRegs = 208, kOtherRegs = 88;
static_assert(2 * kSoftmaxRegs + kOtherRegs <= 3 * kLaunchRegs, "a share that is not there is waited for");

struct ReadItem {
  int first, len, hk;       // -1 len: no more
  int row0[2], head[2], kb[2], ke[2];
};
constexpr int kItems = 3;

struct ReadBars {
  uint64_t full[8], empty[8];
  uint64_t s_full[2], p_full[2], done[2], o_free[2];
  uint64_t q_full[4], q_empty[4];
  uint64_t item_full[kItems], item_empty[kItems], asked, drained;
  uint4 answer;
  uint32_t tmem;
  ReadItem item[kItems];
};
static_assert(sizeof(ReadBars) <= 1024, "barriers fit their place");

template <class C>
__global__ void __launch_bounds__(C::NTHREADS, 1)
    prompt_read_tc_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                          const __grid_constant__ CUtensorMap vmap, const ReadParams p, const int pair_heads) {
  using namespace tc;
  using T = typename C::T;
  constexpr int HD = C::HD, NU = C::NU, NSW = C::NSW, QB = C::QB;
  extern __shared__ __align__(1024) unsigned char smem[];
  ReadBars& B = *reinterpret_cast<ReadBars*>(smem + C::OFF_BAR);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (warp == NSW) {
    if (lane == 0) {
      for (int i = 0; i < NU; ++i) mbar_init(&B.full[i], 1), mbar_init(&B.empty[i], 1);
      for (int i = 0; i < 2; ++i)
        mbar_init(&B.s_full[i], 1), mbar_init(&B.p_full[i], 4), mbar_init(&B.done[i], 1), mbar_init(&B.o_free[i], 4);
      for (int i = 0; i < 2 * QB; ++i) mbar_init(&B.q_full[i], 1), mbar_init(&B.q_empty[i], 1);
      for (int i = 0; i < kItems; ++i) mbar_init(&B.item_full[i], 1), mbar_init(&B.item_empty[i], 3 + NSW);
      mbar_init(&B.asked, 1), mbar_init(&B.drained, 1);
      fence_mbar_init();
    }
    __syncwarp();
  } else if (warp == NSW + 1) {
    tmem_alloc(&B.tmem, 512);
    tmem_relinquish();
  }
  wait_for_producer();
  tc_fence_before();
  __syncthreads();  // barriers and the address of tensor memory are visible
  tc_fence_after();
  const uint32_t tmem = B.tmem;
  // Every role walks the items in the scheduler's order.
  auto next_item = [&](int i, ReadItem& it) {
    if (!warp_wait(&B.item_full[i % kItems], (i / kItems) & 1)) return false;
    it = B.item[i % kItems];
    __syncwarp();
    if (lane == 0) mbar_arrive(&B.item_empty[i % kItems]);
    return true;
  };

  if (warp < NSW) {
    regs_up<kSoftmaxRegs>();
    // ------------------------------------------------------------ softmax
    const int wg = warp >> 2, row = (warp & 3) * 32 + lane;  // lane of tensor memory
    const uint32_t lane_addr = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t sa = tmem + C::TMEM_S + wg * 128 + lane_addr, oa = tmem + C::TMEM_O + wg * HD + lane_addr;
    uint32_t steps = 0, items = 0, tile0 = 0;  // of this warpgroup; tile0: key tiles of the CTA's earlier items
    bool ok = true;
    for (int i = 0; ok; ++i) {
      ReadItem it;
      ok = next_item(i, it);
      if (!ok || it.len < 0) break;
      const int kb = min(it.kb[0], it.kb[1]), ke = max(it.ke[0], it.ke[1]);
      const int r = it.row0[wg] + row;
      const bool live = r < it.len;
      int lo, hi;
      keys_of(p.s, it.len, min(r, it.len - 1), min(r, it.len - 1) + 1, lo, hi);
      const int warp_lo = __reduce_max_sync(0xffffffffu, lo), warp_hi = __reduce_min_sync(0xffffffffu, hi);
      float m = -INFINITY, l = 0.f;
      for (int j = it.kb[wg]; j < it.ke[wg]; ++j) {
        ok = warp_wait(&B.s_full[wg], steps++ & 1);
        if (!ok) break;
        tc_fence_after();
        const int key0 = j * 128;
        float v[128];
#pragma unroll
        for (int c = 0; c < 128; c += 32) tmem_ld32(sa + c, v + c);
        tmem_wait_ld();
        if (key0 < warp_lo || key0 + 128 > warp_hi) {
          const int a = lo - key0;
          const uint32_t seen = static_cast<uint32_t>(hi - lo);
#pragma unroll
          for (int c = 0; c < 128; ++c) v[c] = static_cast<uint32_t>(c - a) < seen ? v[c] : -INFINITY;
        }
        float mx[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
        for (int c = 4; c < 128; c += 8) {
#pragma unroll
          for (int k = 0; k < 4; ++k) mx[k] = c + 4 + k < 128 ? fmax3(mx[k], v[c + k], v[c + 4 + k]) : fmaxf(mx[k], v[c + k]);
        }
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.s.scale_log2;
        const bool raise = top > m + kRowRaise || (m == -INFINITY && top > m);
        if (__any_sync(0xffffffffu, raise)) {
          const float mn = raise ? top : m;
          const float f = raise ? fast_exp2(m - mn) : 1.f;  // 0 for the first keys
          l *= f, m = mn;
          if (j > it.kb[wg]) {  // the accumulator holds the products up to the last tile: S of this one came behind
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
        for (int c = 0; c < 128; c += 32) {
          uint32_t w[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            float a = v[c + 2 * k], d = v[c + 2 * k + 1];
            ffma2(a, d, p.s.scale_log2, neg, neg);
            a = fast_exp2(a), d = fast_exp2(d);
            fadd2(l0, l1, l0, l1, a, d);
            w[k] = pack_pair<T>(a, d);  // one rounding of P to the type of V
          }
          tmem_st16(sa + c / 2, w);
        }
        l += l0 + l1;
        tmem_wait_st();
        // values behind the sequence's end belong to others (NaN included): zeros before the tensor cores
        // read them. The warpgroup whose P V comes first sees to it.
        const int vk = it.len - key0;
        if (vk < 128 && (wg == 0 || j < it.kb[0] || j >= it.ke[0])) {
          const uint32_t u = 2 * (tile0 + j - kb) + 1;
          ok = warp_wait(&B.full[u % NU], (u / NU) & 1);
          if (!ok) break;
          unsigned char* vt = smem + (u % NU) * C::UNIT;
          for (int e = row; e < (128 - vk) * C::NCG * 8; e += 128) {
            const int x = e / (C::NCG * 8), c = e % (C::NCG * 8);
            *reinterpret_cast<uint4*>(vt + (c >> 3) * C::CG + (vk + x) * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&B.p_full[wg]);
      }
      tile0 += ke - kb;
      if (!ok) break;
      if (it.kb[wg] >= it.ke[wg]) continue;  // no tile for this warpgroup
      ok = warp_wait(&B.done[wg], items++ & 1);
      if (!ok) break;
      tc_fence_after();
      const bool some = l > 0.f, wide = rows_on_32(p.out);
      const float inv = some ? 1.f / l : 0.f;
      T* out = static_cast<T*>(p.out.ptr) + static_cast<int64_t>(it.first + r) * p.out.tok + it.head[wg] * p.out.head;
#pragma unroll 1
      for (int c = 0; c < p.s.hd; c += 32) {
        float o[32];
        __syncwarp();
        tmem_ld32(oa + c, o);
        tmem_wait_ld();
        if (live) {
          uint32_t w[16];
#pragma unroll
          for (int k = 0; k < 16; ++k)  // no key: l is 0; a NaN sum reaches the output
            w[k] = some ? pack_pair<T>(o[2 * k] * inv, o[2 * k + 1] * inv) : pack_pair<T>(l, l);
          store_row16(out + c, w, wide, p.s.hd - c);
          store_row16(out + c + 16, w + 8, wide, p.s.hd - c - 16);
        }
      }
      if (live && p.lse)
        p.lse[static_cast<int64_t>(it.head[wg]) * p.s.n + it.first + r] =
            some ? (m - C::SHIFT + __log2f(l)) * kLn2 : (l == 0.f ? -INFINITY : l);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&B.o_free[wg]);
    }
    if (!ok && lane == 0) set_error(p.err, FOLD_DEVERR_TIMEOUT);
  } else {
    regs_down<kOtherRegs>();
    if (warp == NSW) {
      // ------------------------------------------------------------ K and V
      uint32_t u = 0;
      bool ok = true;
      prefetch_tensormap(&kmap);
      prefetch_tensormap(&vmap);
      auto load = [&](const CUtensorMap* map, int hk, int row) {
        const uint32_t slot = u % NU;
        if (u >= NU) ok = warp_wait(&B.empty[slot], (u / NU - 1) & 1);
        if (!ok) return;
        if (lane == 0) {
          mbar_arrive_expect_tx(&B.full[slot], C::UNIT);
#pragma unroll
          for (int c = 0; c < C::NCG; ++c)
            tma_load_3d_plain(smem + slot * C::UNIT + c * C::CG, map, &B.full[slot], c * 64, hk, row);
        }
        __syncwarp();
        ++u;
      };
      for (int i = 0; ok; ++i) {
        ReadItem it;
        ok = next_item(i, it);
        if (!ok || it.len < 0) break;
        const int kb = min(it.kb[0], it.kb[1]), ke = max(it.ke[0], it.ke[1]);
        for (int j = kb; ok && j < ke; ++j) {
          load(&kmap, it.hk, it.first + j * 128);
          if (ok) load(&vmap, it.hk, it.first + j * 128);
        }
      }
      if (!ok && lane == 0) set_error(p.err, FOLD_DEVERR_TIMEOUT);
      for (uint32_t w = u > NU ? u - NU : 0; w < u; ++w) warp_wait(&B.full[w % NU], (w / NU) & 1);  // copies land before exit
    } else if (warp == NSW + 1) {
      // ------------------------------------------------------------ MMAs
      constexpr uint32_t idesc_s = idesc_of(C::F16, 128, 0), idesc_o = idesc_of(C::F16, HD, 1), hi = desc_hi(1024);
      const uint32_t base = uniform(smem_u32(smem)), tm = uniform(tmem);
      struct Step {
        uint32_t v_lo, v_slot, v_parity, fresh;
        bool valid, last, free_v;
      } st[2];
      st[0].valid = st[1].valid = false;
      uint32_t qcnt[2] = {0, 0}, pcnt[2] = {0, 0}, ocnt[2] = {0, 0}, tile0 = 0;
      bool ok = true;
      auto pv = [&](int s) {  // O += P V of the tile whose S this warpgroup got last
        Step& x = st[s];
        if (!x.fresh) {  // the first of a tile of rows: the accumulator has been read
          if (ocnt[s] > 0) ok = mbar_wait(&B.o_free[s], (ocnt[s] - 1) & 1);
          ++ocnt[s];
        }
        ok = ok && mbar_wait(&B.full[x.v_slot], x.v_parity);
        ok = ok && mbar_wait(&B.p_full[s], pcnt[s]++ & 1);
        ok = __all_sync(0xffffffffu, ok);
        x.valid = false;
        if (!ok) return;
        tc_fence_after();
        const uint32_t o = uniform(tm + C::TMEM_O + s * HD), pa = uniform(tm + C::TMEM_S + s * 128), v_lo = uniform(x.v_lo);
        const uint32_t more = uniform(x.fresh);
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < 8; ++k) mma_ts(o, pa + k * 8, v_lo + k * 128, hi, idesc_o, k > 0 ? 1 : more);
          if (x.free_v) tc_commit(&B.empty[x.v_slot]);
          if (x.last) tc_commit(&B.done[s]);
        }
        __syncwarp();
      };
      for (int i = 0; ok; ++i) {
        ReadItem it;
        ok = next_item(i, it);
        if (!ok || it.len < 0) break;
        const int kb = min(it.kb[0], it.kb[1]), ke = max(it.ke[0], it.ke[1]);
        for (int j = kb; ok && j < ke; ++j) {
          const uint32_t u = 2 * (tile0 + j - kb), ks = u % NU, vs = (u + 1) % NU;
          const uint32_t k_lo = uniform(desc_lo(base + ks * C::UNIT, 16)), v_lo = desc_lo(base + vs * C::UNIT, C::CG);
          const bool in[2] = {j >= it.kb[0] && j < it.ke[0], j >= it.kb[1] && j < it.ke[1]};
          bool got_k = false;
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            if (!in[s]) {
              if (st[s].valid) pv(s);  // its values' place in the ring is needed
              if (!ok) break;
              continue;
            }
            if (st[s].valid) pv(s);
            if (!ok) break;
            const uint32_t slot = s * QB + qcnt[s] % QB, qp = (qcnt[s] / QB) & 1;
            if (j == it.kb[s]) {
              // a new Q tile that is still on its way must not hold up the other warpgroup's last products
              if (s == 0 && st[1].valid && !__all_sync(0xffffffffu, mbar_try_wait(&B.q_full[slot], qp))) pv(1);
              ok = ok && mbar_wait(&B.q_full[slot], qp);
            }
            if (!got_k) ok = ok && mbar_wait(&B.full[ks], (u / NU) & 1);
            got_k = true;
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            const uint32_t q_lo = uniform(desc_lo(base + C::OFF_Q + slot * C::UNIT, 16));
            const uint32_t at = uniform(tm + C::TMEM_S + s * 128);
            const bool last_q = j + 1 == it.ke[s], last_k = s == 1 || !in[1];
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < HD / 16; ++k) {
                const uint32_t off = ((k >> 2) * C::CG + (k & 3) * 32) / 16;
                mma_ss(at, q_lo + off, hi, k_lo + off, hi, idesc_s, k > 0);
              }
              tc_commit(&B.s_full[s]);
              if (last_k) tc_commit(&B.empty[ks]);
              if (last_q) tc_commit(&B.q_empty[slot]);
            }
            __syncwarp();
            st[s] = Step{v_lo, vs, ((u + 1) / NU) & 1, j > it.kb[s] ? 1u : 0u, true, last_q, last_k};
            if (last_q) ++qcnt[s];
          }
        }
        tile0 += ke - kb;
      }
      if (ok && st[0].valid) pv(0);
      if (ok && st[1].valid) pv(1);
      if (!ok) {  // let what was issued finish before tensor memory goes
        if (elect_one()) {
          set_error(p.err, FOLD_DEVERR_TIMEOUT);
          tc_commit(&B.drained);
        }
        __syncwarp();
        warp_wait(&B.drained, 0);
      }
    } else if (warp == NSW + 3) {
      // ------------------------------------------------------------ Q
      uint32_t cnt[2] = {0, 0};
      bool ok = true;
      prefetch_tensormap(&qmap);
      for (int i = 0; ok; ++i) {
        ReadItem it;
        ok = next_item(i, it);
        if (!ok || it.len < 0) break;
        for (int s = 0; s < 2; ++s) {
          if (it.kb[s] >= it.ke[s]) continue;
          const uint32_t slot = s * QB + cnt[s] % QB, use = cnt[s] / QB;
          if (use > 0) ok = warp_wait(&B.q_empty[slot], (use - 1) & 1);
          if (!ok) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(&B.q_full[slot], C::UNIT);
#pragma unroll
            for (int c = 0; c < C::NCG; ++c)
              tma_load_3d_plain(smem + C::OFF_Q + slot * C::UNIT + c * C::CG, &qmap, &B.q_full[slot], c * 64, it.head[s],
                                it.first + it.row0[s]);
          }
          __syncwarp();
          ++cnt[s];
        }
      }
      if (!ok && lane == 0) set_error(p.err, FOLD_DEVERR_TIMEOUT);
      for (int s = 0; s < 2; ++s)  // copies land before exit
        for (uint32_t w = cnt[s] > QB ? cnt[s] - QB : 0; w < cnt[s]; ++w) warp_wait(&B.q_full[s * QB + w % QB], (w / QB) & 1);
    } else {
      // ------------------------------------------------------------ scheduler
      const int units = pair_heads ? p.s.hq / 2 : p.s.hq;
      const int numbers = gridDim.x / units;
      uint32_t asked = 0;
      int out = 0;
      bool ok = true;
      auto publish = [&](const ReadItem& it) {
        if (out >= kItems) ok = warp_wait(&B.item_empty[out % kItems], (out / kItems - 1) & 1);
        if (!ok) return;
        if (lane == 0) {
          B.item[out % kItems] = it;
          mbar_arrive(&B.item_full[out % kItems]);
        }
        __syncwarp();
        ++out;
      };
      for (int id = blockIdx.x; ok && id >= 0;) {
        if (lane == 0) ask_next_block(&B.answer, &B.asked);
        __syncwarp();
        // the last rows see most keys: first; heads of one tile follow one another, their keys stay near
        const int x = numbers - 1 - id / units, unit = id % units;
        Tile t;
        const bool live = pair_heads ? find_tile<128>(p.s, x, t) : find_tile<256>(p.s, x, t);
        if (live) {
          ReadItem it;
          it.first = t.first, it.len = t.len;
          it.hk = (pair_heads ? 2 * unit : unit) / p.s.group;
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            it.row0[s] = t.row0 + (pair_heads ? 0 : s * 128), it.head[s] = pair_heads ? 2 * unit + s : unit;
            int lo = 0, hi = 0;
            if (it.row0[s] < t.len) keys_of(p.s, t.len, it.row0[s], min(it.row0[s] + 128, t.len), lo, hi);
            it.kb[s] = lo / 128, it.ke[s] = (hi + 127) / 128;
            if (it.row0[s] >= t.len) it.kb[s] = it.ke[s] = it.ke[0];  // no rows (only the second may have none)
          }
          publish(it);
        }
        ok = warp_wait(&B.asked, asked++ & 1) && ok;  // (an answer lands before exit, too)
        if (!ok) break;
        id = next_block(&B.answer);
        __syncwarp();
      }
      if (ok) {
        ReadItem it{};
        it.len = -1;
        publish(it);
      }
      if (!ok && lane == 0) set_error(p.err, FOLD_DEVERR_TIMEOUT);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == NSW + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int HD, class T>
int launch_tc(const ReadParams& p, cudaStream_t stream) {
  using C = ReadCfg<HD, T>;
  const char* what = "prompt read";
  CUtensorMap qmap, kmap, vmap;
  if (int s = prompt_map(what, p.q, p.s.hq, p.s.n, p.s.hd, 128, C::F16, &qmap)) return s;
  if (int s = prompt_map(what, p.k, p.s.hkv, p.s.n, p.s.hd, 128, C::F16, &kmap)) return s;
  if (int s = prompt_map(what, p.v, p.s.hkv, p.s.n, p.s.hd, 128, C::F16, &vmap)) return s;
  static std::atomic<uint64_t> configured{0};
  if (int s = allow_smem(prompt_read_tc_kernel<C>, C::SMEM, configured, "cudaFuncSetAttribute(prompt_read)")) return s;
  // the register shares the warps take must add up to what a block is launched with
  static const int regs = [] {
    cudaFuncAttributes a{};
    return cudaFuncGetAttributes(&a, prompt_read_tc_kernel<C>) == cudaSuccess ? a.numRegs : 0;
  }();
  if (regs != kLaunchRegs) return fail(FOLD_ERR_UNSUPPORTED, "prompt read: built with other register shares than launched");
  const int pair = p.s.group % 2 == 0;
  const int64_t blocks = static_cast<int64_t>(tile_numbers(p.s.n, p.s.b, pair ? 128 : 256)) * (pair ? p.s.hq / 2 : p.s.hq);
  if (blocks > 0x7fffffff) return fail(FOLD_ERR_INVALID_ARGUMENT, "prompt read: too many rows");
  return launch_behind(prompt_read_tc_kernel<C>, dim3(static_cast<unsigned>(blocks)), C::NTHREADS, C::SMEM, stream,
                       "prompt_read_tc_kernel", qmap, kmap, vmap, p, pair);
}

template <class T>
int launch_read(const ReadParams& p, cudaStream_t stream) {
  const int hd = p.s.hd;
  if (hd <= 64) return launch_tc<64, T>(p, stream);
  if (hd <= 128) return launch_tc<128, T>(p, stream);
  if (hd <= 192) return launch_mma<192, T>(p, stream);
  return launch_mma<256, T>(p, stream);
}

}  // namespace

int prompt_shape(const char* what, const int* qsl, int b, int n, int hq, int hkv, int hd, int dtype, int causal,
                 int window_left, int window_right, float softmax_scale, prompt::Shape* p) {
  const std::string w(what);
  if (n < 0 || b < 0 || hq < 1 || hkv < 1 || hq % hkv || hq > 65535 || (dtype != FOLD_BF16 && dtype != FOLD_FP16))
    return fail(FOLD_ERR_INVALID_ARGUMENT, w + ": bad sizes or type");
  if (hd < 8 || hd > 256 || hd % 8) return fail(FOLD_ERR_UNSUPPORTED, w + ": the head size is a multiple of 8 up to 256");
  if (n > (1 << 30) || b > (1 << 30)) return fail(FOLD_ERR_INVALID_ARGUMENT, w + ": too many rows or sequences");
  if (!(softmax_scale > 0.f) || softmax_scale > 1e30f)
    return fail(FOLD_ERR_INVALID_ARGUMENT, w + ": softmax_scale must be positive and finite");
  if (n && b && !qsl) return fail(FOLD_ERR_INVALID_ARGUMENT, w + ": null pointer");
  auto bound = [](int x) { return x < 0 || x > prompt::kUnbounded ? prompt::kUnbounded : x; };
  *p = prompt::Shape{};
  p->qsl = qsl, p->b = b, p->n = n, p->hq = hq, p->hkv = hkv, p->group = hq / hkv, p->hd = hd;
  p->left = bound(window_left), p->right = causal ? 0 : bound(window_right);
  p->scale = softmax_scale, p->scale_log2 = softmax_scale * kLog2e;
  return FOLD_OK;
}

int prompt_map(const char* what, const prompt::Rows& x, int heads, int n, int hd, int rows, bool f16, CUtensorMap* out) {
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(hd), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(n)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(x.head) * 2, static_cast<cuuint64_t>(x.tok) * 2};
  const cuuint32_t box[3] = {64, 1, static_cast<cuuint32_t>(rows)};
  return tiled_map(what, x.ptr, 3, dims, strides, box, f16, out);
}

int prompt_rows(const char* what, const char* name, const void* ptr, int64_t tok, int64_t head, int n, int heads,
                int hd, bool written, prompt::Rows* out) {
  const std::string w = std::string(what) + ": " + name;
  if (!ptr) return fail(FOLD_ERR_INVALID_ARGUMENT, w + ": null pointer");
  if (n == 1) tok = static_cast<int64_t>(heads) * hd;  // strides of a single row or head are free
  if (heads == 1) head = hd;
  if (!aligned16(ptr) || tok % 8 || head % 8)
    return fail(FOLD_ERR_ALIGNMENT, w + " must have rows on 16-byte boundaries");
  if (tok < 0 || head < 0 || tok >= (int64_t(1) << 38) || head >= (int64_t(1) << 38))
    return fail(FOLD_ERR_INVALID_ARGUMENT, w + ": strides must not be negative");
  if (written) {
    // heads inside a token's row, or tokens inside a head's
    const bool apart = heads == 1 ? tok >= hd : n == 1 ? head >= hd
                       : (head >= hd && tok >= (heads - 1) * head + hd) || (tok >= hd && head >= (n - 1) * tok + hd);
    if (!apart) return fail(FOLD_ERR_INVALID_ARGUMENT, w + ": the rows must not share memory");
  }
  *out = prompt::Rows{const_cast<void*>(ptr), tok, head};
  return FOLD_OK;
}

namespace {
// na pieces of hd elements at stride sa, and nb at stride sb from `off` on: whether any two share an element.
bool pieces_meet(int64_t off, int na, int64_t sa, int nb, int64_t sb, int hd) {
  using wide = __int128;
  if (off >= static_cast<wide>(na - 1) * sa + hd || -off >= static_cast<wide>(nb - 1) * sb + hd) return false;
  // some k of lo .. hi with |x + k s| < hd
  auto near = [&](int64_t x, int64_t s, int64_t lo, int64_t hi) {
    if (s == 0) return x < hd && -x < hd;
    const int64_t a = -x - hd + 1, k = a > 0 ? (a + s - 1) / s : -(-a / s);  // the least k with x + k s > -hd
    const int64_t first = k > lo ? k : lo;
    return first <= hi && x + static_cast<wide>(first) * s < hd;
  };
  if (na == 1 || sa == sb) return near(off, sb, na == 1 ? 0 : 1 - na, nb - 1);
  if (nb > 65536) return true;  // (heads are fewer; tokens at two strides in one range)
  for (int j = 0; j < nb; ++j)
    if (near(-off - j * sb, sa, 0, na - 1)) return true;
  return false;
}
}  // namespace

bool prompt_overlap(prompt::Rows a, int heads_a, prompt::Rows b, int heads_b, int n, int hd) {
  using wide = __int128;
  const int64_t d = (static_cast<const char*>(b.ptr) - static_cast<const char*>(a.ptr)) / 2;
  if (heads_a == 1) a.head = b.head;  // strides of a single head or row are free
  if (heads_b == 1) b.head = a.head;
  auto span = [&](const prompt::Rows& x, int heads) { return static_cast<wide>(n - 1) * x.tok + static_cast<wide>(heads - 1) * x.head + hd; };
  if (d >= span(a, heads_a) || -d >= span(b, heads_b)) return false;
  if (n == 1) return pieces_meet(d, heads_a, a.head, heads_b, b.head, hd);
  // The outer dimension's pieces lie t apart: b's begin m behind one of a's, and t - m before the next.
  auto outer = [&](int64_t t, int na, int nb, auto inner) {
    int64_t k = d / t, m = d % t;
    if (m < 0) m += t, --k;
    return (k > -nb && k < na && inner(m)) || (k + 1 > -nb && k + 1 < na && inner(m - t));
  };
  auto in_token = [&](const prompt::Rows& x, int heads) { return static_cast<wide>(heads - 1) * x.head + hd <= x.tok; };
  auto in_head = [&](const prompt::Rows& x) { return static_cast<wide>(n - 1) * x.tok + hd <= x.head; };
  if (a.tok == b.tok && in_token(a, heads_a) && in_token(b, heads_b))
    return outer(a.tok, n, n, [&](int64_t off) { return pieces_meet(off, heads_a, a.head, heads_b, b.head, hd); });
  if (a.head == b.head && in_head(a) && in_head(b))
    return outer(a.head, heads_a, heads_b, [&](int64_t off) { return pieces_meet(off, n, a.tok, n, b.tok, hd); });
  return true;
}

}  // namespace fold

extern "C" {

int fold_prompt_read(const void* q, int64_t q_stride_tok, int64_t q_stride_head, const void* k, int64_t k_stride_tok,
                     int64_t k_stride_head, const void* v, int64_t v_stride_tok, int64_t v_stride_head, const int* qsl,
                     int b, int causal, int window_left, int window_right, float softmax_scale, void* out,
                     int64_t o_stride_tok, int64_t o_stride_head, float* lse, int n, int hq, int hkv, int hd, int dtype,
                     int* err, void* stream) {
  using namespace fold;
  const char* what = "prompt read";
  ReadParams p{};
  if (int s = prompt_shape(what, qsl, b, n, hq, hkv, hd, dtype, causal, window_left, window_right, softmax_scale, &p.s))
    return s;
  if (n == 0 || b == 0) return FOLD_OK;
  if (int s = prompt_rows(what, "q", q, q_stride_tok, q_stride_head, n, hq, hd, false, &p.q)) return s;
  if (int s = prompt_rows(what, "k", k, k_stride_tok, k_stride_head, n, hkv, hd, false, &p.k)) return s;
  if (int s = prompt_rows(what, "v", v, v_stride_tok, v_stride_head, n, hkv, hd, false, &p.v)) return s;
  if (int s = prompt_rows(what, "out", out, o_stride_tok, o_stride_head, n, hq, hd, true, &p.out)) return s;
  if (prompt_overlap(p.out, hq, p.k, hkv, n, hd) || prompt_overlap(p.out, hq, p.v, hkv, n, hd))
    return fail(FOLD_ERR_INVALID_ARGUMENT, "prompt read: out must not share memory with k or v");
  const bool over_q = p.out.ptr == p.q.ptr && p.out.tok == p.q.tok && p.out.head == p.q.head;
  if (!over_q && prompt_overlap(p.out, hq, p.q, hq, n, hd))
    return fail(FOLD_ERR_INVALID_ARGUMENT, "prompt read: out must be q or share no memory with it");
  p.lse = lse, p.err = err;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == FOLD_BF16 ? launch_read<__nv_bfloat16>(p, st) : launch_read<__half>(p, st);
}

}  // extern "C"
