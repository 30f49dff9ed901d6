// Gradient of the attention over whole prompts (fold_prompt_read_grad).
//
// Mathematics. With x_rj = scale q_r.k_j, P_rj = e^(x_rj - lse_r), o_r = sum_j P_rj v_j, and the
// gradients do_r of o_r and dlse_r of lse_r:
//   delta_r = do_r.o_r - dlse_r
//   dS_rj   = P_rj (do_r.v_j - delta_r)
//   dq_r    = scale sum_j dS_rj k_j,   dk_j = scale sum_r dS_rj q_r,   dv_j = sum_r P_rj do_r
// the sums over r also over the heads of k_j's group. P and dS are found again from q, k, v and lse, once
// by the rows' tiles (dq) and once by the keys' (dk, dv): seven products where one pass with dq added up
// in memory would take five, but no sum depends on the order in which blocks run, and nothing of the
// size of P is written.
//
// Measured (bf16, head size 128, 32 query and 8 KV heads, one causal sequence; the GPU's time of captured calls, a dozen
// in a row): 8192 tokens 1.62 ms (848 TFLOP/s of five products, 1.19 PFLOP/s of the seven made; 1.8-1.9 ms in a long
// run, where the board is at its 1000 W), 2048 tokens 186 us, 64 tokens 19 us; fp16 1.69 ms, 192 us, 23-29 us. A tile
// of 128 x 128 takes a key's item 3300 cycles and a row's 2700, of which the products are 2050 and 1540: what bounds it
// is the chain dP, dS, acc1, dP of the next, and the energy of the products. At head size 64 (1.36 ms at 8192 tokens)
// the exponentials and dS, 2100 to 2800 cycles a tile.
#include "prompt.cuh"
#include "tcgen05.cuh"

namespace fold {
namespace {
using namespace prompt;

struct GradParams {
  Shape s;
  Rows q, k, v, out, dout, dq, dk, dv;
  const float* lse;   // [hq, n]
  const float* dlse;  // [hq, n] or null
  float2* row;        // workspace [hq, n]: shift - lse log2(e), -delta 2^-shift (see Shift)
  float* norm;        // workspace [hq + hkv, n], fp16: |do_r|^2 of a query head, |v_j|^2 of a KV head
  float2* most;       // workspace [n, hq + hkv], fp16: the largest of them, and of |dlse_r|, in the sequence that starts at
                      // a row (see held_up)
  float* part;        // workspace [splits][dk, dv][n, hkv, hd]: sums over some of a group's heads (splits > 1)
  int splits;
  int zero_rest;      // rows outside the sequences get gradients of zero
  int* err;
};

// Weights are rounded to the inputs' type for the products. In fp16 they are held 2^10 up, so that those of
// rows with many keys keep their bits; dS takes the factor back out.
template <class T>
struct Shift {
  static constexpr bool F16 = std::is_same<T, __half>::value;
  static constexpr float kUp = F16 ? 10.f : 0.f;
  static constexpr float kDown = F16 ? 1.f / 1024.f : 1.f;
};

__device__ __forceinline__ float warp_most(float x) {  // of numbers that are not negative
  return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(x)));
}
__device__ __forceinline__ float2* most_of(const GradParams& p, int first) {
  return p.most + static_cast<int64_t>(first) * (p.s.hq + p.s.hkv);
}

// dS of fp16 is held up too, by a power of two that dq and dk take back out: dS of thousands of keys and a small dout
// lies below the type's normal numbers (2^-14) where dq and dk do not (4096 keys, dout of size 0.001: dq was off by
// 3.5 to 4.5 times its own rounding, now by 1.25). The power follows a bound of dS in a sequence,
//   |dS_rj| <= |do_r.v_j| + |delta_r| <= 2 max|do_r| max|v_j| + max|dlse_r|  (norms; o_r lies between the v_j),
// so that nothing passes the type's range that did not before: 1 where the bound is 2^15 or more or not finite.
// Typical dS of n keys lie some 2^5 n below the bound, which leaves 12 binades for smaller rows at 4096 keys. A NaN
// makes its own results NaN whatever the bound, so it is left out. The norms come from the rows' first kernel, their
// maxima from a launch of their own (5 us for 2048 rows of 32 heads): with the factor in the softmax 2048 rows take
// 192 us where they took 185, 8192 rows in a long run 1.95 ms for 1.91, a batch of short sequences 6 to 10 percent
// more. Maxima by atomics in the first kernel took that from 15 to 33 us.
// Rows' items hold dS up through P, which dq has no other use of; keys' need P for dv as it is.
// Heads [h0, h0 + nh) with KV head hk of the sequence from row `first` on; all lanes of a warp call this.
template <class T>
__device__ __forceinline__ float held_up(const GradParams& p, int first, int h0, int nh, int hk) {
  if constexpr (!Shift<T>::F16) return 1.f;
  const float2* at = most_of(p, first);
  const float v = at[p.s.hq + hk].x;
  float d = 0.f, l = 0.f;
  for (int h = h0 + static_cast<int>(threadIdx.x & 31); h < h0 + nh; h += 32) {
    const float2 b = at[h];
    d = fmaxf(d, b.x), l = fmaxf(l, b.y);
  }
  const float m = fmaf(2.02f * sqrtf(warp_most(d)), sqrtf(v), warp_most(l));
  const int e = min(max(141 - static_cast<int>(__float_as_uint(m) >> 23), 0), 60);  // m 2^e < 2^15
  return __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
}
__device__ __forceinline__ float log2_of_power(float x) {
  return static_cast<float>(static_cast<int>(__float_as_uint(x) >> 23) - 127);
}
// GradParams::most from the rows' norms: a warp a sequence and head (8192 rows: four microseconds).
__global__ void __launch_bounds__(256) prompt_most_kernel(const GradParams p) {
  const int64_t x = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int heads = p.s.hq + p.s.hkv, s = static_cast<int>(x / heads), h = static_cast<int>(x - static_cast<int64_t>(s) * heads);
  const int lane = threadIdx.x & 31;
  wait_for_producer();
  if (s >= p.s.b) return;
  int first, last;
  seq_rows(p.s, s, first, last);
  if (first == last) return;
  auto most = [&](const float* row) {  // of the sequence's sizes (fmaxf leaves NaN out)
    float top = 0.f;
    auto take = [&](float y) { top = fmaxf(top, fabsf(y)); };
    const int lead = min(static_cast<int>(-(reinterpret_cast<uintptr_t>(row) >> 2) & 3), last - first);  // before whole quads
    const int quads = (last - first - lead) / 4, rest = lead + quads * 4;
    if (lane < lead) take(row[lane]);
    if (rest + lane < last - first) take(row[rest + lane]);
#pragma unroll 8
    for (int q = lane; q < quads; q += 32) {
      const float4 y = *reinterpret_cast<const float4*>(row + lead + q * 4);
      take(y.x), take(y.y), take(y.z), take(y.w);
    }
    return warp_most(top);
  };
  const float size = most(p.norm + static_cast<int64_t>(h) * p.s.n + first);
  const float slope = p.dlse && h < p.s.hq ? most(p.dlse + static_cast<int64_t>(h) * p.s.n + first) : 0.f;
  if (lane == 0) most_of(p, first)[h] = make_float2(size, slope);
}

// A row that sees up to this many keys has delta from them, as sum_j P_j (do.v_j) in float32, instead of from the
// rounded out: where few keys share the weight, out's rounding is as large as what dP and delta leave of each other
// (in sequences of a few tokens dq was off by 0.0028 of its norm, 1.65 times what rounding dq alone gives; for 2 to
// 6 tokens it is now that rounding).
constexpr int kExactKeys = 8;

// What the other kernels take of a row and head. A warp has one token and 32 / L of its heads, L lanes of eight
// columns each a head, so that the sequence is looked up once for them. Memory bound (out and dout once).
// (Registers for twelve blocks an SM, whatever the rare rows of few keys would take: with theirs 8192 rows of 32
// heads took 80 us longer.)
template <int L, class T>
__global__ void __launch_bounds__(128, 12) prompt_delta_kernel(const GradParams p) {
  constexpr int HEADS = 32 / L;
  const int lane = threadIdx.x & 31, c = (lane % L) * 8, hd = p.s.hd;
  const int groups = (p.s.hq + HEADS - 1) / HEADS;
  const int64_t x = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int t = static_cast<int>(x / groups), own = static_cast<int>(x - static_cast<int64_t>(t) * groups) * HEADS + lane / L;
  const int h = min(own, p.s.hq - 1);  // (lanes behind the last head repeat it)
  const bool mine = own < p.s.hq && c < hd;
  wait_for_producer();
  if (t >= p.s.n) return;
  if (t < __ldg(p.s.qsl) || t >= __ldg(p.s.qsl + p.s.b)) {
    if (!p.zero_rest || !mine) return;
    const uint4 z = make_uint4(0, 0, 0, 0);
    *reinterpret_cast<uint4*>(static_cast<T*>(p.dq.ptr) + t * p.dq.tok + h * p.dq.head + c) = z;
    if (h < p.s.hkv) {
      *reinterpret_cast<uint4*>(static_cast<T*>(p.dk.ptr) + t * p.dk.tok + h * p.dk.head + c) = z;
      *reinterpret_cast<uint4*>(static_cast<T*>(p.dv.ptr) + t * p.dv.tok + h * p.dv.head + c) = z;
    }
    return;
  }
  auto load = [&](const Rows& r, int64_t row, int64_t head, uint32_t (&w)[4]) {  // eight elements
    const uint4 v = c < hd ? *reinterpret_cast<const uint4*>(static_cast<const T*>(r.ptr) + row * r.tok + head * r.head + c)
                           : make_uint4(0, 0, 0, 0);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  };
  auto dot = [](const uint32_t (&a)[4], const uint32_t (&b)[4]) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 fa = unpack_pair<T>(a[i]), fb = unpack_pair<T>(b[i]);
      sum = fmaf(fa.x, fb.x, fmaf(fa.y, fb.y, sum));
    }
    return sum;
  };
  auto total = [](float v) {  // over a head's lanes
#pragma unroll
    for (int o = L / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  };
  uint32_t wo[4], wd[4];
  load(p.out, t, h, wo), load(p.dout, t, h, wd);
  // (fp16) the values' norms by the warps of as many heads
  const bool values = Shift<T>::F16 && own - lane / L < p.s.hkv;
  uint32_t wn[4];
  if (values) load(p.v, t, min(own, p.s.hkv - 1), wn);
  const int seq = last_sequence(p.s, [&](int, int first) { return first <= t; });
  int first, last, lo, hi;
  seq_rows(p.s, max(seq, 0), first, last);
  keys_of(p.s, last - first, t - first, t - first + 1, lo, hi);
  float sum = total(dot(wo, wd));
  if constexpr (Shift<T>::F16) {
    const float d = total(dot(wd, wd)), v = values ? total(dot(wn, wn)) : 0.f;
    if (lane % L == 0) {
      if (own < p.s.hq) p.norm[static_cast<int64_t>(h) * p.s.n + t] = d;
      if (values && own < p.s.hkv) p.norm[static_cast<int64_t>(p.s.hq + own) * p.s.n + t] = v;
    }
  }
  if (t >= first && t < last && hi - lo <= kExactKeys) {
    float top = -INFINITY, num = 0.f, den = 0.f;
    const int hk = h / p.s.group;
    uint32_t wq[4];
    load(p.q, t, h, wq);
    for (int j0 = lo; j0 < hi; j0 += 4) {  // four at a time: their loads are under way together
      uint32_t wk[4][4], wv[4][4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int64_t j = first + min(j0 + k, hi - 1);
        load(p.k, j, hk, wk[k]), load(p.v, j, hk, wv[k]);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float z = total(dot(wq, wk[k])) * p.s.scale_log2, y = total(dot(wd, wv[k]));
        if (j0 + k < hi) {
          const float up = fmaxf(top, z), f = fast_exp2(top - up), e = fast_exp2(z - up);
          num = fmaf(e, y, num * f), den = den * f + e, top = up;
        }
      }
    }
    if (den > 0.f) sum = num / den;
  }
  if (lane % L == 0 && own < p.s.hq) {
    const int64_t at = static_cast<int64_t>(h) * p.s.n + t;
    const float lse = p.lse[at];
    if (p.dlse) sum -= p.dlse[at];
    // a row without a key (lse -inf) has weights of zero
    p.row[at] = make_float2(lse == -INFINITY ? -INFINITY : Shift<T>::kUp - lse * kLog2e, -sum * Shift<T>::kDown);
  }
}

template <class T>
int launch_delta(const GradParams& p, cudaStream_t stream) {
  const int heads = p.s.hd <= 64 ? 4 : p.s.hd <= 128 ? 2 : 1;
  const int64_t warps = static_cast<int64_t>(p.s.n) * ((p.s.hq + heads - 1) / heads);
  const dim3 grid(static_cast<unsigned>((warps + 3) / 4));
  if (heads == 4) return launch_behind(prompt_delta_kernel<8, T>, grid, 128, 0, stream, "prompt_delta_kernel", p);
  if (heads == 2) return launch_behind(prompt_delta_kernel<16, T>, grid, 128, 0, stream, "prompt_delta_kernel", p);
  return launch_behind(prompt_delta_kernel<32, T>, grid, 128, 0, stream, "prompt_delta_kernel", p);
}

// Whether row r sees one key, which then is its own: the weight is 1 whatever the logit, and dS is the
// gradient of lse alone. (From dP and delta, rounded apart, it would be a remainder where the result is 0.)
__device__ __forceinline__ bool lone(const Shape& s, int len, int r) {
  int lo, hi;
  keys_of(s, len, r, r + 1, lo, hi);
  return hi - lo == 1;
}
template <class T>
__device__ __forceinline__ float lone_ds(const GradParams& p, int h, int at, float weight) {
  return p.dlse ? weight * p.dlse[static_cast<int64_t>(h) * p.s.n + at] * Shift<T>::kDown : 0.f;
}

// Whether dS of the rows [row0, row0 + rows) is held in two parts: where the last one sees up to 512 keys, or 2048
// if the rows before it see as many (behind a window, or without causality: gradients do not fall off there). Such
// rows have the largest gradients, and delta, from the rounded out, is least exact for them. Against 64 bits
// dq of 100 to 300 tokens is off by 1.07 (heads of 128) to 1.17 times (64) the rounding of dq alone, by 1.5 times with
// one part; of 1500 tokens 1.18 to 1.26, of 4096 tokens, most rows of which have one, 1.24 to 1.38. The limits are
// where that ratio was found to pass 1.5 for the last rows; beyond them it does so without causality alone (4096
// tokens 1.46 to 1.58). The second part costs a product and its conversions, a fifth of a tile's time.
__device__ __forceinline__ bool two_parts(const Shape& p, int len, int row0, int rows) {
  const int r = min(row0 + rows, len) - 1;
  int lo, hi;
  keys_of(p, len, r, r + 1, lo, hi);
  const bool grows = p.right == 0 && p.left >= r;
  return hi - lo <= (grows ? 512 : 2048);
}

// Columns that a warp sums gradients of: halves, whose accumulators fit the registers. Two warpgroups find the same
// P and dS and take a half each.
template <int DP>
struct Cols {
  static constexpr int N = DP / 2, PARTS = 2, NT = 256;
};
// The A operand of what rounding `hi` left of the fragment's floats.
template <class T>
__device__ __forceinline__ uint32_t low_pair(uint32_t hi, float a, float b) {
  const float2 f = unpack_pair<T>(hi);
  return pack_pair<T>(a - f.x, b - f.y);
}

// ---------------------------------------------------------------- mma.sync: dk and dv of 64 keys
// Eight warps, 16 keys and half of the columns each; tiles of 64 rows of every head of the group pass by. S^T and dP^T have the
// keys as rows, so that P^T and dS^T are A operands as they leave the registers.
template <int DP, class T>
__device__ __forceinline__ void keys_mma(const GradParams& p, const Tile& t, int hk, unsigned char* smem) {
  using Sm = SmemTile<DP>;
  constexpr int NC = Cols<DP>::N / 16, NT = Cols<DP>::NT;
  const int warp = threadIdx.x >> 5 & 3, part = threadIdx.x >> 7, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const int hd = p.s.hd;
  const uint32_t sk = smem_u32(smem), sv = sk + Sm::BYTES, sq = sv + Sm::BYTES, sd = sq + Sm::BYTES;
  float2* rows = reinterpret_cast<float2*>(smem + 4 * Sm::BYTES);
  int lo, hi;
  rows_of(p.s, t.len, t.row0, min(t.row0 + 64, t.len), lo, hi);
  const int rb = lo / 64, re = (hi + 63) / 64;
  stage_rows<DP, NT>(sk, p.k, t.first, t.len, t.row0, hk, hd);
  stage_rows<DP, NT>(sv, p.v, t.first, t.len, t.row0, hk, hd);
  const float up = held_up<T>(p, t.first, hk * p.s.group, p.s.group, hk), down = Shift<T>::kDown * up;
  float dk[2 * NC][4], dv[2 * NC][4];
#pragma unroll
  for (int i = 0; i < 2 * NC; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) dk[i][e] = dv[i][e] = 0.f;
  const int key0 = t.row0 + warp * 16 + g;
  for (int h = hk * p.s.group; h < (hk + 1) * p.s.group; ++h) {
    for (int j = rb; j < re; ++j) {
      __syncthreads();
      stage_rows<DP, NT>(sq, p.q, t.first, t.len, j * 64, h, hd);
      stage_rows<DP, NT>(sd, p.dout, t.first, t.len, j * 64, h, hd);
      cp_commit();
      if (threadIdx.x < 64) {
        float2 rr = make_float2(-INFINITY, 0.f);
        if (j * 64 + threadIdx.x < t.len) rr = p.row[static_cast<int64_t>(h) * p.s.n + t.first + j * 64 + threadIdx.x];
        rows[threadIdx.x] = make_float2(rr.x, rr.y * up);
      }
      cp_wait<0>();
      __syncthreads();
      float x[8][4], d[8][4];
#pragma unroll
      for (int i = 0; i < 32; ++i) (&x[0][0])[i] = (&d[0][0])[i] = 0.f;
      product_t<DP, T>(x, sk, warp * 16, sq);
      product_t<DP, T>(d, sv, warp * 16, sd);
      const bool two = two_parts(p.s, t.len, j * 64, 64);
      uint32_t pa[4][4], da[4][4], dl[4][4];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float pv[4], sv4[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = i * 8 + 2 * t4 + (e & 1), row = j * 64 + r, key = key0 + (e >> 1) * 8;
          const float2 rr = rows[r];  // (-delta as dS is held)
          const bool in = row < t.len && key >= row - p.s.left && key <= row + p.s.right && key < t.len;
          pv[e] = in ? fast_exp2(fmaf(x[i][e], p.s.scale_log2, rr.x)) : 0.f;
          sv4[e] = in ? pv[e] * fmaf(d[i][e], down, rr.y) : 0.f;
          if (row == key && in && lone(p.s, t.len, row)) sv4[e] = lone_ds<T>(p, h, t.first + row, pv[e]) * up;
        }
        pa[i >> 1][(i & 1) * 2] = pack_pair<T>(pv[0], pv[1]);
        pa[i >> 1][(i & 1) * 2 + 1] = pack_pair<T>(pv[2], pv[3]);
        da[i >> 1][(i & 1) * 2] = pack_pair<T>(sv4[0], sv4[1]);
        da[i >> 1][(i & 1) * 2 + 1] = pack_pair<T>(sv4[2], sv4[3]);
        dl[i >> 1][(i & 1) * 2] = low_pair<T>(da[i >> 1][(i & 1) * 2], sv4[0], sv4[1]);
        dl[i >> 1][(i & 1) * 2 + 1] = low_pair<T>(da[i >> 1][(i & 1) * 2 + 1], sv4[2], sv4[3]);
      }
      product<DP, NC, T>(dv, pa, sd, part * NC);
      product<DP, NC, T>(dk, da, sq, part * NC);
      if (two) product<DP, NC, T>(dk, dl, sq, part * NC);
    }
  }
  const float out_scale = p.s.scale / up;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int key = key0 + e * 8;
    if (key >= t.len) continue;
    T* ok = static_cast<T*>(p.dk.ptr) + (t.first + key) * p.dk.tok + hk * p.dk.head;
    T* ov = static_cast<T*>(p.dv.ptr) + (t.first + key) * p.dv.tok + hk * p.dv.head;
#pragma unroll
    for (int i = 0; i < 2 * NC; ++i) {
      const int c = part * NC * 16 + i * 8;
      if (c >= hd) continue;
      *reinterpret_cast<uint32_t*>(ok + c + 2 * t4) = pack_pair<T>(dk[i][2 * e] * out_scale, dk[i][2 * e + 1] * out_scale);
      *reinterpret_cast<uint32_t*>(ov + c + 2 * t4) =
          pack_pair<T>(dv[i][2 * e] * Shift<T>::kDown, dv[i][2 * e + 1] * Shift<T>::kDown);
    }
  }
}

// ---------------------------------------------------------------- mma.sync: dq of 64 rows of one head
template <int DP, class T>
__device__ __forceinline__ void rows_mma(const GradParams& p, const Tile& t, int h, unsigned char* smem) {
  using Sm = SmemTile<DP>;
  constexpr int NC = Cols<DP>::N / 16, NT = Cols<DP>::NT;
  const int warp = threadIdx.x >> 5 & 3, part = threadIdx.x >> 7, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const int hd = p.s.hd;
  const int hk = h / p.s.group;
  const uint32_t sq = smem_u32(smem), sd = sq + Sm::BYTES, sk = sd + Sm::BYTES, sv = sk + Sm::BYTES;
  int lo, hi;
  keys_of(p.s, t.len, t.row0, min(t.row0 + 64, t.len), lo, hi);
  const int kb = lo / 64, ke = (hi + 63) / 64;
  stage_rows<DP, NT>(sq, p.q, t.first, t.len, t.row0, h, hd);
  stage_rows<DP, NT>(sd, p.dout, t.first, t.len, t.row0, h, hd);
  const float up = held_up<T>(p, t.first, h, 1, hk);
  float dq[2 * NC][4];
#pragma unroll
  for (int i = 0; i < 2 * NC; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) dq[i][e] = 0.f;
  const bool two = two_parts(p.s, t.len, t.row0, 64);
  int klo[2], khi[2];
  float2 rr[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = t.row0 + warp * 16 + e * 8 + g;
    keys_of(p.s, t.len, r, r + 1, klo[e], khi[e]);
    if (r >= t.len) khi[e] = 0;
    rr[e] = r < t.len ? p.row[static_cast<int64_t>(h) * p.s.n + t.first + r] : make_float2(-INFINITY, 0.f);
    rr[e].x += log2_of_power(up);
  }
  for (int j = kb; j < ke; ++j) {
    __syncthreads();
    stage_rows<DP, NT>(sk, p.k, t.first, t.len, j * 64, hk, hd);
    stage_rows<DP, NT>(sv, p.v, t.first, t.len, j * 64, hk, hd);
    cp_commit();
    cp_wait<0>();
    __syncthreads();
    float x[8][4], d[8][4];
#pragma unroll
    for (int i = 0; i < 32; ++i) (&x[0][0])[i] = (&d[0][0])[i] = 0.f;
    product_t<DP, T>(x, sq, warp * 16, sk);
    product_t<DP, T>(d, sd, warp * 16, sv);
    uint32_t da[4][4], dl[4][4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float s4[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = j * 64 + i * 8 + 2 * t4 + (e & 1);
        const bool in = key >= klo[e >> 1] && key < khi[e >> 1];
        const float w = in ? fast_exp2(fmaf(x[i][e], p.s.scale_log2, rr[e >> 1].x)) : 0.f;
        s4[e] = in ? w * fmaf(d[i][e], Shift<T>::kDown, rr[e >> 1].y) : 0.f;
        if (in && khi[e >> 1] - klo[e >> 1] == 1) s4[e] = lone_ds<T>(p, h, t.first + key, w);
      }
      da[i >> 1][(i & 1) * 2] = pack_pair<T>(s4[0], s4[1]);
      da[i >> 1][(i & 1) * 2 + 1] = pack_pair<T>(s4[2], s4[3]);
      dl[i >> 1][(i & 1) * 2] = low_pair<T>(da[i >> 1][(i & 1) * 2], s4[0], s4[1]);
      dl[i >> 1][(i & 1) * 2 + 1] = low_pair<T>(da[i >> 1][(i & 1) * 2 + 1], s4[2], s4[3]);
    }
    product<DP, NC, T>(dq, da, sk, part * NC);
    if (two) product<DP, NC, T>(dq, dl, sk, part * NC);
  }
  const float out_scale = p.s.scale / up;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = t.row0 + warp * 16 + e * 8 + g;
    if (r >= t.len) continue;
    T* o = static_cast<T*>(p.dq.ptr) + (t.first + r) * p.dq.tok + h * p.dq.head;
#pragma unroll
    for (int i = 0; i < 2 * NC; ++i) {
      const int c = part * NC * 16 + i * 8;
      if (c < hd)
        *reinterpret_cast<uint32_t*>(o + c + 2 * t4) = pack_pair<T>(dq[i][2 * e] * out_scale, dq[i][2 * e + 1] * out_scale);
    }
  }
}

// Blocks y < hkv: keys' gradients (more work each, so first); the others: a query head's.
template <int DP, class T>
__global__ void __launch_bounds__(Cols<DP>::NT) prompt_grad_mma_kernel(const GradParams p) {
  extern __shared__ __align__(1024) unsigned char smem[];
  wait_for_producer();
  Tile t;
  const bool keys = static_cast<int>(blockIdx.y) < p.s.hkv;
  // the first keys are seen by most rows, the last rows see most keys
  if (!find_tile<64>(p.s, keys ? blockIdx.x : gridDim.x - 1 - blockIdx.x, t)) return;
  if (keys) keys_mma<DP, T>(p, t, blockIdx.y, smem);
  else rows_mma<DP, T>(p, t, blockIdx.y - p.s.hkv, smem);
}

template <int DP, class T>
int launch_mma(const GradParams& p, cudaStream_t stream) {
  constexpr int smem = 4 * SmemTile<DP>::BYTES + 64 * 8;
  static std::atomic<uint64_t> configured{0};
  if (int s = allow_smem(prompt_grad_mma_kernel<DP, T>, smem, configured, "cudaFuncSetAttribute(prompt_grad)")) return s;
  return launch_behind(prompt_grad_mma_kernel<DP, T>, dim3(tile_numbers(p.s.n, p.s.b, 64), p.s.hkv + p.s.hq),
                       Cols<DP>::NT, smem, stream, "prompt_grad_mma_kernel", p);
}

// ---------------------------------------------------------------- tcgen05, head sizes up to 128
// Heads of other sizes than 64 and 128 are loaded with zeros behind them (outside of the maps).
// A block takes an item: 128 keys of one KV head with the rows of some of its group's heads (dk, dv), or 128
// rows of one head with their keys (dq). Both are the same work: two resident tiles r0, r1 and a stream of
// tiles a, b,
//     S = r0 a^T,  dP = r1 b^T,  dS = P (dP - delta),  acc1 += dS a,  and for keys  acc0 += P b
// with (r0, r1, a, b) = (K, V, Q, dO) or (Q, dO, K, V): lanes of tensor memory are the resident rows. S and
// dP have one place of 128 columns each, X and Y, which change places every tile: once dP is read, S of the
// next tile goes over it, and dP of the next tile goes over what P and dS of this one were written to.
// Order of the products: S of the next tile, acc0 of this one, acc1, dP of the next; dS runs beside S and acc0,
// the exponentials of the next tile beside acc1 and dP.
//
// P of dv is rounded once to the type. dS (in fp16 held up, held_up) of a row that sees few keys is held as two numbers
// of the type, its rounding and what that leaves: such rows have the largest gradients, and delta, from the rounded
// out, is least exact for them (two_parts). Of other rows it is rounded once.
template <int HD_, class T_>
struct GradCfg {
  using T = T_;
  static constexpr int HD = HD_, NTHREADS = 384, NSW = 8;
  static constexpr int NWG = NSW / 4, CW = 128 / NWG;  // softmax warpgroups; columns of a tile that each has
  static constexpr int NCG = HD / 64, CG = 128 * 128, UNIT = NCG * CG;
  static constexpr int NA = HD == 64 ? 4 : 3, NB = HD == 64 ? 4 : 2;  // a is needed longer: by S, then by acc1
  static constexpr int MISC = 1024 + 2048;
  static constexpr int OFF_B = NA * UNIT, OFF_R = OFF_B + NB * UNIT, OFF_BAR = OFF_R + 2 * UNIT, OFF_STAT = OFF_BAR + 1024;
  static constexpr int SMEM = OFF_BAR + MISC;
  static constexpr int TMEM_ACC1 = 256, TMEM_ACC0 = 384;
  static constexpr bool F16 = std::is_same<T, __half>::value;
  static_assert(SMEM <= 232448, "shared memory");
};

// Registers a thread: at launch (the build checks it), then of the softmax warps and of the others.
constexpr int kLaunchRegs = 168, kSoftmaxRegs = 208, kOtherRegs = 88;
static_assert(2 * kSoftmaxRegs + kOtherRegs <= 3 * kLaunchRegs, "a share that is not there is waited for");

struct GradItem {
  int keys;               // 1: gradients of keys, 0: of rows, -1: no more
  int first, len, row0;   // the resident tile's first row in its sequence
  int head, h0, nh;       // resident head; heads of the stream
  int jb, je;             // tiles of the stream, of each head
  int split;
};
constexpr int kItems = 3;

struct GradBars {
  uint64_t a_full[4], b_full[4], r_full[2];
  // S may run a tile ahead of a softmax warp that has not looked yet; dP of a tile also tells the loads that the
  // tile before is through (a commit takes the MMA warp some 200 cycles, so there is one for both)
  uint64_t s_full[2], dp_full[4];
  uint64_t p_full[2], dp_read, acc0_done, ds_full[2], acc_done, drained;
  uint64_t st_full[2], st_empty[2];
  uint64_t item_full[kItems], item_empty[kItems], asked;
  uint4 answer;
  uint32_t tmem;
  GradItem item[kItems];
  // fp16: what dS of an item is held up by. One place more than items are published ahead, so that an item's stays
  // until all warps have taken the next one.
  float up[kItems + 1];
  int gave_up;  // a role's wait ran out
};
static_assert(sizeof(GradBars) <= 1024, "barriers fit their place");

// Columns of tensor memory that hold S (then P and dS) and dP of a tile. Keys' items change the two about, since
// their two accumulators fill the rest; rows' items, with one, have a third place, so that S of the next tile need
// not wait until dP of this one is read. The place of acc0 is only ever the spare one of a key's item.
struct Places {
  uint32_t s, d, spare;
  bool keys;
  __device__ __forceinline__ void start(bool k) { s = 0, d = 128, spare = 384, keys = k; }
  // Moves to the next tile; true: its S lies where dP of this one was.
  __device__ __forceinline__ bool step(bool next_keys) {
    const bool over = next_keys ? spare == 384 : keys;
    const uint32_t x = s;
    if (over) s = d, d = x;
    else s = spare, spare = x;
    keys = next_keys;
    return over;
  }
};

template <class C>
__global__ void __launch_bounds__(C::NTHREADS, 1)
    prompt_grad_tc_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap domap,
                          const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                          const GradParams p, const int key_items) {
  using namespace tc;
  using T = typename C::T;
  constexpr int HD = C::HD, NSW = C::NSW, NA = C::NA, NB = C::NB;
  extern __shared__ __align__(1024) unsigned char smem[];
  GradBars& B = *reinterpret_cast<GradBars*>(smem + C::OFF_BAR);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (warp == NSW) {
    if (lane == 0) {
      for (int i = 0; i < NA; ++i) mbar_init(&B.a_full[i], 1);
      for (int i = 0; i < NB; ++i) mbar_init(&B.b_full[i], 1);
      for (int i = 0; i < 4; ++i) mbar_init(&B.dp_full[i], 1);
      for (int i = 0; i < 2; ++i) {
        mbar_init(&B.r_full[i], 1), mbar_init(&B.s_full[i], 1), mbar_init(&B.ds_full[i], NSW / 2);
        mbar_init(&B.st_full[i], 1), mbar_init(&B.st_empty[i], NSW);
      }
      mbar_init(&B.acc0_done, 1), mbar_init(&B.acc_done, 1);
      mbar_init(&B.p_full[0], NSW), mbar_init(&B.p_full[1], NSW), mbar_init(&B.dp_read, NSW);
      for (int i = 0; i < kItems; ++i) mbar_init(&B.item_full[i], 1), mbar_init(&B.item_empty[i], 3 + NSW);
      mbar_init(&B.asked, 1), mbar_init(&B.drained, 1);
      B.gave_up = 0;
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
  auto give_up = [&] {
    *const_cast<volatile int*>(&B.gave_up) = 1;
    set_error(p.err, FOLD_DEVERR_TIMEOUT);
  };
  // Every role walks the items in the scheduler's order.
  auto next_item = [&](int i, GradItem& it) {
    if (!warp_wait(&B.item_full[i % kItems], (i / kItems) & 1)) return false;
    it = B.item[i % kItems];
    __syncwarp();
    if (lane == 0) mbar_arrive(&B.item_empty[i % kItems]);
    return true;
  };

  if (warp < NSW) {
    regs_up<kSoftmaxRegs>();
    // ------------------------------------------------------------ softmax
    // a warp: 32 lanes (resident rows) and the half of a tile's columns that its warpgroup has. The half's 64
    // columns of S take P and, when that has been read, the low part of dS in the first 32, dS in the others.
    constexpr int CW = C::CW;
    const int wg = warp >> 2, res = (warp & 3) * 32 + lane;
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16), mine = lanes + wg * CW;
    const float* stat = reinterpret_cast<const float*>(smem + C::OFF_STAT);
    uint32_t g = 0, gk = 0, g0 = 0;  // tiles so far; of keys' items; of those in two parts
    Places at{};
    bool ok = true;
    for (int i = 0; ok; ++i) {
      GradItem it;
      ok = next_item(i, it);
      if (!ok || it.keys < 0) break;
      const bool keys = it.keys == 1;
      const int r = min(it.row0 + res, it.len - 1);
      const bool live = it.row0 + res < it.len;
      int lo, hi;
      if (keys) rows_of(p.s, it.len, r, r + 1, lo, hi);
      else keys_of(p.s, it.len, r, r + 1, lo, hi);
      const int warp_lo = __reduce_max_sync(0xffffffffu, lo), warp_hi = __reduce_min_sync(0xffffffffu, hi);
      const bool own = lone(p.s, it.len, r);
      float2 rr = make_float2(0.f, 0.f);
      if (!keys) rr = p.row[static_cast<int64_t>(it.head) * p.s.n + it.first + r];
      // (read from shared memory where it is used: the registers are full)
      auto up = [&] { return C::F16 ? B.up[i % (kItems + 1)] : 1.f; };
      if (C::F16 && !keys) rr.x += log2_of_power(up());
      bool two = !keys && two_parts(p.s, it.len, it.row0, 128);
      for (int h = 0, j = it.jb; h < it.nh; ++g) {
        const int col0 = j * 128;  // stream row of column 0
        if (keys) two = two_parts(p.s, it.len, col0, 128);
        if (g == 0) at.start(keys);
        else at.step(keys);
        const uint32_t x = mine + at.s, y = mine + at.d;
        ok = warp_wait(&B.s_full[g & 1], (g >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        float v[CW];
#pragma unroll
        for (int c = 0; c < CW; c += 32) tmem_ld32(x + c, v + c);
        tmem_wait_ld();
        const float* nl = stat + (gk & 1) * 256 + wg * CW;
        if (keys) {
          ok = warp_wait(&B.st_full[gk & 1], (gk >> 1) & 1);
          if (!ok) break;
#pragma unroll
          for (int c = 0; c < CW; c += 4) {
            const float4 a = *reinterpret_cast<const float4*>(nl + c);
            ffma2(v[c], v[c + 1], p.s.scale_log2, a.x, a.y);
            ffma2(v[c + 2], v[c + 3], p.s.scale_log2, a.z, a.w);
          }
        } else {
#pragma unroll
          for (int c = 0; c < CW; c += 2) ffma2(v[c], v[c + 1], p.s.scale_log2, rr.x, rr.x);
        }
#pragma unroll
        for (int c = 0; c < CW; ++c) v[c] = fast_exp2(v[c]);
        const bool masked = col0 < warp_lo || col0 + 128 > warp_hi;
        const int from = lo - col0 - wg * CW;
        const uint32_t seen = static_cast<uint32_t>(hi - lo);
        if (masked) {
#pragma unroll
          for (int c = 0; c < CW; ++c) v[c] = static_cast<uint32_t>(c - from) < seen ? v[c] : 0.f;
        }
        // rows behind the sequence's end belong to others (NaN included): zeros before the tensor cores read
        // them beside weights of zero
        const int left = it.len - col0;
        if (left < 128) {
          ok = warp_wait(&B.b_full[g % NB], (g / NB) & 1);
          if (!ok) break;
          unsigned char *ta = smem + (g % NA) * C::UNIT, *tb = smem + C::OFF_B + (g % NB) * C::UNIT;
          // (each warpgroup those of its half: acc1 of a half waits for that half's dS alone)
          const int zero0 = max(left, wg * CW), zeros = (wg + 1) * CW - zero0;
          for (int e = tid & 127; e < zeros * C::NCG * 8; e += 128) {
            const int at = zero0 + e / (C::NCG * 8), c = e % (C::NCG * 8);
            const int off = (c >> 3) * C::CG + at * 128 + (c & 7) * 16;
            *reinterpret_cast<uint4*>(ta + off) = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(tb + off) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async();
        }
        if (keys) {
#pragma unroll
          for (int c = 0; c < CW; c += 32) {
            uint32_t w[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) w[k] = pack_pair<T>(v[c + 2 * k], v[c + 2 * k + 1]);
            tmem_st16(x + c / 2, w);
          }
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&B.p_full[gk & 1]);
        }
        const float down = Shift<T>::kDown * (keys ? up() : 1.f);
        ok = warp_wait(&B.dp_full[g & 3], (g >> 2) & 1);
        if (!ok) break;
        tc_fence_after();
        float d[CW];
#pragma unroll
        for (int c = 0; c < CW; c += 32) tmem_ld32(y + c, d + c);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&B.dp_read);
        if (keys) {
#pragma unroll
          for (int c = 0; c < CW; c += 4) {
            const float4 a = *reinterpret_cast<const float4*>(nl + 128 + c);
            ffma2(d[c], d[c + 1], down, a.x, a.y);
            ffma2(d[c + 2], d[c + 3], down, a.z, a.w);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&B.st_empty[gk & 1]);
        } else {
#pragma unroll
          for (int c = 0; c < CW; c += 2) ffma2(d[c], d[c + 1], Shift<T>::kDown, rr.y, rr.y);
        }
        if (masked) {
#pragma unroll
          for (int c = 0; c < CW; ++c) d[c] = static_cast<uint32_t>(c - from) < seen ? d[c] : 0.f;
        }
#pragma unroll
        for (int c = 0; c < CW; c += 2) fmul2(d[c], d[c + 1], v[c], v[c + 1]);
        if (masked && __any_sync(0xffffffffu, own)) {
          const int self = r - col0 - wg * CW, head = keys ? it.h0 + h : it.head;
#pragma unroll
          for (int c = 0; c < CW; ++c)
            if (own && c == self) d[c] = lone_ds<T>(p, head, it.first + r, keys ? v[c] * up() : v[c]);
        }
#pragma unroll
        for (int c = 0; c < CW; c += 32) {
          uint32_t w[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) w[k] = pack_pair<T>(d[c + 2 * k], d[c + 2 * k + 1]);
          tmem_st16(x + CW / 2 + c / 2, w);
          if (two) {
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const float2 f = unpack_pair<T>(w[k]);
              fsub2(d[c + 2 * k], d[c + 2 * k + 1], f.x, f.y);
            }
          }
        }
        if (two) {
          if (keys) {  // P has been read
            ok = warp_wait(&B.acc0_done, g0++ & 1);
            if (!ok) break;
            tc_fence_after();
          }
#pragma unroll
          for (int c = 0; c < CW; c += 32) {
            uint32_t w[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) w[k] = pack_pair<T>(d[c + 2 * k], d[c + 2 * k + 1]);
            tmem_st16(x + c / 2, w);
          }
        }
        if (keys) ++gk;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&B.ds_full[wg * CW / 64]);
        if (++j == it.je) j = it.jb, ++h;
      }
      if (!ok) break;
      ok = warp_wait(&B.acc_done, i & 1);
      if (!ok) break;
      tc_fence_after();
      // keys: half of the warpgroups for dv, half for dk; rows: dq's columns shared out
      const bool dv = keys && wg < C::NWG / 2;
      const int cols = keys ? HD * 2 / C::NWG : HD / C::NWG, c0 = (keys ? wg % (C::NWG / 2) : wg) * cols;
      const uint32_t acc = lanes + (dv ? C::TMEM_ACC0 : C::TMEM_ACC1) + c0;
      const float f = dv ? Shift<T>::kDown : p.s.scale / up();
      const Rows& to = dv ? p.dv : keys ? p.dk : p.dq;
      const int64_t row = it.first + r;
      T* out = static_cast<T*>(to.ptr) + row * to.tok + it.head * to.head + c0;
      float* part = p.part + ((static_cast<int64_t>(2 * it.split + dv) * p.s.n + row) * p.s.hkv + it.head) * p.s.hd + c0;
      const bool partial = keys && p.splits > 1, wide = rows_on_32(to);
#pragma unroll 1
      for (int c = 0; c < cols; c += 16) {
        float o[16];
        __syncwarp();
        tmem_ld16(acc + c, o);
        if (!live) continue;
        if (partial) {
#pragma unroll
          for (int k = 0; k < 16; k += 4)
            if (c0 + c + k < p.s.hd)
              *reinterpret_cast<float4*>(part + c + k) = make_float4(o[k] * f, o[k + 1] * f, o[k + 2] * f, o[k + 3] * f);
        } else {
          uint32_t w[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) w[k] = pack_pair<T>(o[2 * k] * f, o[2 * k + 1] * f);
          store_row16(out + c, w, wide, p.s.hd - c0 - c);
        }
      }
      __syncwarp();
      tc_fence_before();  // the next item's acc0 comes behind its first tile's P, acc1 behind all reads of its dP
    }
    if (!ok && lane == 0) give_up();
  } else {
    regs_down<kOtherRegs>();
    if (warp == NSW) {
      // ------------------------------------------------------------ loads
      uint32_t g = 0, a_sent = 0, b_sent = 0, r0_sent = 0, r1_sent = 0;  // tiles so far; copies of each kind
      bool ok = true;
      if (lane == 0) prefetch_tensormap(&qmap), prefetch_tensormap(&domap), prefetch_tensormap(&kmap), prefetch_tensormap(&vmap);
      // dP of tile n, and with it all products of the tiles before
      auto through = [&](uint32_t n) { return warp_wait(&B.dp_full[n & 3], (n >> 2) & 1); };
      auto load = [&](const CUtensorMap* map, int offset, uint64_t* full, int head, int row) {
        if (lane == 0) {
          mbar_arrive_expect_tx(full, C::UNIT);
#pragma unroll
          for (int c = 0; c < C::NCG; ++c) tma_load_3d_plain(smem + offset + c * C::CG, map, full, c * 64, head, row);
        }
        __syncwarp();
      };
      for (int i = 0; ok; ++i) {
        GradItem it;
        ok = next_item(i, it);
        if (!ok || it.keys < 0) break;
        const bool keys = it.keys == 1;
        for (int h = 0, j = it.jb; ok && h < it.nh; ++g) {
          const int row = it.first + j * 128, head = it.h0 + h;
          const bool first = h == 0 && j == it.jb;
          if (++j == it.je) j = it.jb, ++h;
          if (first) {
            if (i > 0) ok = through(g - 1);
            if (!ok) break;
            load(keys ? &kmap : &qmap, C::OFF_R, &B.r_full[0], it.head, it.first + it.row0);
            ++r0_sent;
          }
          if (g >= NA) ok = through(g - NA + 1);
          if (!ok) break;
          load(keys ? &qmap : &kmap, (g % NA) * C::UNIT, &B.a_full[g % NA], head, row);
          ++a_sent;
          if (first) {
            load(keys ? &vmap : &domap, C::OFF_R + C::UNIT, &B.r_full[1], it.head, it.first + it.row0);
            ++r1_sent;
          }
          if (g >= NB) ok = through(g - NB + 1);
          if (!ok) break;
          load(keys ? &domap : &vmap, C::OFF_B + (g % NB) * C::UNIT, &B.b_full[g % NB], head, row);
          ++b_sent;
        }
      }
      if (!ok && lane == 0) give_up();
      // copies land before exit, those of a tile that another wait gave up on too
      for (uint32_t w = a_sent > NA ? a_sent - NA : 0; w < a_sent; ++w) warp_wait(&B.a_full[w % NA], (w / NA) & 1);
      for (uint32_t w = b_sent > NB ? b_sent - NB : 0; w < b_sent; ++w) warp_wait(&B.b_full[w % NB], (w / NB) & 1);
      if (r0_sent > 0) warp_wait(&B.r_full[0], (r0_sent - 1) & 1);
      if (r1_sent > 0) warp_wait(&B.r_full[1], (r1_sent - 1) & 1);
    } else if (warp == NSW + 1) {
      // ------------------------------------------------------------ MMAs
      constexpr uint32_t idesc_s = idesc_of(C::F16, 128, 0), idesc_o = idesc_of(C::F16, HD, 1), hi = desc_hi(1024);
      const uint32_t base = uniform(smem_u32(smem)), tm = uniform(tmem);
      GradItem it;
      int items = 0, j = 0, heads = 0;  // items so far; the next tile's place in the current one, heads left
      uint32_t n = 0;                   // tiles so far
      bool ok = true;
      struct Step {
        bool valid, keys, first, last, two;
        uint32_t item;              // parity
        uint32_t s, d, aslot, bslot;
        bool early;                 // S may come before dP of the tile before has been read
      } now{}, next{};
      Places at{};
      bool was_keys[2] = {false, false};  // of the two tiles before
      uint32_t aslot = 0, bslot = 0;
      auto advance = [&](Step& x) {  // the tile behind the last one
        if (heads == 0) {
          x.valid = false;
          ok = next_item(items, it);
          if (!ok || it.keys < 0) return;
          ++items, j = it.jb, heads = it.nh;
        }
        x.valid = true, x.keys = it.keys == 1, x.item = (items - 1) & 1;
        x.first = heads == it.nh && j == it.jb;
        x.two = two_parts(p.s, it.len, x.keys ? j * 128 : it.row0, 128);
        if (++j == it.je) j = it.jb, --heads;
        x.last = heads == 0;
        bool over = false;
        if (n == 0) at.start(x.keys);
        else over = at.step(x.keys);
        // (the spare place of the first rows behind a key's item may still be read as its acc0)
        x.early = !over && !was_keys[1];
        was_keys[1] = was_keys[0], was_keys[0] = x.keys;
        x.s = at.s, x.d = at.d, x.aslot = aslot, x.bslot = bslot;
        if (++aslot == NA) aslot = 0;
        if (++bslot == NB) bslot = 0;
        ++n;
      };
      constexpr uint32_t kmajor = 1u << 16, mnmajor = static_cast<uint32_t>(C::CG >> 4) << 16;  // leading offsets
      const uint32_t r0 = uniform(desc_lo(base + C::OFF_R, 16)), r1 = uniform(desc_lo(base + C::OFF_R + C::UNIT, 16));
      uint32_t aphase = 0, bphase = 0;  // parities of the rings, a bit a slot
      auto landed = [&](const Step& x, int w) {  // the operands of S (w 0) or dP (1)
        const uint32_t slot = w == 0 ? x.aslot : x.bslot;
        uint32_t& phase = w == 0 ? aphase : bphase;
        if (x.first) ok = ok && mbar_wait(&B.r_full[w], x.item);
        ok = ok && mbar_wait(w == 0 ? &B.a_full[slot] : &B.b_full[slot], phase >> slot & 1);
        phase ^= 1u << slot;
        ok = __all_sync(0xffffffffu, ok);
      };
      auto a_at = [&](const Step& x) { return (base + x.aslot * C::UNIT) >> 4; };
      auto b_at = [&](const Step& x) { return (base + C::OFF_B + x.bslot * C::UNIT) >> 4; };
      auto product = [&](uint32_t to, uint32_t r, uint32_t x) {  // by one lane
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          const uint32_t off = ((k >> 2) * C::CG + (k & 3) * 32) / 16;
          mma_ss(to, r + off, hi, x + kmajor + off, hi, idesc_s, k > 0);
        }
      };
      uint32_t gk = 0, g = 0;
      advance(now);
      if (ok && now.valid) {
        const uint32_t s_at = uniform(tm + now.s), d_at = uniform(tm + now.d), xa = uniform(a_at(now)), xb = uniform(b_at(now));
        landed(now, 0);
        tc_fence_after();
        if (ok && elect_one()) {
          product(s_at, r0, xa);
          tc_commit(&B.s_full[0]);
        }
        __syncwarp();
        if (ok) landed(now, 1);
        tc_fence_after();
        if (ok && elect_one()) {
          product(d_at, r1, xb);
          tc_commit(&B.dp_full[0]);
        }
        __syncwarp();
      }
      while (ok && now.valid) {
        // The issue of MMAs lasts about as long as they run, so all else comes where it hides behind the last
        // ones issued, dP's.
        const uint32_t more = uniform(now.first ? 0u : 1u), x = uniform(tm + now.s);
        const uint32_t am = uniform(a_at(now) + mnmajor), bm = uniform(b_at(now) + mnmajor);
        advance(next);
        const uint32_t s_at = uniform(tm + next.s), d_at = uniform(tm + next.d);
        const uint32_t xa = uniform(a_at(next)), xb = uniform(b_at(next));
        if (!ok) break;
        if (next.valid) {
          // S of the next tile first: the softmax warps come to it when they are through with dS
          landed(next, 0);
          if (ok && !next.early) ok = warp_wait(&B.dp_read, g & 1);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            product(s_at, r0, xa);
            tc_commit(&B.s_full[(g + 1) & 1]);
          }
          __syncwarp();
        }
        if (now.keys) {
          ok = warp_wait(&B.p_full[gk & 1], gk >> 1 & 1);
          ++gk;
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
              mma_ts(tm + C::TMEM_ACC0, x + (k * 16 / C::CW) * C::CW + k * 16 % C::CW / 2, bm + k * 128, hi, idesc_o, k > 0 ? 1 : more);
            if (now.two) tc_commit(&B.acc0_done);
          }
          __syncwarp();
        }
        if (next.valid) landed(next, 1);
        // An item's first product overwrites acc1, which either warpgroup may still be reading for the item before:
        // once all have read dP they are through with it (dS of one half tells of one warpgroup only).
        if (now.first) ok = ok && warp_wait(&B.dp_read, g & 1);
#pragma unroll
        for (int half = 0; ok && half < 2; ++half) {
          ok = warp_wait(&B.ds_full[half], g & 1);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int k = half * 4; k < half * 4 + 4; ++k)
              mma_ts(tm + C::TMEM_ACC1, x + (k * 16 / C::CW) * C::CW + k * 16 % C::CW / 2 + C::CW / 2, am + k * 128, hi, idesc_o, k > 0 ? 1 : more);
            if (now.two) {  // what the roundings left
#pragma unroll
              for (int k = half * 4; k < half * 4 + 4; ++k)
                mma_ts(tm + C::TMEM_ACC1, x + (k * 16 / C::CW) * C::CW + k * 16 % C::CW / 2, am + k * 128, hi, idesc_o, 1);
            }
            if (half == 1) {
              if (now.last) tc_commit(&B.acc_done);
              if (next.valid) {
                product(d_at, r1, xb);
                tc_commit(&B.dp_full[(g + 1) & 3]);
              }
            }
          }
          __syncwarp();
        }
        if (!ok) break;
        now = next, ++g;
      }
      if (!ok) {  // let what was issued finish before tensor memory goes
        if (elect_one()) {
          give_up();
          tc_commit(&B.drained);
        }
        __syncwarp();
        warp_wait(&B.drained, 0);
      }
    } else if (warp == NSW + 3) {
      // ------------------------------------------------------------ lse and delta of streamed rows
      float* stat = reinterpret_cast<float*>(smem + C::OFF_STAT);
      uint32_t gk = 0;
      bool ok = true;
      for (int i = 0; ok; ++i) {
        GradItem it;
        ok = next_item(i, it);
        if (!ok || it.keys < 0) break;
        if (it.keys == 0) continue;
        const float up = C::F16 ? B.up[i % (kItems + 1)] : 1.f;
        for (int h = 0, j = it.jb; h < it.nh; ++gk) {
          const int r0 = j * 128;
          const float2* src = p.row + static_cast<int64_t>(it.h0 + h) * p.s.n + it.first + r0;
          if (++j == it.je) j = it.jb, ++h;
          float2 v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            v[k] = r0 + k * 32 + lane < it.len ? src[k * 32 + lane] : make_float2(-INFINITY, 0.f);
          if (gk >= 2) ok = warp_wait(&B.st_empty[gk & 1], (gk / 2 - 1) & 1);
          if (!ok) break;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            stat[(gk & 1) * 256 + k * 32 + lane] = v[k].x, stat[(gk & 1) * 256 + 128 + k * 32 + lane] = v[k].y * up;
          __syncwarp();
          if (lane == 0) mbar_arrive(&B.st_full[gk & 1]);
        }
      }
      if (!ok && lane == 0) give_up();
    } else {
      // ------------------------------------------------------------ scheduler
      const int key_heads = p.s.hkv * p.splits, numbers = key_items / key_heads;
      uint32_t asked = 0;
      int out = 0;
      bool ok = true;
      auto publish = [&](const GradItem& it, float up) {
        // An item lasts for seconds where many heads share a KV head and a million rows (128 heads: 1.8 s), so this
        // wait goes on while no other role has given up.
        if (out >= kItems)
          for (int tries = 0; !(ok = warp_wait(&B.item_empty[out % kItems], (out / kItems - 1) & 1)) && tries < 64; ++tries)
            if (__any_sync(0xffffffffu, *const_cast<const volatile int*>(&B.gave_up))) break;
        if (!ok) return;
        if (lane == 0) {
          B.item[out % kItems] = it;
          if (C::F16) B.up[out % (kItems + 1)] = up;
          mbar_arrive(&B.item_full[out % kItems]);
        }
        __syncwarp();
        ++out;
      };
      for (int id = blockIdx.x; ok && id >= 0;) {
        if (lane == 0) ask_next_block(&B.answer, &B.asked);
        __syncwarp();
        // the longest first: the first keys are seen by most rows, the last rows see most keys
        const bool keys = id < key_items;
        const int k = keys ? id : id - key_items, heads = keys ? key_heads : p.s.hq;
        const int x = keys ? k / heads : numbers - 1 - k / heads, h = k % heads;
        Tile t;
        if (find_tile<128>(p.s, x, t)) {
          GradItem it;
          int lo, hi;
          it.keys = keys, it.first = t.first, it.len = t.len, it.row0 = t.row0;
          if (keys) {
            it.head = h / p.splits, it.split = h % p.splits;
            it.nh = p.s.group / p.splits, it.h0 = it.head * p.s.group + it.split * it.nh;
            rows_of(p.s, t.len, t.row0, min(t.row0 + 128, t.len), lo, hi);
          } else {
            it.head = h, it.split = 0, it.h0 = h / p.s.group, it.nh = 1;
            keys_of(p.s, t.len, t.row0, min(t.row0 + 128, t.len), lo, hi);
          }
          it.jb = lo / 128, it.je = (hi + 127) / 128;
          publish(it, held_up<T>(p, t.first, keys ? it.h0 : h, it.nh, keys ? it.head : it.h0));
        }
        ok = warp_wait(&B.asked, asked++ & 1) && ok;  // (an answer lands before exit, too)
        if (!ok) break;
        id = next_block(&B.answer);
        __syncwarp();
      }
      if (ok) {
        GradItem it{};
        it.keys = -1;
        publish(it, 1.f);
      }
      if (!ok && lane == 0) give_up();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == NSW + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// dk and dv from the sums over some heads each, added in their order. Memory bound.
template <class T>
__global__ void __launch_bounds__(256) prompt_grad_join_kernel(const GradParams p) {
  const int64_t x = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;  // four elements of dk and of dv
  const int per = p.s.hd / 4, c = static_cast<int>(x % per) * 4;
  const int64_t row = x / per, t = row / p.s.hkv;
  wait_for_producer();
  if (t >= p.s.n || t < __ldg(p.s.qsl) || t >= __ldg(p.s.qsl + p.s.b)) return;
  const int h = static_cast<int>(row - t * p.s.hkv);
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < p.splits; ++s) {
      const float4 a = *reinterpret_cast<const float4*>(p.part + (static_cast<int64_t>(2 * s + w) * p.s.n * p.s.hkv + row) * p.s.hd + c);
      sum.x += a.x, sum.y += a.y, sum.z += a.z, sum.w += a.w;
    }
    const Rows& to = w == 0 ? p.dk : p.dv;
    *reinterpret_cast<uint2*>(static_cast<T*>(to.ptr) + t * to.tok + h * to.head + c) =
        make_uint2(pack_pair<T>(sum.x, sum.y), pack_pair<T>(sum.z, sum.w));
  }
}

// Into how many the heads of a group are split for the gradients of keys: enough that the device's blocks have
// three items each, or every head by itself.
int key_splits(int n, int hkv, int group) {
  const int want = 3 * 148;
  const int64_t items = (static_cast<int64_t>(n) + 127) / 128 * hkv;
  for (int s = 1; s < group; ++s)
    if (group % s == 0 && items * s >= want) return s;
  return group;
}
// Bytes of the partial sums of a call, and of the largest call of up to n rows.
int64_t part_bytes(int64_t n, int splits, int hkv, int hd) { return splits > 1 ? splits * 2 * n * hkv * hd * 4 : 0; }
int64_t most_part_bytes(int n, int hkv, int group, int hd) {
  int64_t most = 0;
  for (int s = 2, below = 1; s <= group; ++s) {
    if (group % s) continue;
    // the next smaller split is not enough for this many tiles of 128 rows
    const int64_t rows = ((3 * 148 + hkv * below - 1) / (hkv * below) - 1) * int64_t(128);
    const int64_t x = part_bytes(rows < n ? rows : n, s, hkv, hd);
    most = x > most ? x : most, below = s;
  }
  return most;
}
// Bytes of the workspace's other parts: GradParams::row, and most and norm (fp16).
int64_t row_bytes(int64_t n, int hq) { return (n * hq * 8 + 15) / 16 * 16; }
int64_t most_bytes(int64_t n, int hq, int hkv) { return (n * (hq + hkv) * 12 + 15) / 16 * 16; }
bool tensor_memory_size(int hd) { return hd <= 128; }
// The kernel of the other head sizes has a head of keys or queries in each of the grid's y blocks.
bool heads_fit(int hq, int hkv, int hd) { return tensor_memory_size(hd) || hq + hkv <= 65535; }

template <int HD, class T>
int launch_tc(const GradParams& p, cudaStream_t stream) {
  using C = GradCfg<HD, T>;
  const char* what = "prompt read grad";
  CUtensorMap qmap, domap, kmap, vmap;
  if (int s = prompt_map(what, p.q, p.s.hq, p.s.n, p.s.hd, 128, C::F16, &qmap)) return s;
  if (int s = prompt_map(what, p.dout, p.s.hq, p.s.n, p.s.hd, 128, C::F16, &domap)) return s;
  if (int s = prompt_map(what, p.k, p.s.hkv, p.s.n, p.s.hd, 128, C::F16, &kmap)) return s;
  if (int s = prompt_map(what, p.v, p.s.hkv, p.s.n, p.s.hd, 128, C::F16, &vmap)) return s;
  static std::atomic<uint64_t> configured{0};
  if (int s = allow_smem(prompt_grad_tc_kernel<C>, C::SMEM, configured, "cudaFuncSetAttribute(prompt_grad)")) return s;
  // the register shares the warps take must add up to what a block is launched with
  static const int regs = [] {
    cudaFuncAttributes a{};
    return cudaFuncGetAttributes(&a, prompt_grad_tc_kernel<C>) == cudaSuccess ? a.numRegs : 0;
  }();
  if (regs != kLaunchRegs) return fail(FOLD_ERR_UNSUPPORTED, "prompt read grad: built with other register shares than launched");
  const int64_t numbers = tile_numbers(p.s.n, p.s.b, 128), key_items = numbers * p.s.hkv * p.splits;
  const int64_t blocks = key_items + numbers * p.s.hq;
  if (blocks > 0x7fffffff) return fail(FOLD_ERR_INVALID_ARGUMENT, "prompt read grad: too many rows");
  if (int s = launch_behind(prompt_grad_tc_kernel<C>, dim3(static_cast<unsigned>(blocks)), C::NTHREADS, C::SMEM, stream,
                            "prompt_grad_tc_kernel", qmap, domap, kmap, vmap, p, static_cast<int>(key_items)))
    return s;
  if (p.splits == 1) return FOLD_OK;
  const int64_t quads = static_cast<int64_t>(p.s.n) * p.s.hkv * (p.s.hd / 4);
  if (quads > (int64_t(0x7fffffff) << 8)) return fail(FOLD_ERR_INVALID_ARGUMENT, "prompt read grad: too many rows");
  return launch_behind(prompt_grad_join_kernel<T>, dim3(static_cast<unsigned>((quads + 255) / 256)), 256, 0, stream,
                       "prompt_grad_join_kernel", p);
}

template <class T>
int launch_grad(const GradParams& p, cudaStream_t stream) {
  if (int s = launch_delta<T>(p, stream)) return s;
  if constexpr (Shift<T>::F16) {
    const int64_t warps = static_cast<int64_t>(p.s.b) * (p.s.hq + p.s.hkv);
    if (warps / 8 >= 0x7fffffff) return fail(FOLD_ERR_INVALID_ARGUMENT, "prompt read grad: too many sequences");
    if (int s = launch_behind(prompt_most_kernel, dim3(static_cast<unsigned>((warps + 7) / 8)), 256, 0, stream, "prompt_most_kernel", p)) return s;
  }
  const int hd = p.s.hd;
  if (hd <= 64) return launch_tc<64, T>(p, stream);
  if (hd <= 128) return launch_tc<128, T>(p, stream);
  if (hd <= 192) return launch_mma<192, T>(p, stream);
  return launch_mma<256, T>(p, stream);
}

}  // namespace
}  // namespace fold

extern "C" {

int64_t fold_prompt_read_grad_workspace(int n, int hq, int hkv, int hd) {
  if (n < 0 || hq < 1 || hkv < 1 || hq % hkv || hq > 65535 || hd < 8 || hd > 256 || hd % 8 || !fold::heads_fit(hq, hkv, hd)) return -1;
  return fold::row_bytes(n, hq) + fold::most_bytes(n, hq, hkv) + 16 + (fold::tensor_memory_size(hd) ? fold::most_part_bytes(n, hkv, hq / hkv, hd) : 0);
}

int fold_prompt_read_grad(const void* dout, int64_t do_stride_tok, int64_t do_stride_head, const void* q,
                          int64_t q_stride_tok, int64_t q_stride_head, const void* k, int64_t k_stride_tok,
                          int64_t k_stride_head, const void* v, int64_t v_stride_tok, int64_t v_stride_head,
                          const void* out, int64_t o_stride_tok, int64_t o_stride_head, const float* lse,
                          const float* dlse, const int* qsl, int b, int causal, int window_left, int window_right,
                          float softmax_scale, void* dq, int64_t dq_stride_tok, int64_t dq_stride_head, void* dk,
                          int64_t dk_stride_tok, int64_t dk_stride_head, void* dv, int64_t dv_stride_tok,
                          int64_t dv_stride_head, int zero_rest, void* workspace, int64_t workspace_bytes, int n,
                          int hq, int hkv, int hd, int dtype, int* err, void* stream) {
  using namespace fold;
  const char* what = "prompt read grad";
  GradParams p{};
  if (int s = prompt_shape(what, qsl, b, n, hq, hkv, hd, dtype, causal, window_left, window_right, softmax_scale, &p.s))
    return s;
  if (!heads_fit(hq, hkv, hd)) return fail(FOLD_ERR_UNSUPPORTED, "prompt read grad: too many heads for this head size");
  if (n == 0) return FOLD_OK;
  if (b == 0 && !zero_rest) return FOLD_OK;
  if (b == 0) return fail(FOLD_ERR_INVALID_ARGUMENT, "prompt read grad: no sequences");
  struct { const char* name; const void* ptr; int64_t tok, head; int heads; bool written; Rows* to; } const rows[] = {
      {"dout", dout, do_stride_tok, do_stride_head, hq, false, &p.dout}, {"q", q, q_stride_tok, q_stride_head, hq, false, &p.q},
      {"k", k, k_stride_tok, k_stride_head, hkv, false, &p.k}, {"v", v, v_stride_tok, v_stride_head, hkv, false, &p.v},
      {"out", out, o_stride_tok, o_stride_head, hq, false, &p.out}, {"dq", dq, dq_stride_tok, dq_stride_head, hq, true, &p.dq},
      {"dk", dk, dk_stride_tok, dk_stride_head, hkv, true, &p.dk}, {"dv", dv, dv_stride_tok, dv_stride_head, hkv, true, &p.dv}};
  for (const auto& r : rows)
    if (int s = prompt_rows(what, r.name, r.ptr, r.tok, r.head, n, r.heads, hd, r.written, r.to)) return s;
  for (int i = 5; i < 8; ++i)
    for (int k = 0; k < i; ++k)
      if (prompt_overlap(*rows[i].to, rows[i].heads, *rows[k].to, rows[k].heads, n, hd))
        return fail(FOLD_ERR_INVALID_ARGUMENT,
                    std::string("prompt read grad: ") + rows[i].name + " must not share memory with " + rows[k].name);
  if (!lse) return fail(FOLD_ERR_INVALID_ARGUMENT, "prompt read grad: null pointer");
  if (static_cast<int64_t>(n) * hq > (int64_t(1) << 32)) return fail(FOLD_ERR_INVALID_ARGUMENT, "prompt read grad: too many rows");
  p.splits = tensor_memory_size(hd) ? key_splits(n, hkv, p.s.group) : 1;
  const int64_t part_at = row_bytes(n, hq) + (dtype == FOLD_FP16 ? most_bytes(n, hq, hkv) : 0);
  if (!workspace || workspace_bytes < part_at + part_bytes(n, p.splits, hkv, hd))
    return fail(FOLD_ERR_INVALID_ARGUMENT, "prompt read grad: the workspace holds fold_prompt_read_grad_workspace bytes");
  if (!aligned16(workspace)) return fail(FOLD_ERR_ALIGNMENT, "prompt read grad: the workspace must be 16-byte aligned");
  p.lse = lse, p.dlse = dlse, p.row = static_cast<float2*>(workspace), p.zero_rest = zero_rest, p.err = err;
  p.most = reinterpret_cast<float2*>(static_cast<char*>(workspace) + row_bytes(n, hq));
  p.norm = reinterpret_cast<float*>(p.most + static_cast<int64_t>(n) * (hq + hkv));
  p.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + part_at);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == FOLD_BF16 ? launch_grad<__nv_bfloat16>(p, st) : launch_grad<__half>(p, st);
}

}  // extern "C"
