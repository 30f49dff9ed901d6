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
#include "prompt.cuh"

namespace fold {
namespace {
using namespace prompt;

struct GradParams {
  Shape s;
  Rows q, k, v, out, dout, dq, dk, dv;
  const float* lse;   // [hq, n]
  const float* dlse;  // [hq, n] or null
  float2* row;        // workspace [hq, n]: lse log2(e) - shift, delta 2^-shift (see Shift)
  int zero_rest;      // rows outside the sequences get gradients of zero
  int* err;
};

// Weights are rounded to the inputs' type for the products. In fp16 they are held 2^10 up, so that those of
// rows with many keys keep their bits; dS takes the factor back out.
template <class T>
struct Shift {
  static constexpr float kUp = std::is_same<T, __nv_bfloat16>::value ? 0.f : 10.f;
  static constexpr float kDown = std::is_same<T, __nv_bfloat16>::value ? 1.f : 1.f / 1024.f;
};

// A warp a row and head: what the other kernels take of it. Memory bound (out and dout once).
template <class T>
__global__ void __launch_bounds__(128) prompt_delta_kernel(const GradParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t x = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int t = static_cast<int>(x / p.s.hq), h = static_cast<int>(x - static_cast<int64_t>(t) * p.s.hq);
  wait_for_producer();
  if (t >= p.s.n) return;
  const int hd = p.s.hd;
  if (t < __ldg(p.s.qsl) || t >= __ldg(p.s.qsl + p.s.b)) {
    if (!p.zero_rest) return;
    for (int c = lane * 8; c < hd; c += 256) {
      const uint4 z = make_uint4(0, 0, 0, 0);
      *reinterpret_cast<uint4*>(static_cast<T*>(p.dq.ptr) + t * p.dq.tok + h * p.dq.head + c) = z;
      if (h < p.s.hkv) {
        *reinterpret_cast<uint4*>(static_cast<T*>(p.dk.ptr) + t * p.dk.tok + h * p.dk.head + c) = z;
        *reinterpret_cast<uint4*>(static_cast<T*>(p.dv.ptr) + t * p.dv.tok + h * p.dv.head + c) = z;
      }
    }
    return;
  }
  float sum = 0.f;
  for (int c = lane * 8; c < hd; c += 256) {
    const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.out.ptr) + t * p.out.tok + h * p.out.head + c);
    const uint4 b = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.dout.ptr) + t * p.dout.tok + h * p.dout.head + c);
    const uint32_t ua[4] = {a.x, a.y, a.z, a.w}, ub[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 fa = unpack_pair<T>(ua[i]), fb = unpack_pair<T>(ub[i]);
      sum = fmaf(fa.x, fb.x, sum), sum = fmaf(fa.y, fb.y, sum);
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) {
    const int64_t at = static_cast<int64_t>(h) * p.s.n + t;
    const float lse = p.lse[at];
    if (p.dlse) sum -= p.dlse[at];
    // a row without a key (lse -inf) has weights of zero
    p.row[at] = make_float2(lse == -INFINITY ? INFINITY : lse * kLog2e - Shift<T>::kUp, sum * Shift<T>::kDown);
  }
}

// Columns a CTA sums gradients of: all, or halves above 128, whose accumulators would not fit the registers.
template <int DP>
struct Cols {
  static constexpr int N = DP > 128 ? DP / 2 : DP, PARTS = DP / N;
};

// ---------------------------------------------------------------- mma.sync: dk and dv of 64 keys
// Four warps, 16 keys each; tiles of 64 rows of every head of the group pass by. S^T and dP^T have the
// keys as rows, so that P^T and dS^T are A operands as they leave the registers.
template <int DP, class T>
__device__ __forceinline__ void keys_mma(const GradParams& p, const Tile& t, int hk, int part, unsigned char* smem) {
  using Sm = SmemTile<DP>;
  constexpr int NC = Cols<DP>::N / 16;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3, hd = p.s.hd;
  const uint32_t sk = smem_u32(smem), sv = sk + Sm::BYTES, sq = sv + Sm::BYTES, sd = sq + Sm::BYTES;
  float2* rows = reinterpret_cast<float2*>(smem + 4 * Sm::BYTES);
  int lo, hi;
  rows_of(p.s, t.len, t.row0, min(t.row0 + 64, t.len), lo, hi);
  const int rb = lo / 64, re = (hi + 63) / 64;
  stage_rows<DP, 128>(sk, p.k, t.first, t.len, t.row0, hk, hd);
  stage_rows<DP, 128>(sv, p.v, t.first, t.len, t.row0, hk, hd);
  float dk[2 * NC][4], dv[2 * NC][4];
#pragma unroll
  for (int i = 0; i < 2 * NC; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) dk[i][e] = dv[i][e] = 0.f;
  const int key0 = t.row0 + warp * 16 + g;
  for (int h = hk * p.s.group; h < (hk + 1) * p.s.group; ++h) {
    for (int j = rb; j < re; ++j) {
      __syncthreads();
      stage_rows<DP, 128>(sq, p.q, t.first, t.len, j * 64, h, hd);
      stage_rows<DP, 128>(sd, p.dout, t.first, t.len, j * 64, h, hd);
      cp_commit();
      if (threadIdx.x < 64)
        rows[threadIdx.x] = j * 64 + threadIdx.x < t.len
                                ? p.row[static_cast<int64_t>(h) * p.s.n + t.first + j * 64 + threadIdx.x]
                                : make_float2(INFINITY, 0.f);
      cp_wait<0>();
      __syncthreads();
      float x[8][4], d[8][4];
#pragma unroll
      for (int i = 0; i < 32; ++i) (&x[0][0])[i] = (&d[0][0])[i] = 0.f;
      product_t<DP, T>(x, sk, warp * 16, sq);
      product_t<DP, T>(d, sv, warp * 16, sd);
      uint32_t pa[4][4], da[4][4];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float pv[4], sv4[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = i * 8 + 2 * t4 + (e & 1), row = j * 64 + r, key = key0 + (e >> 1) * 8;
          const float2 rr = rows[r];
          const bool in = row < t.len && key >= row - p.s.left && key <= row + p.s.right && key < t.len;
          pv[e] = in ? fast_exp2(fmaf(x[i][e], p.s.scale_log2, -rr.x)) : 0.f;
          sv4[e] = in ? pv[e] * fmaf(d[i][e], Shift<T>::kDown, -rr.y) : 0.f;
        }
        pa[i >> 1][(i & 1) * 2] = pack_pair<T>(pv[0], pv[1]);
        pa[i >> 1][(i & 1) * 2 + 1] = pack_pair<T>(pv[2], pv[3]);
        da[i >> 1][(i & 1) * 2] = pack_pair<T>(sv4[0], sv4[1]);
        da[i >> 1][(i & 1) * 2 + 1] = pack_pair<T>(sv4[2], sv4[3]);
      }
      product<DP, NC, T>(dv, pa, sd, part * NC);
      product<DP, NC, T>(dk, da, sq, part * NC);
    }
  }
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
      *reinterpret_cast<uint32_t*>(ok + c + 2 * t4) = pack_pair<T>(dk[i][2 * e] * p.s.scale, dk[i][2 * e + 1] * p.s.scale);
      *reinterpret_cast<uint32_t*>(ov + c + 2 * t4) =
          pack_pair<T>(dv[i][2 * e] * Shift<T>::kDown, dv[i][2 * e + 1] * Shift<T>::kDown);
    }
  }
}

// ---------------------------------------------------------------- mma.sync: dq of 64 rows of one head
template <int DP, class T>
__device__ __forceinline__ void rows_mma(const GradParams& p, const Tile& t, int h, int part, unsigned char* smem) {
  using Sm = SmemTile<DP>;
  constexpr int NC = Cols<DP>::N / 16;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3, hd = p.s.hd;
  const int hk = h / p.s.group;
  const uint32_t sq = smem_u32(smem), sd = sq + Sm::BYTES, sk = sd + Sm::BYTES, sv = sk + Sm::BYTES;
  int lo, hi;
  keys_of(p.s, t.len, t.row0, min(t.row0 + 64, t.len), lo, hi);
  const int kb = lo / 64, ke = (hi + 63) / 64;
  stage_rows<DP, 128>(sq, p.q, t.first, t.len, t.row0, h, hd);
  stage_rows<DP, 128>(sd, p.dout, t.first, t.len, t.row0, h, hd);
  float dq[2 * NC][4];
#pragma unroll
  for (int i = 0; i < 2 * NC; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) dq[i][e] = 0.f;
  int klo[2], khi[2];
  float2 rr[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = t.row0 + warp * 16 + e * 8 + g;
    keys_of(p.s, t.len, r, r + 1, klo[e], khi[e]);
    if (r >= t.len) khi[e] = 0;
    rr[e] = r < t.len ? p.row[static_cast<int64_t>(h) * p.s.n + t.first + r] : make_float2(INFINITY, 0.f);
  }
  for (int j = kb; j < ke; ++j) {
    __syncthreads();
    stage_rows<DP, 128>(sk, p.k, t.first, t.len, j * 64, hk, hd);
    stage_rows<DP, 128>(sv, p.v, t.first, t.len, j * 64, hk, hd);
    cp_commit();
    cp_wait<0>();
    __syncthreads();
    float x[8][4], d[8][4];
#pragma unroll
    for (int i = 0; i < 32; ++i) (&x[0][0])[i] = (&d[0][0])[i] = 0.f;
    product_t<DP, T>(x, sq, warp * 16, sk);
    product_t<DP, T>(d, sd, warp * 16, sv);
    uint32_t da[4][4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float s4[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = j * 64 + i * 8 + 2 * t4 + (e & 1);
        const bool in = key >= klo[e >> 1] && key < khi[e >> 1];
        s4[e] = in ? fast_exp2(fmaf(x[i][e], p.s.scale_log2, -rr[e >> 1].x)) *
                         fmaf(d[i][e], Shift<T>::kDown, -rr[e >> 1].y)
                   : 0.f;
      }
      da[i >> 1][(i & 1) * 2] = pack_pair<T>(s4[0], s4[1]);
      da[i >> 1][(i & 1) * 2 + 1] = pack_pair<T>(s4[2], s4[3]);
    }
    product<DP, NC, T>(dq, da, sk, part * NC);
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = t.row0 + warp * 16 + e * 8 + g;
    if (r >= t.len) continue;
    T* o = static_cast<T*>(p.dq.ptr) + (t.first + r) * p.dq.tok + h * p.dq.head;
#pragma unroll
    for (int i = 0; i < 2 * NC; ++i) {
      const int c = part * NC * 16 + i * 8;
      if (c < hd)
        *reinterpret_cast<uint32_t*>(o + c + 2 * t4) = pack_pair<T>(dq[i][2 * e] * p.s.scale, dq[i][2 * e + 1] * p.s.scale);
    }
  }
}

// Blocks y < hkv: keys' gradients (more work each, so first); the others: a query head's.
template <int DP, class T>
__global__ void __launch_bounds__(128) prompt_grad_mma_kernel(const GradParams p) {
  extern __shared__ __align__(128) unsigned char smem[];
  wait_for_producer();
  Tile t;
  const bool keys = static_cast<int>(blockIdx.y) < p.s.hkv;
  // the first keys are seen by most rows, the last rows see most keys
  if (!find_tile<64>(p.s, keys ? blockIdx.x : gridDim.x - 1 - blockIdx.x, t)) return;
  if (keys) keys_mma<DP, T>(p, t, blockIdx.y, blockIdx.z, smem);
  else rows_mma<DP, T>(p, t, blockIdx.y - p.s.hkv, blockIdx.z, smem);
}

template <int DP, class T>
int launch_mma(const GradParams& p, cudaStream_t stream) {
  constexpr int smem = 4 * SmemTile<DP>::BYTES + 64 * 8;
  static std::atomic<uint64_t> configured{0};
  if (int s = allow_smem(prompt_grad_mma_kernel<DP, T>, smem, configured, "cudaFuncSetAttribute(prompt_grad)")) return s;
  return launch_behind(prompt_grad_mma_kernel<DP, T>, dim3(tile_numbers(p.s.n, p.s.b, 64), p.s.hkv + p.s.hq, Cols<DP>::PARTS),
                       128, smem, stream, "prompt_grad_mma_kernel", p);
}

template <class T>
int launch_grad(const GradParams& p, cudaStream_t stream) {
  const int64_t rows = static_cast<int64_t>(p.s.n) * p.s.hq;
  if (int s = launch_behind(prompt_delta_kernel<T>, dim3(static_cast<unsigned>((rows + 3) / 4)), 128, 0, stream,
                            "prompt_delta_kernel", p))
    return s;
  const int hd = p.s.hd;
  if (hd <= 64) return launch_mma<64, T>(p, stream);
  if (hd <= 96) return launch_mma<96, T>(p, stream);
  if (hd <= 128) return launch_mma<128, T>(p, stream);
  if (hd <= 192) return launch_mma<192, T>(p, stream);
  return launch_mma<256, T>(p, stream);
}

}  // namespace
}  // namespace fold

extern "C" {

int64_t fold_prompt_read_grad_workspace(int n, int hq, int hkv, int hd) {
  if (n < 0 || hq < 1 || hkv < 1 || hq % hkv || hq > 65535 || hd < 8 || hd > 256 || hd % 8) return -1;
  return static_cast<int64_t>(n) * hq * 8 + 16;
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
  if (!lse) return fail(FOLD_ERR_INVALID_ARGUMENT, "prompt read grad: null pointer");
  if (static_cast<int64_t>(n) * hq > (int64_t(1) << 32)) return fail(FOLD_ERR_INVALID_ARGUMENT, "prompt read grad: too many rows");
  if (!workspace || workspace_bytes < fold_prompt_read_grad_workspace(n, hq, hkv, hd))
    return fail(FOLD_ERR_INVALID_ARGUMENT, "prompt read grad: the workspace holds fold_prompt_read_grad_workspace bytes");
  if (!aligned16(workspace)) return fail(FOLD_ERR_ALIGNMENT, "prompt read grad: the workspace must be 16-byte aligned");
  p.lse = lse, p.dlse = dlse, p.row = static_cast<float2*>(workspace), p.zero_rest = zero_rest, p.err = err;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == FOLD_BF16 ? launch_grad<__nv_bfloat16>(p, st) : launch_grad<__half>(p, st);
}

}  // extern "C"
