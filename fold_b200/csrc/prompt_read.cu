// Attention over whole prompts (fold_prompt_read): sequences of different lengths packed one behind the
// other, heads in groups that share keys and values, causal or with a window.
//
// Mathematics. With x_rj = scale q_r.k_j for the keys j in [r - left, r + right] of r's sequence,
// o_r = sum_j e^(x_rj - lse_r) v_j and lse_r = log sum_j e^(x_rj). One pass over the keys keeps a running
// maximum m and sum l of each row and rescales what was summed when the maximum rises.
#include "prompt.cuh"

namespace fold {
namespace {
using namespace prompt;

struct ReadParams {
  Shape s;
  Rows q, k, v, out;
  float* lse;
  int* err;
};

// ---------------------------------------------------------------- mma.sync, any head size up to 256
// A CTA of four warps takes 64 rows of one head, a warp 16 of them; keys in tiles of 64, two stages.
template <int DP, class T>
__global__ void __launch_bounds__(128) prompt_read_mma_kernel(const ReadParams p) {
  using Sm = SmemTile<DP>;
  // weights in fp16 are held 2^10 up: small ones of many keys stay above its smallest step
  constexpr float kShift = std::is_same<T, __half>::value ? 10.f : 0.f;
  extern __shared__ __align__(128) unsigned char smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const uint32_t sq = smem_u32(smem), sk = sq + Sm::BYTES, sv = sk + 2 * Sm::BYTES;
  wait_for_producer();
  Tile t;
  if (!find_tile<64>(p.s, gridDim.x - 1 - blockIdx.x, t)) return;  // the last rows see most keys: first
  const int h = blockIdx.y, hk = h / p.s.group, hd = p.s.hd;
  int lo, hi;
  keys_of(p.s, t.len, t.row0, min(t.row0 + 64, t.len), lo, hi);
  const int kb = lo / 64, ke = (hi + 63) / 64;
  stage_rows<DP, 128>(sq, p.q, t.first, t.len, t.row0, h, hd);
  stage_rows<DP, 128>(sk, p.k, t.first, t.len, kb * 64, hk, hd);
  stage_rows<DP, 128>(sv, p.v, t.first, t.len, kb * 64, hk, hd);
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
      stage_rows<DP, 128>(sk + (st ^ 1) * Sm::BYTES, p.k, t.first, t.len, (j + 1) * 64, hk, hd);
      stage_rows<DP, 128>(sv + (st ^ 1) * Sm::BYTES, p.v, t.first, t.len, (j + 1) * 64, hk, hd);
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
  constexpr int smem = 5 * SmemTile<DP>::BYTES;
  static std::atomic<uint64_t> configured{0};
  if (int s = allow_smem(prompt_read_mma_kernel<DP, T>, smem, configured, "cudaFuncSetAttribute(prompt_read)")) return s;
  return launch_behind(prompt_read_mma_kernel<DP, T>, dim3(tile_numbers(p.s.n, p.s.b, 64), p.s.hq), 128, smem, stream,
                       "prompt_read_mma_kernel", p);
}

template <class T>
int launch_read(const ReadParams& p, cudaStream_t stream) {
  const int hd = p.s.hd;
  if (hd <= 64) return launch_mma<64, T>(p, stream);
  if (hd <= 96) return launch_mma<96, T>(p, stream);
  if (hd <= 128) return launch_mma<128, T>(p, stream);
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
  p.lse = lse, p.err = err;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == FOLD_BF16 ? launch_read<__nv_bfloat16>(p, st) : launch_read<__half>(p, st);
}

}  // extern "C"
