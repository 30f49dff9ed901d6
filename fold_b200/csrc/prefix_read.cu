// Attention of a batch of sequences that share a prefix (fold_prefix_read). One warp per (token,
// query head): 32 keys at a time, lane = key for the logits, lanes = head dims for the values.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "host_common.h"

namespace fold {
namespace {

struct PrefixParams {
  const void* q;
  int64_t q_st, q_sh;
  const int* qsl;
  const int* own_lens;
  const int* prefix_len;
  int b;
  const void* k;
  const void* v;
  int64_t num_blocks;
  int block_size;
  int64_t cs_block, cs_head, cs_slot;
  const int* prefix_table;
  const int* tables;
  int64_t table_stride;
  int prefix_cap, own_cap;
  int causal;
  float scale_log2;
  void* out;
  int64_t o_st, o_sh;
  float* lse;
  int n, hq, group, hd;
  int* err;
};

__device__ __forceinline__ float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void store(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }
__device__ __forceinline__ void store(__half* p, float x) { *p = __float2half_rn(x); }

__device__ __forceinline__ int capped(int len, int cap, int* err) {
  if (len > cap) {
    set_error(err, FOLD_DEVERR_CAPACITY);
    len = cap;
  }
  return max(len, 0);
}

template <class T>
__global__ void prefix_read_kernel(const PrefixParams p) {
  __shared__ float qs[4][256];
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = blockIdx.x * 4ll + w;
  const int t = static_cast<int>(row / p.hq), h = static_cast<int>(row - static_cast<int64_t>(t) * p.hq);
  if (t >= p.n || t < p.qsl[0] || t >= p.qsl[p.b]) return;
  int s = 0;
  while (s + 1 < p.b && t >= p.qsl[s + 1]) ++s;
  const int hk = h / p.group;
  const T* qr = static_cast<const T*>(p.q) + t * p.q_st + h * p.q_sh;
  for (int d = lane; d < p.hd; d += 32) qs[w][d] = load(qr + d) * p.scale_log2;
  __syncwarp();
  float m = -INFINITY, l = 0.f, acc[8];
  for (int i = 0; i < 8; ++i) acc[i] = 0.f;
  for (int part = 0; part < 2; ++part) {
    int len = part == 0 ? capped(*p.prefix_len, p.prefix_cap, p.err) : capped(p.own_lens[s], p.own_cap, p.err);
    if (part == 1 && p.causal) len = max(min(len, len - (p.qsl[s + 1] - p.qsl[s]) + (t - p.qsl[s]) + 1), 0);
    const int* table = part == 0 ? p.prefix_table : p.tables + s * p.table_stride;
    for (int j0 = 0; j0 < len; j0 += 32) {
      const int j = j0 + lane;
      int64_t off = -1;
      if (j < len) {
        const int blk = table[j / p.block_size];
        if (blk < 0 || blk >= p.num_blocks) set_error(p.err, FOLD_DEVERR_BLOCK_TABLE);
        else off = blk * p.cs_block + hk * p.cs_head + (j % p.block_size) * p.cs_slot;
      }
      float x = j < len ? 0.f : -INFINITY;
      if (off >= 0)
        for (int d = 0; d < p.hd; ++d) x += qs[w][d] * load(static_cast<const T*>(p.k) + off + d);
      float mx = x;
      for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, o));
      const float mn = fmaxf(m, mx), c = exp2f(m - mn), e = exp2f(x - mn);
      m = mn, l = l * c + e;
      for (int i = 0; i < 8; ++i) acc[i] *= c;
      for (int k = 0; k < 32 && j0 + k < len; ++k) {
        const float pk = __shfl_sync(~0u, e, k);
        const int64_t ok = __shfl_sync(~0u, off, k);
        if (ok >= 0)
          for (int i = 0; i < p.hd / 32; ++i) acc[i] += pk * load(static_cast<const T*>(p.v) + ok + lane + 32 * i);
      }
    }
  }
  for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(~0u, l, o);
  T* o = static_cast<T*>(p.out) + t * p.o_st + h * p.o_sh;
  for (int i = 0; i < p.hd / 32; ++i) store(o + lane + 32 * i, l > 0.f ? acc[i] / l : 0.f);
  if (lane == 0 && p.lse) p.lse[static_cast<int64_t>(h) * p.n + t] = l > 0.f ? (m + log2f(l)) * kLn2 : -INFINITY;
}

}  // namespace
}  // namespace fold

extern "C" {

int64_t fold_prefix_read_workspace(int n, int hq, int hkv, int hd) {
  return n < 0 || hq < 1 || hkv < 1 || hq % hkv || (hd != 64 && hd != 128 && hd != 256) ? -1 : 0;
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
  if (n == 0 || b == 0) return FOLD_OK;
  if (!q || !qsl || !own_lens || !prefix_len || !k_cache || !v_cache || !prefix_table || !block_tables || !out)
    return fail(FOLD_ERR_INVALID_ARGUMENT, "prefix read: null pointer");
  PrefixParams p{q, q_stride_tok, q_stride_head, qsl, own_lens, prefix_len, b, k_cache, v_cache, num_blocks,
                 block_size, cache_stride_block, cache_stride_head, cache_stride_slot, prefix_table, block_tables,
                 block_tables_stride, prefix_table_len * block_size, block_tables_len * block_size, causal,
                 softmax_scale * kLog2e, out, o_stride_tok, o_stride_head, lse, n, hq, hq / hkv, hd, err};
  const unsigned grid = static_cast<unsigned>((static_cast<int64_t>(n) * hq + 3) / 4);
  if (dtype == FOLD_BF16) prefix_read_kernel<__nv_bfloat16><<<grid, 128, 0, static_cast<cudaStream_t>(stream)>>>(p);
  else prefix_read_kernel<__half><<<grid, 128, 0, static_cast<cudaStream_t>(stream)>>>(p);
  return check_launch("prefix_read_kernel");
}

}  // extern "C"
