// Shared by the attention over whole prompts and its gradient: the packed sequences' row tiles, the
// keys a row sees, tiles staged by cp.async, fragments of mma.sync.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "host_common.h"

namespace fold {
namespace prompt {

// A [n, heads, hd] operand: element strides of tokens and heads, heads contiguous.
struct Rows {
  void* ptr;
  int64_t tok, head;
};

struct Shape {
  const int* qsl;
  int b, n, hq, hkv, group, hd;
  int left, right;   // row r sees keys [r - left, r + right] of its sequence
  float scale, scale_log2;
};

constexpr int kUnbounded = 0x3fffffff;  // of left and right: more than any sequence holds

// Rows [first, last) of sequence s, kept inside [0, n] whatever qsl holds.
__device__ __forceinline__ void seq_rows(const Shape& p, int s, int& first, int& last) {
  first = min(max(__ldg(p.qsl + s), 0), p.n);
  last = min(max(__ldg(p.qsl + s + 1), first), p.n);
}

// The packed sequences are cut into tiles of T rows that start at each sequence's first row. Tile t of
// sequence s has the number qsl[s] / T + s + t: a sequence of len rows from row a on has
// ceil(len / T) <= (a + len) / T - a / T + 1 tiles, so the numbers do not meet, and n / T + b of them
// cover every packing without a look at the lengths on the host. Numbers that no tile has are idle.
__host__ __device__ __forceinline__ int tile_numbers(int n, int b, int T) { return n / T + b; }

struct Tile {
  int seq, first, len, row0;  // row0: the tile's first row in the sequence
};

// The last sequence s with before(s, qsl[s]), which holds up to some sequence and not behind it; -1: none. A search
// of 32 probes a round; all lanes of a warp call this.
template <class F>
__device__ __forceinline__ int last_sequence(const Shape& p, F before) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = p.b;  // the sequence lies in [lo, hi)
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, s = lo + lane * step;
    const uint32_t m = __ballot_sync(0xffffffffu, s < hi && before(s, min(max(__ldg(p.qsl + s), 0), p.n)));
    if (m == 0) return -1;
    const int at = 31 - __clz(m);
    lo += at * step;
    hi = min(hi, lo + step);
  }
  return lo;
}

// Tile number x; false: idle.
template <int T>
__device__ __forceinline__ bool find_tile(const Shape& p, int x, Tile& t) {
  const int lo = last_sequence(p, [&](int s, int first) { return first / T + s <= x; });
  if (lo < 0) return false;
  int first, last;
  seq_rows(p, lo, first, last);
  t.seq = lo, t.first = first, t.len = last - first;
  t.row0 = (x - first / T - lo) * T;
  return t.row0 >= 0 && t.row0 < t.len;
}

// Keys that any of rows [r0, r1) of a sequence of len sees: [lo, hi).
__device__ __forceinline__ void keys_of(const Shape& p, int len, int r0, int r1, int& lo, int& hi) {
  lo = max(r0 - p.left, 0), hi = min(r1 + p.right, len);  // right at most kUnbounded, r1 at most 2^30
}
// Rows that see any of keys [k0, k1): [lo, hi).
__device__ __forceinline__ void rows_of(const Shape& p, int len, int k0, int k1, int& lo, int& hi) {
  lo = max(k0 - p.right, 0), hi = min(k1 + p.left, len);
}

template <class T>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    return pack_bf16(lo, hi);
  } else {  // past the f16 range: infinite, as a scaler of losses looks for
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
template <class T>
__device__ __forceinline__ float2 unpack_pair(uint32_t x) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
  else return __half22float2(*reinterpret_cast<const __half2*>(&x));
}

// Sixteen elements of a row: one sector where rows lie on 32 bytes (`wide`), else two halves; `cols`: how many of them
// the row has (16 or 8). A warp that stores a row a lane moves a line a cycle, so fewer, wider stores.
__device__ __forceinline__ void store_row16(void* dst, const uint32_t* w, bool wide, int cols) {
  if (wide && cols >= 16) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                 "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  } else {
    if (cols >= 8) static_cast<uint4*>(dst)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    if (cols >= 16) static_cast<uint4*>(dst)[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}
__device__ __forceinline__ bool rows_on_32(const Rows& x) {
  return ((reinterpret_cast<uintptr_t>(x.ptr) | static_cast<uintptr_t>(x.tok) * 2 | static_cast<uintptr_t>(x.head) * 2) & 31u) == 0;
}

template <class T>
__device__ __forceinline__ void mma_t(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) mma_bf16(d, a[0], a[1], a[2], a[3], b0, b1);
  else mma_f16(d, a[0], a[1], a[2], a[3], b0, b1);
}

// ---------------------------------------------------------------- blocks that take tiles as they come
// The grid has a block a tile; one that is through asks for the number of a block that has not started yet, and
// that block never does: long and short tiles even out, and a tile's start overlaps the end of the one before.
__device__ __forceinline__ void ask_next_block(void* answer, uint64_t* bar) {
  fence_proxy_async_smem();  // the last answer has been read
  mbar_arrive_expect_tx(bar, 16);
  asm volatile(
      "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(smem_u32(answer)),
      "r"(smem_u32(bar))
      : "memory");
}
// The number that was answered, or -1: all blocks have started.
__device__ __forceinline__ int next_block(const void* answer) {
  uint32_t got, x;
  asm volatile(
      "{\n\t.reg .b128 a;\n\t.reg .pred p;\n\t"
      "mov.u32 %1, 0;\n\t"
      "ld.shared.b128 a, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, a;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, a;\n\t}"
      : "=&r"(got), "=&r"(x)
      : "r"(smem_u32(answer))
      : "memory");
  return got ? static_cast<int>(x) : -1;
}

// ---------------------------------------------------------------- tiles of 16-bit rows in shared memory
// Rows of DP columns, padded by 16 bytes so that eight rows' chunks of 16 bytes hit all banks.
template <int DP>
struct SmemTile {
  static constexpr int ROW = DP * 2 + 16, BYTES = 64 * ROW;  // of 64 rows
};

// Copies rows [r0, r0 + R) of a sequence (rows from `len` on and columns from hd on become zeros).
template <int DP, int NT, int R = 64>
__device__ __forceinline__ void stage_rows(uint32_t dst, const Rows& x, int first, int len, int r0, int head, int hd) {
  const char* base = static_cast<const char*>(x.ptr) + head * x.head * 2;
  for (int e = threadIdx.x; e < R * (DP / 8); e += NT) {
    const int r = e / (DP / 8), c = e - r * (DP / 8);
    const bool in = r0 + r < len && c * 8 < hd;
    const char* src = in ? base + (static_cast<int64_t>(first + r0 + r) * x.tok + c * 8) * 2 : static_cast<const char*>(x.ptr);
    cp_async_16(dst + r * SmemTile<DP>::ROW + c * 16, src, in ? 16u : 0u);
  }
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A operand: 16 rows from row0 on, columns [16 kk, 16 kk + 16).
template <int DP>
__device__ __forceinline__ void frag_a(uint32_t tile, int row0, int kk, uint32_t (&a)[4]) {
  const int lane = threadIdx.x & 31, mi = lane >> 3, mr = lane & 7;
  ldsm_x4(tile + (row0 + (mi & 1) * 8 + mr) * SmemTile<DP>::ROW + (2 * kk + (mi >> 1)) * 16, a[0], a[1], a[2], a[3]);
}
// B operand of X Y^T: rows of Y are the columns of the product; b[0..1] columns n0 .. n0 + 7, b[2..3] the next 8.
template <int DP>
__device__ __forceinline__ void frag_bt(uint32_t tile, int n0, int kk, uint32_t (&b)[4]) {
  const int lane = threadIdx.x & 31, mi = lane >> 3, mr = lane & 7;
  ldsm_x4(tile + (n0 + (mi >> 1) * 8 + mr) * SmemTile<DP>::ROW + (2 * kk + (mi & 1)) * 16, b[0], b[1], b[2], b[3]);
}
// B operand of X Y: 16 rows k0 .. k0 + 15 of Y, columns [16 c, 16 c + 16).
template <int DP>
__device__ __forceinline__ void frag_b(uint32_t tile, int k0, int c, uint32_t (&b)[4]) {
  const int lane = threadIdx.x & 31, mi = lane >> 3, mr = lane & 7;
  ldsm_x4_t(tile + (k0 + (mi & 1) * 8 + mr) * SmemTile<DP>::ROW + (2 * c + (mi >> 1)) * 16, b[0], b[1], b[2], b[3]);
}
// 16 x 64 += (16 rows from row0 of A) (64 rows of B)^T.
template <int DP, class T>
__device__ __forceinline__ void product_t(float (&d)[8][4], uint32_t ta, int row0, uint32_t tb) {
#pragma unroll
  for (int kk = 0; kk < DP / 16; ++kk) {
    uint32_t a[4];
    frag_a<DP>(ta, row0, kk, a);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      uint32_t b[4];
      frag_bt<DP>(tb, c * 16, kk, b);
      mma_t<T>(d[2 * c], a, b[0], b[1]);
      mma_t<T>(d[2 * c + 1], a, b[2], b[3]);
    }
  }
}
// 16 x 16 NC += (16 x 64, as A fragments) (64 rows of B, columns from 16 c0 on).
template <int DP, int NC, class T>
__device__ __forceinline__ void product(float (&d)[2 * NC][4], const uint32_t (&a)[4][4], uint32_t tb, int c0) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      uint32_t b[4];
      frag_b<DP>(tb, k * 16, c0 + c, b);
      mma_t<T>(d[2 * c], a[k], b[0], b[1]);
      mma_t<T>(d[2 * c + 1], a[k], b[2], b[3]);
    }
  }
}

}  // namespace prompt

// ---------------------------------------------------------------- host
// Shared checks of fold_prompt_read and fold_prompt_read_grad; fills `p`. `what` opens the messages.
int prompt_shape(const char* what, const int* qsl, int b, int n, int hq, int hkv, int hd, int dtype, int causal,
                 int window_left, int window_right, float softmax_scale, prompt::Shape* p);
// An operand's pointer, alignment and strides; `written`: its rows must not share memory.
int prompt_rows(const char* what, const char* name, const void* ptr, int64_t tok, int64_t head, int n, int heads,
                int hd, bool written, prompt::Rows* out);
// Whether two operands of n rows share memory: exact for views of one tensor, whose tokens (or heads, where those come
// first) lie at one stride; operands at other strides that reach into each other are taken to.
bool prompt_overlap(prompt::Rows a, int heads_a, prompt::Rows b, int heads_b, int n, int hd);
// Map of an operand: columns, heads, rows; a box is 64 columns of `rows` rows of one head.
int prompt_map(const char* what, const prompt::Rows& x, int heads, int n, int hd, int rows, bool f16, CUtensorMap* out);

}  // namespace fold
