// Rotary positions (fold_rotary) and the append of keys and values to a paged cache with the
// rotation applied on the way (fold_append_paged).
//
// A pair (lo, hi) of a row at position p turns by the angle p * f_i:
//   lo' = lo cos - hi sin,   hi' = hi cos + lo sin      (inverse: sin negated, the transpose)
// with cos and sin taken from a float32 table formed in float64 (row p: cos then sin, both times
// the attention factor of scaled frequencies). Pairs are (i, i + rot/2) or, interleaved,
// (2i, 2i+1); dims past rot pass through. Arithmetic is float32 with one rounding to the type.
//
// Bound: HBM bytes, each row read once and written once; a token's table row is shared by all its
// heads. So one thread owns one unit, two chunks of W bytes that hold whole pairs (chunk c of each
// half; two neighbouring chunks when interleaved or passed through), of HU heads of one token: the
// table values are loaded once for the HU heads, and 2 * HU loads are in flight while the position
// and then the table row are fetched. W is 16, or 8 or 4 where the halves or the rows start on such
// boundaries only. What counts besides is how many threads wait at once:
// 64 registers and blocks of 128. At 8192 tokens of 32 + 8 heads of 128 (168 MB) HU 4 with blocks of
// 256 took 40.5 us, HU 2 37.3, HU 2 with blocks of 128 35.5 us (4.7 TB/s; a device copy of as much
// by torch takes 59 us); 16K tokens appended with their queries (403 MB) 93.5, 76.2 and 72.4 us
// (5.6 TB/s). Streaming loads and stores, and the table before the rows, were slower.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <initializer_list>
#include <utility>

#include "common.cuh"
#include "host_common.h"

namespace fold {
namespace {

constexpr int kRopeThreads = 128;

struct RopeRows {  // rows [n, heads, hd] with the innermost dim contiguous
  const void* in;
  void* out;
  int64_t in_st, in_sh, out_st, out_sh;
  int heads;
};

struct RopeParams {
  RopeRows q, k, v;  // v.heads = 0 outside the append
  const int64_t* positions;
  const int64_t* slots;  // null: k goes to its out rows; else k and v go to the cache
  int64_t num_slots, cs_block, cs_head, cs_slot;
  int block_size;
  const float* table;  // null: nothing is rotated
  int64_t table_rows;
  int n, hd, rot;
  float sgn;  // -1: the transposed rotation
  int* err;
};

template <class T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_f32(float x) { return x; }
template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f32(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ float from_f32(float x) { return x; }

template <int W>
struct Word;
template <>
struct Word<16> { using type = uint4; };
template <>
struct Word<8> { using type = uint2; };
template <>
struct Word<4> { using type = uint32_t; };
// A chunk of W bytes.
template <class T, int W>
union Chunk {
  typename Word<W>::type raw;
  T e[W / sizeof(T)];
};
// N consecutive floats of the table (N * 4 bytes aligned, or 16).
template <int N>
__device__ __forceinline__ void load_floats(const float* p, float* v) {
  if constexpr (N >= 4) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 u = __ldg(reinterpret_cast<const float4*>(p + i));
      v[i] = u.x, v[i + 1] = u.y, v[i + 2] = u.z, v[i + 3] = u.w;
    }
  } else if constexpr (N == 2) {
    const float2 u = __ldg(reinterpret_cast<const float2*>(p));
    v[0] = u.x, v[1] = u.y;
  } else {
    v[0] = __ldg(p);
  }
}

// The table row of token t (a position outside the table is clamped and, where asked, reported).
__device__ __forceinline__ const float* table_row(const RopeParams& p, int t, bool report) {
  if (!p.table) return nullptr;
  int64_t pos = __ldg(p.positions + t);
  if (pos < 0 || pos >= p.table_rows) {
    if (report) set_error(p.err, FOLD_DEVERR_ROPE_RANGE);
    pos = pos < 0 ? 0 : p.table_rows - 1;
  }
  return p.table + pos * p.rot;
}

// Source and destination rows of head hh of token t, heads counted q, then k, then v. No
// destination (false): the token's slot is negative or outside the cache.
template <class T>
__device__ __forceinline__ bool locate(const RopeParams& p, int t, int hh, const T*& src, T*& dst) {
  const bool is_q = hh < p.q.heads;
  const RopeRows& r = is_q ? p.q : hh < p.q.heads + p.k.heads ? p.k : p.v;
  const int h = is_q ? hh : hh < p.q.heads + p.k.heads ? hh - p.q.heads : hh - p.q.heads - p.k.heads;
  src = static_cast<const T*>(r.in) + t * r.in_st + h * r.in_sh;
  if (is_q || !p.slots) {
    dst = static_cast<T*>(r.out) + t * r.out_st + h * r.out_sh;
    return true;
  }
  const int64_t slot = __ldg(p.slots + t);
  if (slot < 0) return false;
  if (slot >= p.num_slots) {
    set_error(p.err, FOLD_DEVERR_APPEND_RANGE);
    return false;
  }
  const int64_t block = (slot >> 32) == 0 ? static_cast<int64_t>(static_cast<uint32_t>(slot) /
                                                                 static_cast<uint32_t>(p.block_size))
                                          : slot / p.block_size;
  dst = static_cast<T*>(r.out) + block * p.cs_block + h * p.cs_head + (slot - block * p.block_size) * p.cs_slot;
  return true;
}

// One thread per (token, group of HU heads, unit); neighbouring threads walk a row's units.
template <class T, bool INTER, int W, int HU>
__global__ void __launch_bounds__(kRopeThreads, 8) rope_kernel(const RopeParams p) {
  constexpr int E = W / sizeof(T);
  using word = typename Word<W>::type;
  if (p.q.heads == 0) release_dependents();  // no query is written: a read behind may load its own early
  const int units = p.hd / (2 * E), runits = p.table ? p.rot / (2 * E) : 0;
  const int heads = p.q.heads + p.k.heads + p.v.heads, groups = (heads + HU - 1) / HU;
  const int rotated = p.q.heads + p.k.heads;  // v is stored as it is
  const int64_t total = static_cast<int64_t>(p.n) * groups * units;
  for (int64_t idx = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; idx < total;
       idx += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    // one 64-bit division a thread at most, none where the product fits 32 bits
    int t, rest;
    const int per = groups * units;
    if ((idx >> 32) == 0) {
      t = static_cast<int>(static_cast<uint32_t>(idx) / static_cast<uint32_t>(per));
      rest = static_cast<int>(static_cast<uint32_t>(idx) - static_cast<uint32_t>(t) * static_cast<uint32_t>(per));
    } else {
      t = static_cast<int>(idx / per), rest = static_cast<int>(idx - static_cast<int64_t>(t) * per);
    }
    const int g = rest / units, c = rest - g * units;
    const bool turn = c < runits;
    // element offsets of the unit's two chunks
    int a, b;
    if (turn && !INTER) a = c * E, b = (p.rot >> 1) + c * E;
    else if (turn) a = 2 * c * E, b = a + E;
    else a = runits * 2 * E + 2 * (c - runits) * E, b = a + E;

    Chunk<T, W> x[HU], y[HU];
    T* dst[HU];
    bool live[HU], any = false;  // any: a head of these is turned and written
#pragma unroll
    for (int j = 0; j < HU; ++j) {
      const T* src = nullptr;
      const int hh = g * HU + j;
      live[j] = hh < heads && locate<T>(p, t, hh, src, dst[j]);
      any |= live[j] && hh < rotated;
      if (live[j]) {
        x[j].raw = *reinterpret_cast<const word*>(src + a);
        y[j].raw = *reinterpret_cast<const word*>(src + b);
      }
    }
    float cs[E], sn[E];
    if (turn && g * HU < rotated) {
      // the row is fetched beside the slot, whatever that says; a skipped token's position is no error
      const float* row = table_row(p, t, any);
      load_floats<E>(row + c * E, cs);
      load_floats<E>(row + (p.rot >> 1) + c * E, sn);
#pragma unroll
      for (int i = 0; i < E; ++i) sn[i] *= p.sgn;
    }
#pragma unroll
    for (int j = 0; j < HU; ++j) {
      if (!live[j]) continue;
      if (turn && g * HU + j < rotated) {
        Chunk<T, W> ox, oy;
        if constexpr (INTER && E > 1) {  // pair i of the unit: elements 2i, 2i + 1 of the two chunks in a row
#pragma unroll
          for (int i = 0; i < E; ++i) {
            const Chunk<T, W>& s = i < E / 2 ? x[j] : y[j];
            Chunk<T, W>& o = i < E / 2 ? ox : oy;
            const int e = 2 * (i < E / 2 ? i : i - E / 2);
            const float lo = to_f32(s.e[e]), hi = to_f32(s.e[e + 1]);
            o.e[e] = from_f32<T>(lo * cs[i] - hi * sn[i]);
            o.e[e + 1] = from_f32<T>(hi * cs[i] + lo * sn[i]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < E; ++i) {
            const float lo = to_f32(x[j].e[i]), hi = to_f32(y[j].e[i]);
            ox.e[i] = from_f32<T>(lo * cs[i] - hi * sn[i]);
            oy.e[i] = from_f32<T>(hi * cs[i] + lo * sn[i]);
          }
        }
        x[j] = ox, y[j] = oy;
      }
      *reinterpret_cast<word*>(dst[j] + a) = x[j].raw;
      *reinterpret_cast<word*>(dst[j] + b) = y[j].raw;
    }
  }
}

// Rows that no such unit covers (an odd number of pairs in halves of 2-byte elements, rows off every
// boundary): a warp per row, a lane per pair and per passed-through element.
template <class T, bool INTER>
__global__ void __launch_bounds__(kRopeThreads) rope_scalar_kernel(const RopeParams p) {
  if (p.q.heads == 0) release_dependents();
  const int rot = p.table ? p.rot : 0, half = rot >> 1;
  const uint32_t heads = p.q.heads + p.k.heads + p.v.heads;
  const int rotated = p.q.heads + p.k.heads, lane = threadIdx.x & 31;
  const int64_t rows = static_cast<int64_t>(p.n) * heads, warps = static_cast<int64_t>(gridDim.x) * (kRopeThreads / 32);
  for (int64_t row = blockIdx.x * static_cast<int64_t>(kRopeThreads / 32) + (threadIdx.x >> 5); row < rows; row += warps) {
    const int t = (row >> 32) == 0 ? static_cast<int>(static_cast<uint32_t>(row) / heads) : static_cast<int>(row / heads);
    const int hh = static_cast<int>(row - static_cast<int64_t>(t) * heads);
    const T* src;
    T* dst;
    if (!locate<T>(p, t, hh, src, dst)) continue;
    if (hh >= rotated || half == 0) {
      for (int i = lane; i < p.hd; i += 32) dst[i] = src[i];
      continue;
    }
    const float* tr = table_row(p, t, true);
    for (int c = lane; c < half; c += 32) {
      const int a = INTER ? 2 * c : c, b = INTER ? 2 * c + 1 : c + half;
      const float lo = to_f32(src[a]), hi = to_f32(src[b]), cs = __ldg(tr + c), sn = p.sgn * __ldg(tr + half + c);
      dst[a] = from_f32<T>(lo * cs - hi * sn), dst[b] = from_f32<T>(hi * cs + lo * sn);
    }
    for (int i = rot + lane; i < p.hd; i += 32) dst[i] = src[i];
  }
}

// Whether every row of r starts on a boundary of `bytes` (es: element size).
bool rows_aligned(const RopeRows& r, int es, int bytes, bool with_out) {
  if (r.heads == 0) return true;
  const int64_t e = bytes / es;
  auto on = [&](const void* x) { return (reinterpret_cast<uintptr_t>(x) & (bytes - 1)) == 0; };
  return on(r.in) && r.in_st % e == 0 && r.in_sh % e == 0 &&
         (!with_out || (on(r.out) && r.out_st % e == 0 && r.out_sh % e == 0));
}

// Whether units of two chunks of W bytes cover the rows.
template <class T, int W>
bool units_fit(const RopeParams& p) {
  constexpr int E = W / sizeof(T);
  const bool to_cache = p.slots != nullptr;
  bool fit = p.hd % (2 * E) == 0 && (!p.table || (p.rot % (2 * E) == 0 && aligned16(p.table))) &&
             rows_aligned(p.q, sizeof(T), W, true) && rows_aligned(p.k, sizeof(T), W, !to_cache) &&
             rows_aligned(p.v, sizeof(T), W, false);
  if (to_cache)
    fit = fit && (reinterpret_cast<uintptr_t>(p.k.out) & (W - 1)) == 0 &&
          (reinterpret_cast<uintptr_t>(p.v.out) & (W - 1)) == 0 && p.cs_block % E == 0 && p.cs_head % E == 0 &&
          p.cs_slot % E == 0;
  return fit;
}

unsigned rope_grid(int64_t threads) {
  int sms = device_sm_count();
  if (sms <= 0) sms = 148;
  const int64_t want = (threads + kRopeThreads - 1) / kRopeThreads, cap = static_cast<int64_t>(sms) * 64;
  return static_cast<unsigned>(want < cap ? want : cap);
}

template <class T, bool INTER, int W>
int launch_units(const RopeParams& p, cudaStream_t stream) {
  constexpr int E = W / sizeof(T);
  const int heads = p.q.heads + p.k.heads + p.v.heads, units = p.hd / (2 * E);
  const int64_t all = static_cast<int64_t>(p.n) * heads * units;
  // up to about 1000 units an SM one head a thread is the shortest chain (1 to 256 tokens of 40 heads:
  // 2.1-2.9 us, two heads 2.7-3.4 us; equal at 512 tokens, 4.0 us); from there two heads, 10.6 against
  // 12.1 us at 2048
  if (all <= 148 * 1024)
    rope_kernel<T, INTER, W, 1><<<rope_grid(all), kRopeThreads, 0, stream>>>(p);
  else
    rope_kernel<T, INTER, W, 2><<<rope_grid(static_cast<int64_t>(p.n) * ((heads + 1) / 2) * units), kRopeThreads, 0, stream>>>(p);
  return check_launch("rope_kernel");
}

template <class T, bool INTER>
int launch_rope(const RopeParams& p, cudaStream_t stream) {
  if (units_fit<T, 16>(p)) return launch_units<T, INTER, 16>(p, stream);
  if (units_fit<T, 8>(p)) return launch_units<T, INTER, 8>(p, stream);
  if constexpr (sizeof(T) == 2) {
    if (units_fit<T, 4>(p)) return launch_units<T, INTER, 4>(p, stream);
  }
  const int64_t rows = static_cast<int64_t>(p.n) * (p.q.heads + p.k.heads + p.v.heads);
  rope_scalar_kernel<T, INTER><<<rope_grid(rows * 32), kRopeThreads, 0, stream>>>(p);
  return check_launch("rope_scalar_kernel");
}

int dispatch_rope(const RopeParams& p, int dtype, int interleaved, cudaStream_t stream) {
  switch (dtype) {
    case FOLD_BF16:
      return interleaved ? launch_rope<__nv_bfloat16, true>(p, stream) : launch_rope<__nv_bfloat16, false>(p, stream);
    case FOLD_FP16: return interleaved ? launch_rope<__half, true>(p, stream) : launch_rope<__half, false>(p, stream);
    default: return interleaved ? launch_rope<float, true>(p, stream) : launch_rope<float, false>(p, stream);
  }
}

int check_rope(const float* table, int64_t table_rows, int rot_dim, int n, int hd, int dtype, const char* what) {
  const std::string w(what);
  if (n < 0 || hd < 1) return fail(FOLD_ERR_INVALID_ARGUMENT, w + ": bad sizes");
  if (hd > 8192) return fail(FOLD_ERR_UNSUPPORTED, w + ": heads of at most 8192 elements");
  if (dtype != FOLD_BF16 && dtype != FOLD_FP16 && dtype != FOLD_FP32)
    return fail(FOLD_ERR_INVALID_ARGUMENT, w + ": unknown type");
  if (table && (table_rows < 1 || rot_dim < 2 || rot_dim % 2 || rot_dim > hd))
    return fail(FOLD_ERR_INVALID_ARGUMENT, w + ": the table has rows of rot_dim floats, rot_dim even and at most hd");
  return FOLD_OK;
}

// Whether rows of hd elements at these strides (of dims of `size` each) cannot be told apart in memory:
// two neighbours of some dim overlap.
bool neighbours_overlap(int hd, std::initializer_list<std::pair<int64_t, int64_t>> dims) {
  for (const auto& [size, stride] : dims)
    if (size > 1 && stride < hd && stride > -hd) return true;
  return false;
}

}  // namespace
}  // namespace fold

extern "C" {

int fold_rotary(const void* q, int64_t q_stride_tok, int64_t q_stride_head, void* q_out, int64_t qo_stride_tok,
                int64_t qo_stride_head, int hq, const void* k, int64_t k_stride_tok, int64_t k_stride_head,
                void* k_out, int64_t ko_stride_tok, int64_t ko_stride_head, int hk, const int64_t* positions,
                const float* rope_table, int64_t table_rows, int rot_dim, int n, int hd, int dtype, int interleaved,
                int inverse, int* err, void* stream) {
  using namespace fold;
  if (int s = check_rope(rope_table, table_rows, rot_dim, n, hd, dtype, "rotary")) return s;
  if (hq < 0 || hk < 0 || hq > 16384 || hk > 16384) return fail(FOLD_ERR_INVALID_ARGUMENT, "rotary: bad sizes");
  if (n == 0 || hq + hk == 0) return FOLD_OK;
  if (!positions || !rope_table || (hq && (!q || !q_out)) || (hk && (!k || !k_out)))
    return fail(FOLD_ERR_INVALID_ARGUMENT, "rotary: null pointer");
  if ((hq && neighbours_overlap(hd, {{n, qo_stride_tok}, {hq, qo_stride_head}})) ||
      (hk && neighbours_overlap(hd, {{n, ko_stride_tok}, {hk, ko_stride_head}})))
    return fail(FOLD_ERR_INVALID_ARGUMENT, "rotary: the rows of an output must not share memory");
  RopeParams p{};
  p.q = RopeRows{q, q_out, q_stride_tok, q_stride_head, qo_stride_tok, qo_stride_head, hq};
  p.k = RopeRows{k, k_out, k_stride_tok, k_stride_head, ko_stride_tok, ko_stride_head, hk};
  // a call of keys alone still writes rows that a read behind it may load: count them as queries
  if (hq == 0) p.q = p.k, p.k = RopeRows{};
  p.positions = positions, p.table = rope_table, p.table_rows = table_rows;
  p.n = n, p.hd = hd, p.rot = rot_dim, p.sgn = inverse ? -1.f : 1.f, p.err = err;
  return dispatch_rope(p, dtype, interleaved, static_cast<cudaStream_t>(stream));
}

int fold_append_paged(const void* k, int64_t k_stride_tok, int64_t k_stride_head, const void* v, int64_t v_stride_tok,
                      int64_t v_stride_head, const int64_t* positions, const int64_t* slots, int n, void* k_cache,
                      void* v_cache, int64_t num_blocks, int block_size, int64_t cache_stride_block,
                      int64_t cache_stride_head, int64_t cache_stride_slot, const float* rope_table,
                      int64_t table_rows, int rot_dim, int hkv, int hd, int dtype, int interleaved, const void* q,
                      int64_t q_stride_tok, int64_t q_stride_head, void* q_out, int64_t qo_stride_tok,
                      int64_t qo_stride_head, int hq, int* err, void* stream) {
  using namespace fold;
  if (int s = check_rope(rope_table, table_rows, rot_dim, n, hd, dtype, "paged append")) return s;
  if (hkv < 1 || hkv > 16384 || hq < 0 || hq > 16384 || num_blocks < 1 || block_size < 1 ||
      num_blocks > (int64_t(1) << 40))
    return fail(FOLD_ERR_INVALID_ARGUMENT, "paged append: bad sizes");
  if (n == 0) return FOLD_OK;
  if (!k || !v || !slots || !k_cache || !v_cache || (rope_table && !positions) || (hq && (!q || !q_out)))
    return fail(FOLD_ERR_INVALID_ARGUMENT, "paged append: null pointer");
  if (hq && !rope_table) return fail(FOLD_ERR_INVALID_ARGUMENT, "paged append: queries are given only to be rotated");
  if (hq && neighbours_overlap(hd, {{n, qo_stride_tok}, {hq, qo_stride_head}}))
    return fail(FOLD_ERR_INVALID_ARGUMENT, "paged append: the rows of an output must not share memory");
  const int64_t apart = static_cast<const char*>(v_cache) - static_cast<const char*>(k_cache);
  const int64_t row_bytes = static_cast<int64_t>(hd) * (dtype == FOLD_FP32 ? 4 : 2);
  if (neighbours_overlap(hd, {{num_blocks, cache_stride_block}, {hkv, cache_stride_head}, {block_size, cache_stride_slot}}) ||
      (apart < row_bytes && apart > -row_bytes))
    return fail(FOLD_ERR_INVALID_ARGUMENT, "paged append: the slots of the cache's planes must not share memory");
  RopeParams p{};
  p.q = RopeRows{q, q_out, q_stride_tok, q_stride_head, qo_stride_tok, qo_stride_head, hq};
  p.k = RopeRows{k, k_cache, k_stride_tok, k_stride_head, 0, 0, hkv};
  p.v = RopeRows{v, v_cache, v_stride_tok, v_stride_head, 0, 0, hkv};
  p.positions = positions, p.slots = slots, p.num_slots = num_blocks * block_size, p.block_size = block_size;
  p.cs_block = cache_stride_block, p.cs_head = cache_stride_head, p.cs_slot = cache_stride_slot;
  p.table = rope_table, p.table_rows = table_rows, p.rot = rope_table ? rot_dim : 0;
  p.n = n, p.hd = hd, p.sgn = 1.f, p.err = err;
  return dispatch_rope(p, dtype, interleaved, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
