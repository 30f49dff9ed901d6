// Who holds which page of a paged cache, kept on the device: pages for new tokens (fold_grow_pages),
// sequences forked (fold_fork_pages), tokens dropped and pages given back (fold_free_pages).
//
// State. refs[p] counts the rows of the block tables that hold page p (0: free); a row of lens[r] tokens
// holds the first ceil(lens[r] / block_size) entries of its table. The k-th page that a call takes is the
// k-th lowest free one, so the result does not depend on the order in which threads run.
//
// A page that more than one row holds is never written: a fork shares the full pages and copies a partly
// filled last one, and a row whose partly filled last page is shared (it was trimmed into it) cannot grow.
//
// What bounds them: grow and the plan of a fork are chains of a few dependent reads in one block; the
// search reads refs from the start until it has found enough free pages (16K counts a round). The copy of
// a fork is memory bound. Measured (the GPU's time): five tokens of one sequence grown and trimmed 7 us (two
// launches), 20000 tokens of 250 sequences 17.5 us; 160 children of 40 sequences in 24 layers, 237 MB copied, with
// their rows freed before, 80 us (5.9 TB/s, 0.90 of the measured copy rate).
#include "common.cuh"
#include "host_common.h"

namespace fold {
namespace {

constexpr int kThreads = 1024;
constexpr int kMaxSeqs = 16384;  // sequences a call: three words each in shared memory
constexpr int kPer = 16;         // counts a thread looks at in a round of the search

struct Pool {
  int* refs;
  int pages;
  int* tables;
  int64_t stride;
  int width;  // entries of a table
  int* lens;
  int rows;
  int bs;
  int* err;

  __device__ __forceinline__ int pages_of(int tokens) const { return tokens / bs + (tokens % bs != 0); }
  // tokens that a table can hold
  __device__ __forceinline__ int capacity() const {
    const int64_t c = static_cast<int64_t>(width) * bs;
    return c < 0x7fffffff ? static_cast<int>(c) : 0x7fffffff;
  }
  __device__ __forceinline__ int* entry(int row, int j) const { return tables + row * stride + j; }
};

// Sum of `x` over the block's threads before this one; `total` of all. One word a warp in `scratch`.
__device__ __forceinline__ int block_scan(int x, int* scratch, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  __syncthreads();  // scratch may still be read
  if (lane == 31) scratch[warp] = incl;
  __syncthreads();
  const int w = scratch[lane];
  int before = w;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += y;
  }
  total = __shfl_sync(0xffffffffu, before, 31);
  const int base = __shfl_sync(0xffffffffu, before - w, warp);
  return base + incl - x;
}

// Exclusive sums of need[0, m), in place; returns their total.
__device__ __forceinline__ int64_t exclusive(int* need, int m, int* scratch) {
  int64_t base = 0;
  for (int i0 = 0; i0 < m; i0 += kThreads) {
    const int i = i0 + threadIdx.x;
    int total;
    const int x = i < m ? need[i] : 0;
    const int at = block_scan(x, scratch, total);
    if (i < m) need[i] = static_cast<int>(base) + at;
    base += total;
  }
  __syncthreads();
  return base;
}

// The largest i in [0, m) with at[i] <= k (at ascending, at[0] <= k).
__device__ __forceinline__ int owner(const int* at, int m, int k) {
  int lo = 0, hi = m;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (at[mid] <= k) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Calls take(k, page) for the k-th lowest free page, k < want; returns how many there were.
template <class F>
__device__ __forceinline__ int find_free(const Pool& p, int want, int* scratch, F take) {
  int found = 0;
  const bool wide = (reinterpret_cast<uintptr_t>(p.refs) & 15u) == 0;
  auto look = [&](int at) {  // bit i: page at + i is free
    uint32_t free = 0;
    if (wide && at + kPer <= p.pages) {
#pragma unroll
      for (int i = 0; i < kPer / 4; ++i) {
        const int4 r = *reinterpret_cast<const int4*>(p.refs + at + 4 * i);
        free |= ((r.x <= 0 ? 1u : 0u) | (r.y <= 0 ? 2u : 0u) | (r.z <= 0 ? 4u : 0u) | (r.w <= 0 ? 8u : 0u)) << (4 * i);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (at + i < p.pages && p.refs[at + i] <= 0) free |= 1u << i;
    }
    return free;
  };
  for (int64_t p0 = 0; found < want && p0 < p.pages; p0 += kThreads * kPer) {
    const int64_t at = p0 + threadIdx.x * kPer;
    uint32_t free = at < p.pages ? look(static_cast<int>(at)) : 0;
    int total;
    int k = found + block_scan(__popc(free), scratch, total);  // its barriers: all have looked before any takes
    for (; free && k < want; free &= free - 1, ++k) take(k, static_cast<int>(at) + __ffs(free) - 1);
    found += total;
  }
  __syncthreads();
  return found < want ? found : want;
}

// ---------------------------------------------------------------- grow
struct GrowParams {
  Pool pool;
  const int* table_rows;  // row of each sequence, or null: sequence i is row i
  const int* qsl;         // [m + 1]
  int m, n;
  int64_t* positions;
  int64_t* slots;
};

// Calls of up to this many tokens need one launch. A block of 1024 threads takes about a microsecond for each 1024
// of them: 20000 tokens of 250 sequences took 31 us in one block.
constexpr int kFewTokens = 1024;

// Position and slot of token t, from those of its sequence's first token (at: the sequences' first tokens).
__device__ __forceinline__ void grow_token(const GrowParams& p, const int* at, int t) {
  const Pool& pool = p.pool;
  const int i = p.m > 0 && t >= at[0] ? owner(at, p.m, t) : -1;
  const int first = i < 0 ? 0 : at[i];
  if (i >= 0 && t < min(max(p.qsl[i + 1], first), p.n)) {
    if (t == first) return;  // written already
    if (p.slots[first] >= 0) {
      const int64_t pos = p.positions[first] + (t - first);
      const int r = p.table_rows ? p.table_rows[i] : i;
      // (a row that grew: its table has an entry for each of its tokens)
      if (r >= 0 && r < pool.rows && pos < pool.capacity()) {
        const int x = static_cast<int>(pos);
        p.positions[t] = pos;
        p.slots[t] = static_cast<int64_t>(*pool.entry(r, x / pool.bs)) * pool.bs + x % pool.bs;
        return;
      }
    }
  }
  p.positions[t] = 0, p.slots[t] = -1;
}

__global__ void __launch_bounds__(kThreads) grow_pages_kernel(const GrowParams p) {
  extern __shared__ int dyn[];
  __shared__ int scratch[32];
  const Pool& pool = p.pool;
  const int m = p.m, tid = threadIdx.x;
  int* at = dyn;           // pages needed, then taken before sequence i
  int* old = dyn + m;      // tokens held before the call; -1: the sequence is left alone
  int* row = dyn + 2 * m;
  wait_for_producer();
  auto tokens = [&](int i, int& first, int& last) {
    first = min(max(p.qsl[i], 0), p.n), last = min(max(p.qsl[i + 1], first), p.n);
  };
  int bad = 0;
  for (int i = tid; i < m; i += kThreads) {
    int r = p.table_rows ? p.table_rows[i] : i;
    if (r >= pool.rows) bad |= FOLD_DEVERR_ROW, r = -1;
    row[i] = r;
    old[i] = r >= 0 ? pool.lens[r] : -1;
  }
  if (p.table_rows) {
    // a row named twice grows for the first: each leaves a mark below every length, the lowest stays
    __syncthreads();
    for (int i = tid; i < m; i += kThreads)
      if (row[i] >= 0) atomicMin(pool.lens + row[i], i - m);
    __syncthreads();
    for (int i = tid; i < m; i += kThreads)
      if (row[i] >= 0 && *static_cast<volatile int*>(pool.lens + row[i]) != i - m) bad |= FOLD_DEVERR_ROW, row[i] = -1;
    __syncthreads();
  }
  for (int i = tid; i < m; i += kThreads) {
    int need = 0;
    const int r = row[i];
    if (r >= 0) {
      const int held = max(old[i], 0);
      int first, last;
      tokens(i, first, last);
      const int add = last - first;
      bool ok = true;
      if (old[i] < 0 || held > pool.capacity() || add > pool.capacity() - held) bad |= FOLD_DEVERR_CAPACITY, ok = false;
      else if (add > 0 && held % pool.bs) {
        const int page = *pool.entry(r, held / pool.bs);
        if (page < 0 || page >= pool.pages) bad |= FOLD_DEVERR_BLOCK_TABLE, ok = false;
        else if (pool.refs[page] > 1) bad |= FOLD_DEVERR_SHARED, ok = false;
      }
      if (p.table_rows) pool.lens[r] = old[i];  // the mark goes
      if (ok) need = pool.pages_of(held + add) - pool.pages_of(held);
      else row[i] = -1;
    }
    at[i] = need;
  }
  __syncthreads();
  const int64_t want64 = exclusive(at, m, scratch);
  const int want = static_cast<int>(want64 < pool.pages ? want64 : pool.pages);
  const int got = find_free(pool, want, scratch, [&](int k, int page) {
    const int i = owner(at, m, k), held = old[i];
    *pool.entry(row[i], pool.pages_of(held) + k - at[i]) = page;
    pool.refs[page] = 1;
  });
  // sequences are served in their order while the pages last
  for (int i = tid; i < m; i += kThreads) {
    if (row[i] < 0) continue;
    int first, last;
    tokens(i, first, last);
    const int held = old[i], grown = held + last - first;
    const int need = pool.pages_of(grown) - pool.pages_of(held);
    if (need && at[i] + static_cast<int64_t>(need) > got) {
      bad |= FOLD_DEVERR_PAGES;
      for (int k = at[i]; k < got; ++k) pool.refs[*pool.entry(row[i], pool.pages_of(held) + k - at[i])] = 0;
      row[i] = -1;
    } else {
      pool.lens[row[i]] = grown;
    }
  }
  if (bad) set_error(pool.err, bad);
  __syncthreads();
  // position and slot of each sequence's first token; the others from those (grow_tokens)
  for (int i = tid; i < m; i += kThreads) {
    int first, last;
    tokens(i, first, last);
    if (first == last) continue;
    const int x = old[i];
    p.positions[first] = row[i] < 0 ? 0 : x;
    p.slots[first] = row[i] < 0 ? -1 : static_cast<int64_t>(*pool.entry(row[i], x / pool.bs)) * pool.bs + x % pool.bs;
  }
  if (p.n > kFewTokens) return;
  __syncthreads();
  for (int i = tid; i < m; i += kThreads) at[i] = min(max(p.qsl[i], 0), p.n);
  __syncthreads();
  for (int t = tid; t < p.n; t += kThreads) grow_token(p, at, t);
}

// The tokens of a large call, 256 a block.
__global__ void __launch_bounds__(256) grow_tokens_kernel(const GrowParams p) {
  extern __shared__ int dyn[];
  wait_for_producer();
  for (int i = threadIdx.x; i < p.m; i += 256) dyn[i] = min(max(p.qsl[i], 0), p.n);
  __syncthreads();
  const int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (t < p.n) grow_token(p, dyn, static_cast<int>(t));
}

// ---------------------------------------------------------------- free
// A warp a row: the length goes down to `keep` in one step, and the pages between belong to whoever
// took it down, so a row named twice gives each page back once.
__global__ void __launch_bounds__(256) free_pages_kernel(const Pool pool, const int* rows, const int* keep, int m) {
  const int i = (blockIdx.x * 256 + threadIdx.x) >> 5, lane = threadIdx.x & 31;
  wait_for_producer();
  if (i >= m) return;
  const int r = rows ? rows[i] : i;
  if (r < 0) return;
  if (r >= pool.rows) {
    if (lane == 0) set_error(pool.err, FOLD_DEVERR_ROW);
    return;
  }
  const int k = keep ? max(keep[i], 0) : 0;
  int was = 0;
  if (lane == 0) was = atomicMin(pool.lens + r, k);
  was = __shfl_sync(0xffffffffu, was, 0);
  int bad = 0;
  if (was > pool.capacity()) bad |= FOLD_DEVERR_CAPACITY, was = pool.capacity();
  const int end = pool.pages_of(max(was, 0));
  for (int j = pool.pages_of(min(k, pool.capacity())) + lane; j < end; j += 32) {
    const int page = *pool.entry(r, j);
    if (page < 0 || page >= pool.pages) bad |= FOLD_DEVERR_BLOCK_TABLE;
    else if (atomicSub(pool.refs + page, 1) <= 0) atomicAdd(pool.refs + page, 1), bad |= FOLD_DEVERR_REFS;
  }
  if (bad) set_error(pool.err, bad);
}

// ---------------------------------------------------------------- fork
struct ForkParams {
  Pool pool;
  const int* src;
  const int* dst;
  int m;
  int4* plan;  // [m]: page to copy from, to, tokens of it, tokens of the row; -1 tokens of the row: left alone
};

__global__ void __launch_bounds__(kThreads) fork_plan_kernel(const ForkParams p) {
  extern __shared__ int dyn[];
  __shared__ int scratch[32];
  const Pool& pool = p.pool;
  const int m = p.m, tid = threadIdx.x;
  int* at = dyn;
  int* len = dyn + m;  // of the parent; -1: the pair is left alone
  wait_for_producer();
  int bad = 0;
  for (int i = tid; i < m; i += kThreads) {
    const int s = p.src[i], d = p.dst[i];
    int n = -1;
    if (s >= 0 && d >= 0) {
      if (s >= pool.rows || d >= pool.rows || pool.lens[d] != 0) bad |= FOLD_DEVERR_ROW;
      else {
        n = pool.lens[s];
        if (n < 0 || n > pool.capacity()) bad |= FOLD_DEVERR_CAPACITY, n = -1;
      }
    }
    len[i] = n;
  }
  __syncthreads();
  // of children of one row the first stays (marks below every length, as in grow_pages_kernel)
  for (int i = tid; i < m; i += kThreads)
    if (len[i] >= 0) atomicMin(pool.lens + p.dst[i], i - m);
  __syncthreads();
  for (int i = tid; i < m; i += kThreads) {
    int need = 0;
    if (len[i] >= 0 && *static_cast<volatile int*>(pool.lens + p.dst[i]) != i - m) bad |= FOLD_DEVERR_ROW, len[i] = -2;
    else if (len[i] > 0 && len[i] % pool.bs) {
      const int page = *pool.entry(p.src[i], len[i] / pool.bs);
      if (page < 0 || page >= pool.pages) bad |= FOLD_DEVERR_BLOCK_TABLE, len[i] = 0;
      else need = 1;
    }
    at[i] = need;
  }
  __syncthreads();
  exclusive(at, m, scratch);
  const int want = m > 0 ? at[m - 1] + (len[m - 1] > 0 && len[m - 1] % pool.bs ? 1 : 0) : 0;
  const int got = find_free(pool, want, scratch, [&](int k, int page) {
    const int i = owner(at, m, k);  // the last of those with at[i] == k is the one that needs it
    const int x = len[i] / pool.bs;
    p.plan[i] = make_int4(*pool.entry(p.src[i], x), page, len[i] % pool.bs, len[i]);
    pool.refs[page] = 1;
  });
  for (int i = tid; i < m; i += kThreads) {
    if (len[i] < 0) {
      p.plan[i] = make_int4(0, 0, 0, -1);
      continue;
    }
    const bool part = len[i] % pool.bs != 0;
    int n = len[i];
    if (part && at[i] >= got) bad |= FOLD_DEVERR_PAGES, n = 0;
    if (!part || n == 0) p.plan[i] = make_int4(0, 0, 0, n);
    pool.lens[p.dst[i]] = n;
  }
  if (bad) set_error(pool.err, bad);
}

constexpr int kLayers = 192;  // caches a launch: their addresses are kernel arguments
struct CopyParams {
  ForkParams f;
  void* cache[kLayers];
  int layers, heads;
  int64_t block, head, slot;  // strides in bytes
  int width;                  // bytes of a slot's row
  int tables;                 // the first launch also writes the tables
};

// Blocks x < m: the table of child x. The others: one head of one layer's page, V bytes at a time.
template <class V>
__global__ void __launch_bounds__(128) fork_copy_kernel(const __grid_constant__ CopyParams p) {
  const Pool& pool = p.f.pool;
  int64_t x = blockIdx.x;
  wait_for_producer();
  if (p.tables) {
    if (x < p.f.m) {
      const int i = static_cast<int>(x);
      const int4 plan = p.f.plan[i];
      if (plan.w < 0) return;
      const int full = plan.w / pool.bs, s = p.f.src[i], d = p.f.dst[i];
      int bad = 0;
      for (int j = threadIdx.x; j < full; j += 128) {
        const int page = *pool.entry(s, j);
        bad |= page < 0 || page >= pool.pages;
      }
      if (__syncthreads_or(bad)) {  // the child stays empty, and gives back the page it took
        if (threadIdx.x == 0) {
          pool.lens[d] = 0;
          if (plan.z > 0) atomicSub(pool.refs + plan.y, 1);
          set_error(pool.err, FOLD_DEVERR_BLOCK_TABLE);
        }
        return;
      }
      for (int j = threadIdx.x; j < full; j += 128) {
        const int page = *pool.entry(s, j);
        *pool.entry(d, j) = page;
        atomicAdd(pool.refs + page, 1);
      }
      if (threadIdx.x == 0 && plan.z > 0) *pool.entry(d, full) = plan.y;
      return;
    }
    x -= p.f.m;
  }
  const int head = static_cast<int>(x % p.heads), rest = static_cast<int>(x / p.heads);
  const int layer = rest % p.layers, i = rest / p.layers;
  const int4 plan = p.f.plan[i];
  if (plan.z <= 0) return;
  char* base = static_cast<char*>(p.cache[layer]) + head * p.head;
  const char* from = base + plan.x * p.block;
  char* to = base + plan.y * p.block;
  const int per = p.width / static_cast<int>(sizeof(V)), total = plan.z * per;
  if (p.slot == p.width) {  // the tokens' rows follow one another
#pragma unroll 4
    for (int e = threadIdx.x; e < total; e += 128)
      reinterpret_cast<V*>(to)[e] = reinterpret_cast<const V*>(from)[e];
  } else {
#pragma unroll 4
    for (int e = threadIdx.x; e < total; e += 128) {
      const int t = e / per, c = e - t * per;
      reinterpret_cast<V*>(to + t * p.slot)[c] = reinterpret_cast<const V*>(from + t * p.slot)[c];
    }
  }
}

int check_pool(const std::string& what, int* refs, int pages, int* tables, int64_t stride, int width, int* lens, int rows,
               int bs, int m, int* err, Pool* out) {
  if (pages < 1 || width < 0 || rows < 0 || bs < 1 || m < 0 || (rows > 1 && stride < width))
    return fail(FOLD_ERR_INVALID_ARGUMENT, what + ": bad sizes");
  if (m > kMaxSeqs) return fail(FOLD_ERR_UNSUPPORTED, what + ": at most 16384 sequences a call");
  if (m && (!refs || (width && rows && !tables) || (rows && !lens))) return fail(FOLD_ERR_INVALID_ARGUMENT, what + ": null pointer");
  *out = Pool{refs, pages, tables, stride, width, lens, rows, bs, err};
  return FOLD_OK;
}

template <class V>
int launch_copy(const CopyParams& p, cudaStream_t stream) {
  const int64_t blocks = (p.tables ? p.f.m : 0) + static_cast<int64_t>(p.f.m) * p.layers * p.heads;
  if (blocks > 0x7fffffff) return fail(FOLD_ERR_INVALID_ARGUMENT, "fork pages: too many heads and layers");
  return launch_behind(fork_copy_kernel<V>, dim3(static_cast<unsigned>(blocks)), 128, 0, stream, "fork_copy_kernel", p);
}

}  // namespace
}  // namespace fold

extern "C" {

int fold_grow_pages(int* refs, int num_pages, int* block_tables, int64_t block_tables_stride, int block_tables_len,
                    int* lens, int num_rows, const int* rows, const int* qsl, int m, int n, int block_size,
                    void* positions, void* slots, int* err, void* stream) {
  using namespace fold;
  GrowParams p{};
  if (int s = check_pool("grow pages", refs, num_pages, block_tables, block_tables_stride, block_tables_len, lens, num_rows,
                         block_size, m, err, &p.pool))
    return s;
  if (n < 0 || static_cast<int64_t>(m) * block_tables_len > 0x7fffffff)  // pages are counted in 32 bits
    return fail(FOLD_ERR_INVALID_ARGUMENT, "grow pages: bad sizes");
  if (!rows && m > num_rows) return fail(FOLD_ERR_INVALID_ARGUMENT, "grow pages: more sequences than rows");
  if (n == 0) return FOLD_OK;
  if (!qsl || !positions || !slots) return fail(FOLD_ERR_INVALID_ARGUMENT, "grow pages: null pointer");
  p.table_rows = rows, p.qsl = qsl, p.m = m, p.n = n, p.positions = static_cast<int64_t*>(positions), p.slots = static_cast<int64_t*>(slots);
  static std::atomic<uint64_t> configured{0};
  const int smem = 12 * (m > 0 ? m : 1);
  if (smem > 46 * 1024)
    if (int s = allow_smem(grow_pages_kernel, 12 * kMaxSeqs, configured, "cudaFuncSetAttribute(grow_pages)")) return s;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (int s = launch_behind(grow_pages_kernel, dim3(1), kThreads, smem, st, "grow_pages_kernel", p)) return s;
  if (n <= kFewTokens) return FOLD_OK;
  static std::atomic<uint64_t> configured_tokens{0};
  if (4 * m > 46 * 1024)
    if (int s = allow_smem(grow_tokens_kernel, 4 * kMaxSeqs, configured_tokens, "cudaFuncSetAttribute(grow_tokens)")) return s;
  return launch_behind(grow_tokens_kernel, dim3((n + 255) / 256), 256, 4 * m, st, "grow_tokens_kernel", p);
}

int fold_free_pages(int* refs, int num_pages, int* block_tables, int64_t block_tables_stride, int block_tables_len, int* lens,
                    int num_rows, const int* rows, const int* keep, int m, int block_size, int* err, void* stream) {
  using namespace fold;
  Pool pool{};
  if (int s = check_pool("free pages", refs, num_pages, block_tables, block_tables_stride, block_tables_len, lens, num_rows,
                         block_size, m, err, &pool))
    return s;
  if (!rows && m > num_rows) return fail(FOLD_ERR_INVALID_ARGUMENT, "free pages: more sequences than rows");
  if (m == 0) return FOLD_OK;
  return launch_behind(free_pages_kernel, dim3((m + 7) / 8), 256, 0, static_cast<cudaStream_t>(stream), "free_pages_kernel",
                       pool, rows, keep, m);
}

int64_t fold_fork_pages_workspace(int m) { return m < 0 || m > fold::kMaxSeqs ? -1 : 16 * (static_cast<int64_t>(m) + 1); }

int fold_fork_pages(int* refs, int num_pages, int* block_tables, int64_t block_tables_stride, int block_tables_len, int* lens,
                    int num_rows, const int* src, const int* dst, int m, const int64_t* caches, int num_caches, int heads,
                    int block_size, int row_bytes, int64_t cache_stride_block, int64_t cache_stride_head,
                    int64_t cache_stride_slot, void* workspace, int64_t workspace_bytes, int* err, void* stream) {
  using namespace fold;
  CopyParams p{};
  if (int s = check_pool("fork pages", refs, num_pages, block_tables, block_tables_stride, block_tables_len, lens, num_rows,
                         block_size, m, err, &p.f.pool))
    return s;
  if (num_caches < 0 || heads < 1 || row_bytes < 1 || cache_stride_block < 0 || cache_stride_head < 0 || cache_stride_slot < 0)
    return fail(FOLD_ERR_INVALID_ARGUMENT, "fork pages: bad sizes");
  if ((num_pages > 1 && cache_stride_block < row_bytes) || (heads > 1 && cache_stride_head < row_bytes) ||
      (block_size > 1 && cache_stride_slot < row_bytes))
    return fail(FOLD_ERR_INVALID_ARGUMENT, "fork pages: the slots of a cache must not share memory");
  if (m == 0) return FOLD_OK;
  if (!src || !dst || (num_caches && !caches)) return fail(FOLD_ERR_INVALID_ARGUMENT, "fork pages: null pointer");
  if (!workspace || workspace_bytes < fold_fork_pages_workspace(m))
    return fail(FOLD_ERR_INVALID_ARGUMENT, "fork pages: the workspace holds fold_fork_pages_workspace bytes");
  if (!aligned16(workspace)) return fail(FOLD_ERR_ALIGNMENT, "fork pages: the workspace must be 16-byte aligned");
  p.f.src = src, p.f.dst = dst, p.f.m = m, p.f.plan = static_cast<int4*>(workspace);
  uint64_t unit = static_cast<uint64_t>(row_bytes) | cache_stride_block | cache_stride_head | cache_stride_slot;
  for (int i = 0; i < num_caches; ++i) {
    if (!caches[i]) return fail(FOLD_ERR_INVALID_ARGUMENT, "fork pages: null pointer");
    unit |= static_cast<uint64_t>(caches[i]);
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  static std::atomic<uint64_t> configured{0};
  if (8 * m > 46 * 1024)
    if (int s = allow_smem(fork_plan_kernel, 8 * kMaxSeqs, configured, "cudaFuncSetAttribute(fork_plan)")) return s;
  if (int s = launch_behind(fork_plan_kernel, dim3(1), kThreads, 8 * m, st, "fork_plan_kernel", p.f)) return s;
  p.heads = heads, p.block = cache_stride_block, p.head = cache_stride_head, p.slot = cache_stride_slot, p.width = row_bytes;
  int done = 0;
  do {
    p.layers = num_caches - done < kLayers ? num_caches - done : kLayers;
    for (int i = 0; i < p.layers; ++i) p.cache[i] = reinterpret_cast<void*>(caches[done + i]);
    p.tables = done == 0;
    int s;
    if (unit % 16 == 0) s = launch_copy<uint4>(p, st);
    else if (unit % 4 == 0) s = launch_copy<uint32_t>(p, st);
    else if (unit % 2 == 0) s = launch_copy<uint16_t>(p, st);
    else s = launch_copy<uint8_t>(p, st);
    if (s) return s;
    done += p.layers;
  } while (done < num_caches);
  return FOLD_OK;
}

}  // extern "C"
