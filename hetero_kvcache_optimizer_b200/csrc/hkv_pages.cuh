// Pages of a paged INT4 store as things that sequences own, share and give up.
// Included by hetero_kv.cu.
//
// State (all on the device): page_table [U][max_pages] (U = B H units, unit
// b H + h), lengths [B], and refs [num_pages], how many table entries name each
// page; a page with refs == 0 is free. Every operation gives the same ids for
// the same state: new pages are the lowest free ids, handed out in table order.
//
// A few launches each (with programmatic dependent launch): map (parallel over
// the table: what changes, reference counts, which entries want a page), give
// (ranks the wants and the free pages against each other), apply (the new table,
// and the page bytes, copied by every SM).
// Bound: HBM for the copies, launch latency for a few pages. A copy item is 16 KB,
// kPgUnroll 16-byte loads a thread before their stores; measured for 16,128 pages
// of 40 KB (1.32 GB moved): 220 us = 6.0 TB/s, 210 of them copying, with up to 64
// CTAs queued per SM (245 us with 8 per SM that loop: their ends do not line up),
// the same with 8 loads a thread. 4 samples of a short prompt: 7.8 us, 64 of eight
// long ones (12.6 MB copied): 12.9 us, both launch latency.
#pragma once
#include "hkv_common.cuh"

namespace hkv {

constexpr int kPgThreads = 256;    // map and apply
constexpr int kPgGive = 1024;      // give: one CTA
constexpr int kPgUnroll = 4;
constexpr int kPgChunk = kPgThreads * kPgUnroll * 16;  // bytes of a copy item

struct PagesParams {
  uint8_t* pool;
  const uint8_t* src_pool;   // apply: where the copied pages come from (the pool itself when forking)
  int64_t stride, src_stride;  // bytes between pages
  int32_t* table;            // [U][max_pages]
  int32_t* lengths;          // [B]
  int32_t* refs;             // [num_pages]
  const int32_t* parents;    // fork: [B]
  const int32_t* src_table;  // compact: the source's table, row length src_max_pages
  const int32_t* src_lengths;
  int B, H, max_pages, src_max_pages, num_pages, src_num_pages, page_tokens;
  int block_bytes;           // of 128 tokens
  int extra;                 // reserve: tokens of room beyond the lengths
  const int32_t* extra_of;   // reserve: [B] tokens of room, or NULL
  // workspace
  int32_t* new_table;        // [U][max_pages]
  int32_t* new_lengths;      // [B]
  int32_t* want;             // [wants] table entry that wants a page, or -1, in table order
                             // (compact: [U][src_max_pages] new id of a page at its first entry)
  int32_t* from;             // [wants] page copied into it, or -1
  int32_t* vecs;             // [wants] 16-byte vectors to copy
  int32_t* list;             // [copies][3]: source page, destination page, vectors
  int32_t* count;            // [1]: entries of list
  int32_t* first;            // compact: [src_num_pages] first entry naming the page and whether any is in use (pg_see)
  int wants;                 // length of want
};

__device__ __forceinline__ bool pg_ok(int page, int num_pages) { return page >= 0 && page < num_pages; }

// Sum of v over the CTA's threads before this one, and over all of them.
__device__ __forceinline__ int pg_scan(int v, int& total, int* s_warp) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  int incl = v;
#pragma unroll
  for (int k = 1; k < 32; k <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, incl, k);
    if (lane >= k) incl += o;
  }
  __syncthreads();  // s_warp's readers of the last call are through
  if (lane == 31) s_warp[w] = incl;
  __syncthreads();
  const int x = lane < nw ? s_warp[lane] : 0;
  int sum = x;
#pragma unroll
  for (int k = 1; k < 32; k <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, sum, k);
    if (lane >= k) sum += o;
  }
  total = __shfl_sync(0xffffffffu, sum, 31);
  return __shfl_sync(0xffffffffu, sum - x, w) + incl - v;
}

// ---------------------------------------------------------------- values from the host
// They travel as kernel parameters: a copy from pageable memory would wait for the
// stream, and could not be captured. Launch bound, 2.5 us.
constexpr int kPgPut = 960;
struct PutParams {
  int32_t* dst;
  int n;
  int32_t v[kPgPut];
};
__global__ void __launch_bounds__(kPgThreads) put_i32_kernel(const __grid_constant__ PutParams p) {
  for (int i = threadIdx.x; i < p.n; i += kPgThreads) p.dst[i] = p.v[i];
}

// ---------------------------------------------------------------- fork
// Sequence b becomes sequence parents[b] as it was (all at once). The lowest b
// with a given parent keeps the parent's row; the others share its full pages
// and want a page of their own for a partly filled last one.
__global__ void __launch_bounds__(kPgThreads) pages_fork_map_kernel(const __grid_constant__ PagesParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int b = blockIdx.x;
  __shared__ int s_twin;
  if (threadIdx.x == 0) s_twin = 0;
  int a = p.parents[b];
  if (a < -1 || a >= p.B) {
    if (threadIdx.x == 0 && blockIdx.y == 0) hkv_flag_error(HKV_DEVERR_BAD_PAGE);
    a = -1;
  }
  __syncthreads();
  if (a >= 0)
    for (int o = threadIdx.x; o < b; o += kPgThreads)
      if (p.parents[o] == a) s_twin = 1;
  __syncthreads();
  const bool keeps = a >= 0 && !s_twin;
  const int len = a >= 0 ? max(0, p.lengths[a]) : 0;
  const int full = len / p.page_tokens, rest = len - full * p.page_tokens;
  if (threadIdx.x == 0 && blockIdx.y == 0) p.new_lengths[b] = len;
  const int per = p.H * p.max_pages;
  for (int e = blockIdx.y * kPgThreads + threadIdx.x; e < per; e += gridDim.y * kPgThreads) {
    const int h = e / p.max_pages, i = e - h * p.max_pages;
    const int64_t at = (int64_t)b * per + e;
    const int old = p.table[at];
    int page = a >= 0 ? p.table[(int64_t)a * per + e] : -1;
    if (!pg_ok(page, p.num_pages)) {
      if (page >= 0 || (i < full && a >= 0)) hkv_flag_error(HKV_DEVERR_BAD_PAGE);
      page = -1;
    }
    if (i == full || (i == 0 && full >= p.max_pages)) {  // one thread of the unit says what it wants
      const int u = b * p.H + h;
      const bool copy = a >= 0 && !keeps && rest > 0 && i == full && page >= 0;
      p.want[u] = copy ? (int)at : -1;
      p.from[u] = page;
      p.vecs[u] = copy ? (rest + HKV_BLOCK_TOKENS - 1) / HKV_BLOCK_TOKENS * (p.block_bytes >> 4) : 0;
    }
    if (!keeps && i >= full) page = -1;
    p.new_table[at] = page;
    if (old != page) {
      if (pg_ok(old, p.num_pages)) atomicSub(p.refs + old, 1);
      if (page >= 0) atomicAdd(p.refs + page, 1);
    }
  }
}

// ---------------------------------------------------------------- reserve
// Entries len / P .. (len + extra - 1) / P of each unit that hold no page want one.
__global__ void __launch_bounds__(kPgThreads) pages_reserve_map_kernel(const __grid_constant__ PagesParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int per = p.wants / (p.B * p.H);
  for (int64_t k = (int64_t)blockIdx.x * kPgThreads + threadIdx.x; k < p.wants; k += (int64_t)gridDim.x * kPgThreads) {
    const int u = (int)(k / per), j = (int)(k - (int64_t)u * per), b = u / p.H;
    const int len = max(0, p.lengths[b]);
    const int64_t extra = min((int64_t)p.extra, max((int64_t)0, p.extra_of ? (int64_t)p.extra_of[b] : (int64_t)p.extra));
    const int i = len / p.page_tokens + j;
    const int64_t end = ((int64_t)len + extra + p.page_tokens - 1) / p.page_tokens;  // pages held afterwards
    if (j == 0 && end > p.max_pages) hkv_flag_error(HKV_DEVERR_CAPACITY);  // the row is too short for the last ones
    const int64_t at = (int64_t)u * p.max_pages + i;
    p.want[k] = i < min(end, (int64_t)p.max_pages) && p.table[at] < 0 ? (int)at : -1;
    p.from[k] = -1;
    p.vecs[k] = 0;
  }
}

// ---------------------------------------------------------------- give
// The r-th want, in order, gets the r-th lowest free page. `table` is where the
// ids go (the new table when forking). One CTA; a round takes kPgGive wants or
// kPgGive * kPgPages pages.
constexpr int kPgPages = 8;
__global__ void __launch_bounds__(kPgGive) pages_give_kernel(const __grid_constant__ PagesParams p, int32_t* table) {
  __shared__ int s_warp[32];
  griddep_wait();
  griddep_launch_dependents();
  int n = 0;  // wants so far
  for (int k0 = 0; k0 < p.wants; k0 += kPgGive) {
    const int k = k0 + threadIdx.x;
    const int e = k < p.wants ? p.want[k] : -1;
    int total;
    const int r = n + pg_scan(e >= 0, total, s_warp);
    if (e >= 0) p.list[3 * r] = p.from[k], p.list[3 * r + 1] = e, p.list[3 * r + 2] = p.vecs[k];
    n += total;
  }
  __syncthreads();
  int given = 0;
  for (int p0 = 0; p0 < p.num_pages && given < n; p0 += kPgPages * kPgGive) {
    const int g0 = p0 + kPgPages * threadIdx.x;
    unsigned mask = 0;  // which of the thread's pages are free
#pragma unroll
    for (int j = 0; j < kPgPages; ++j)
      if (g0 + j < p.num_pages && p.refs[g0 + j] <= 0) mask |= 1u << j;
    int total;
    int r = given + pg_scan(__popc(mask), total, s_warp);
#pragma unroll
    for (int j = 0; j < kPgPages; ++j)
      if (mask >> j & 1) {
        if (r < n) {
          table[p.list[3 * r + 1]] = g0 + j;
          p.list[3 * r + 1] = g0 + j;
          p.refs[g0 + j] = 1;
        }
        ++r;
      }
    given += total;
  }
  if (threadIdx.x == 0) {
    p.count[0] = min(n, given);
    if (given < n) hkv_flag_error(HKV_DEVERR_CAPACITY);  // the entries left over stay without a page
  }
}

// Copies items of the list (source page, destination page, 16-byte vectors).
__device__ __forceinline__ void pg_copy(const PagesParams& p, int item0, int step) {
  const int n = p.count[0];
  const int per = (int)((p.src_stride + kPgChunk - 1) / kPgChunk);  // chunks of a page
  const int64_t items = (int64_t)n * per;
  for (int64_t it = item0; it < items; it += step) {
    const int k = (int)(it / per);
    const int c = (int)(it - (int64_t)k * per) * (kPgChunk / 16);
    const int vecs = p.list[3 * k + 2];
    if (c >= vecs) continue;
    const uint4* s = reinterpret_cast<const uint4*>(p.src_pool + (int64_t)p.list[3 * k] * p.src_stride);
    uint4* d = reinterpret_cast<uint4*>(p.pool + (int64_t)p.list[3 * k + 1] * p.stride);
    uint4 r[kPgUnroll];
#pragma unroll
    for (int j = 0; j < kPgUnroll; ++j) {
      const int i = c + j * kPgThreads + threadIdx.x;
      if (i < vecs) r[j] = s[i];
    }
#pragma unroll
    for (int j = 0; j < kPgUnroll; ++j) {
      const int i = c + j * kPgThreads + threadIdx.x;
      if (i < vecs) d[i] = r[j];
    }
  }
}

__global__ void __launch_bounds__(kPgThreads) pages_fork_apply_kernel(const __grid_constant__ PagesParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int64_t n = (int64_t)p.B * p.H * p.max_pages;
  for (int64_t e = (int64_t)blockIdx.x * kPgThreads + threadIdx.x; e < n; e += (int64_t)gridDim.x * kPgThreads)
    p.table[e] = p.new_table[e];
  for (int b = blockIdx.x * kPgThreads + threadIdx.x; b < p.B; b += gridDim.x * kPgThreads) p.lengths[b] = p.new_lengths[b];
  pg_copy(p, blockIdx.x, gridDim.x);
}

// ---------------------------------------------------------------- compact
// The source's pages in order of their first table entry become pages 0, 1, ...
// of another pool. The ranking is spread over CTAs of kPgSpan entries (one CTA
// took 38 us of 256 for 16,128 pages): with more than one, each first publishes how
// many first entries it has, then adds up those before it.
constexpr int kPgSpan = kPgPages * kPgGive;

// What the table says of a page, in one word that entries join in any order: the
// lowest entry e that names it as kPgEntry - e (0: none; e < 2^30), and kPgUsed if any
// that names it lies within its sequence's length.
constexpr int kPgEntry = (1 << 30) - 1, kPgUsed = 1 << 30;
__device__ __forceinline__ void pg_see(int* seen, int mine) {
  for (int w = 0;;) {  // nobody yet, as a rule
    const int both = max(w & kPgEntry, mine & kPgEntry) | ((w | mine) & kPgUsed);
    if (both == w) return;
    const int old = atomicCAS(seen, w, both);
    if (old == w) return;
    w = old;
  }
}

__global__ void __launch_bounds__(kPgThreads) pages_compact_clear_kernel(const __grid_constant__ PagesParams p) {
  griddep_wait();
  griddep_launch_dependents();
  for (int i = blockIdx.x * kPgThreads + threadIdx.x; i < max(p.src_num_pages, p.num_pages); i += gridDim.x * kPgThreads) {
    if (i < p.src_num_pages) p.first[i] = 0;
    if (i < p.num_pages) p.refs[i] = 0;
  }
}

__global__ void __launch_bounds__(kPgThreads) pages_compact_map_kernel(const __grid_constant__ PagesParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int n = p.B * p.H * p.src_max_pages;
  for (int e = blockIdx.x * kPgThreads + threadIdx.x; e < n; e += gridDim.x * kPgThreads) {
    const int page = p.src_table[e];
    if (pg_ok(page, p.src_num_pages)) {
      const int u = e / p.src_max_pages, i = e - u * p.src_max_pages;
      pg_see(p.first + page, (kPgEntry - e) | ((int64_t)i * p.page_tokens < p.src_lengths[u / p.H] ? kPgUsed : 0));
    } else if (page >= 0) {
      hkv_flag_error(HKV_DEVERR_BAD_PAGE);
    }
  }
}

// Which of the thread's kPgPages entries from e1 on name a page first (and, in the
// bits from kPgPages on, which of those pages any sequence uses).
__device__ __forceinline__ unsigned pg_firsts(const PagesParams& p, int e1, int n, int (&page)[kPgPages]) {
  unsigned mask = 0;
#pragma unroll
  for (int j = 0; j < kPgPages; ++j) page[j] = e1 + j < n ? p.src_table[e1 + j] : -1;
#pragma unroll
  for (int j = 0; j < kPgPages; ++j)
    if (pg_ok(page[j], p.src_num_pages)) {
      const int w = p.first[page[j]];
      if ((w & kPgEntry) == kPgEntry - (e1 + j)) mask |= (w & kPgUsed ? (1u << kPgPages) + 1u : 1u) << j;
    }
  return mask;
}

__global__ void __launch_bounds__(kPgGive) pages_compact_count_kernel(const __grid_constant__ PagesParams p) {
  griddep_wait();
  griddep_launch_dependents();
  __shared__ int s_warp[32];
  int page[kPgPages], total;
  const unsigned mask = pg_firsts(p, blockIdx.x * kPgSpan + kPgPages * threadIdx.x, p.B * p.H * p.src_max_pages, page);
  pg_scan(__popc(mask & ((1u << kPgPages) - 1)), total, s_warp);
  if (threadIdx.x == 0) p.from[blockIdx.x] = total;
}

// list[3 r]: the page of rank r, want[e]: the rank at its first entry e. Pages behind
// the length of every sequence that names them keep their place but are not copied
// (list[3 r + 2] = 0).
__global__ void __launch_bounds__(kPgGive) pages_compact_give_kernel(const __grid_constant__ PagesParams p) {
  griddep_wait();
  griddep_launch_dependents();
  __shared__ int s_warp[32];
  const int n = p.B * p.H * p.src_max_pages, e1 = blockIdx.x * kPgSpan + kPgPages * threadIdx.x;
  int before = 0, total;
  for (int i = threadIdx.x; i < blockIdx.x; i += kPgGive) before += p.from[i];
  pg_scan(before, total, s_warp);
  before = total;
  int page[kPgPages];
  const unsigned mask = pg_firsts(p, e1, n, page);
  int r = before + pg_scan(__popc(mask & ((1u << kPgPages) - 1)), total, s_warp);
#pragma unroll
  for (int j = 0; j < kPgPages; ++j)
    if (mask >> j & 1) {
      p.want[e1 + j] = r;
      p.list[3 * r] = page[j];
      p.list[3 * r + 1] = r;
      p.list[3 * r + 2] = mask >> (kPgPages + j) & 1 ? p.page_tokens / HKV_BLOCK_TOKENS * (p.block_bytes >> 4) : 0;
      ++r;
    }
  if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) {
    const int live = before + total;
    p.count[0] = min(live, p.num_pages);
    if (live > p.num_pages) hkv_flag_error(HKV_DEVERR_CAPACITY);
  }
}

__global__ void __launch_bounds__(kPgThreads) pages_compact_apply_kernel(const __grid_constant__ PagesParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int64_t n = (int64_t)p.B * p.H * p.max_pages;
  for (int64_t e = (int64_t)blockIdx.x * kPgThreads + threadIdx.x; e < n; e += (int64_t)gridDim.x * kPgThreads) {
    const int u = (int)(e / p.max_pages), i = (int)(e - (int64_t)u * p.max_pages);
    int id = -1;
    if (i < p.src_max_pages) {
      const int page = p.src_table[(int64_t)u * p.src_max_pages + i];
      if (pg_ok(page, p.src_num_pages)) {
        id = p.want[kPgEntry - (p.first[page] & kPgEntry)];
        if (id < p.num_pages) atomicAdd(p.refs + id, 1);
        else id = -1;
      }
    }
    p.table[e] = id;
  }
  for (int b = blockIdx.x * kPgThreads + threadIdx.x; b < p.B; b += gridDim.x * kPgThreads) p.lengths[b] = p.src_lengths[b];
  pg_copy(p, blockIdx.x, gridDim.x);
}

}  // namespace hkv
