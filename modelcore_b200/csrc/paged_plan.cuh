// The paged cache's bookkeeping on the GPU: block tables, slot maps and the free-page queue, from
// the requests' lengths alone (no host copy of them is needed, so a step can sit in a CUDA graph).
//
// Pages of 2^page_shift positions.  Request r holds L_r cached positions and takes n_r new tokens:
//   cu_r    = sum of n_i over i < r                      offsets of the packed batch
//   first_r = ceil(L_r / page), last_r = ceil((L_r + n_r) / page), both at most max_pages
//   a_r     = sum of (last_i - first_i) over i < r
//   table[r, j] = queue[(head + a_r + j - first_r) mod n_pages]         first_r <= j < last_r
//   pos_t   = L_r + t - cu_r, slot_t = table[r, pos_t / page] * page + pos_t % page
// The free pages are a queue of n_pages entries between two counters that only grow, head and
// tail (entry x at x mod n_pages).  A plan neither moves the lengths nor overwrites a table entry
// below first_r, so planning again from the same lengths and counters gives the same answer.
//
// One thread-block cluster does a whole call: every CTA scans the lengths itself (1,024 rows at a
// time, two sums in one 64-bit scan) and expands its share of the tokens and pages.  Integers
// only, a few KB to a few MB: launch and dependent-load latency bound it, not bytes.  A cluster,
// not a grid, because free_state_out (and seqlens_out) may be the inputs: every CTA has read them
// before the cluster barrier, and only then are they written.
#pragma once

#include "common.cuh"

namespace mcb {

constexpr int kPlanMaxThreads = 1024;
constexpr int kPlanMaxCluster = 8;

struct PagePlanParams {
  const int32_t* seqlens;
  const int32_t* new_lens;
  int32_t* block_table;
  long long table_stride;
  const int32_t* free_pages;
  const long long* free_state;
  long long* free_state_out;
  int32_t* cu_new;      // (R + 1,)
  int32_t* positions;   // (N,)
  long long* slot_map;  // (N,)
  int R, N, n_pages, max_pages, page_shift;
};

struct PageReleaseParams {
  const int32_t* done;
  const int32_t* seqlens;
  const int32_t* block_table;
  long long table_stride;
  int32_t* free_pages;
  const long long* free_state;
  long long* free_state_out;
  int32_t* seqlens_out;
  int R, n_pages, max_pages, page_shift;
};

// Inclusive scan of one 64-bit value a thread over the block; `warp_sums` is 33 shared words, the
// last of them the block's total.
__device__ __forceinline__ unsigned long long block_scan(unsigned long long v, unsigned long long* warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const unsigned long long o = __shfl_up_sync(0xffffffffu, v, m);
    if (lane >= m) v += o;
  }
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  if (warp == 0) {
    unsigned long long w = lane < warps ? warp_sums[lane] : 0;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const unsigned long long o = __shfl_up_sync(0xffffffffu, w, m);
      if (lane >= m) w += o;
    }
    warp_sums[lane] = w;
    if (lane == 31) warp_sums[32] = w;
  }
  __syncthreads();
  return warp > 0 ? v + warp_sums[warp - 1] : v;
}

// The last i in [0, n) with start[i] <= x (start[0] <= x): of rows with equal starts, the one that
// is not empty.
__device__ __forceinline__ int row_of(const uint32_t* start, int n, uint32_t x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// x mod n for 0 <= x < 2 n.
__device__ __forceinline__ int wrap(long long x, int n) { return static_cast<int>(x >= n ? x - n : x); }

__device__ __forceinline__ int pages_of(long long len, int shift, int max_pages) {
  const long long n = (len + (1ll << shift) - 1) >> shift;
  return static_cast<int>(n < max_pages ? n : max_pages);
}

__global__ void __launch_bounds__(kPlanMaxThreads) page_plan_kernel(const PagePlanParams p) {
  __shared__ unsigned long long warp_sums[33];
  __shared__ uint32_t s_tok[kPlanMaxThreads], s_page[kPlanMaxThreads];
  __shared__ int s_len[kPlanMaxThreads];
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, nthr = blockDim.x;
  const int rank = blockIdx.x, nc = gridDim.x;  // the grid is one cluster
  const long long head = p.free_state[0], tail = p.free_state[1];
  const long long avail = min(max(tail - head, 0ll), static_cast<long long>(p.n_pages));
  const int head0 = static_cast<int>(((head % p.n_pages) + p.n_pages) % p.n_pages);
  uint32_t tok0 = 0, page0 = 0;  // sums over the rows of earlier chunks
  if (rank == 0 && tid == 0) p.cu_new[0] = 0;
  for (int base = 0; base < p.R; base += nthr) {
    const int r = base + tid, rows = min(nthr, p.R - base);
    int len = 0, fresh = 0, need = 0;
    if (r < p.R) {
      len = p.seqlens[r];
      fresh = max(p.new_lens[r], 0);
      if (len < 0 || ((static_cast<long long>(len) + fresh + (1 << p.page_shift) - 1) >> p.page_shift) > p.max_pages) {
        if (rank == 0) record_error(kErrPositionBeyondCache);
        len = max(len, 0);
      }
      need = pages_of(static_cast<long long>(len) + fresh, p.page_shift, p.max_pages) -
             pages_of(len, p.page_shift, p.max_pages);
    }
    const unsigned long long mine = static_cast<unsigned long long>(need) << 32 | static_cast<uint32_t>(fresh);
    const unsigned long long incl = block_scan(mine, warp_sums);
    const unsigned long long total = warp_sums[32];
    s_tok[tid] = tok0 + static_cast<uint32_t>(incl - mine);
    s_page[tid] = page0 + static_cast<uint32_t>((incl - mine) >> 32);
    s_len[tid] = len;
    if (rank == 0 && r < p.R) p.cu_new[r + 1] = static_cast<int>(tok0 + static_cast<uint32_t>(incl));
    __syncthreads();
    const uint32_t tok1 = tok0 + static_cast<uint32_t>(total), page1 = page0 + static_cast<uint32_t>(total >> 32);
    // new table entries
    for (uint32_t k = page0 + rank * nthr + tid; k < page1; k += nc * nthr) {
      const int i = row_of(s_page, rows, k);
      const int j = pages_of(s_len[i], p.page_shift, p.max_pages) + static_cast<int>(k - s_page[i]);
      int page = -1;
      if (k < avail) page = p.free_pages[wrap(static_cast<long long>(head0) + k, p.n_pages)];
      else record_error(kErrPagesExhausted);
      p.block_table[(base + i) * p.table_stride + j] = page;
    }
    // positions and slots
    for (uint32_t t = tok0 + rank * nthr + tid; t < min(tok1, static_cast<uint32_t>(p.N)); t += nc * nthr) {
      const int i = row_of(s_tok, rows, t);
      const int row_len = s_len[i];
      const long long pos = static_cast<long long>(row_len) + (t - s_tok[i]);
      const long long j = pos >> p.page_shift;
      int page = -1;
      if (j < p.max_pages) {
        const int first = pages_of(row_len, p.page_shift, p.max_pages);
        if (j < first) {
          page = p.block_table[(base + i) * p.table_stride + j];
        } else {
          const uint32_t k = s_page[i] + static_cast<uint32_t>(j - first);
          if (k < avail) page = p.free_pages[wrap(static_cast<long long>(head0) + k, p.n_pages)];
        }
        if (page < 0 || page >= p.n_pages) {
          record_error(kErrPageOutOfRange);  // (a page the queue lacked: error 5 came first)
          page = -1;
        }
      }
      p.positions[t] = static_cast<int>(pos);
      p.slot_map[t] = page < 0 ? -1 : (static_cast<long long>(page) << p.page_shift) +
                                          (pos & ((1ll << p.page_shift) - 1));
    }
    tok0 = tok1;
    page0 = page1;
    __syncthreads();
  }
  if (tok0 > static_cast<uint32_t>(p.N) && rank == 0 && tid == 0) record_error(kErrTooManyTokens);
  for (long long t = static_cast<long long>(tok0) + rank * nthr + tid; t < p.N; t += nc * nthr) {  // padding
    p.positions[t] = -1;
    p.slot_map[t] = -1;
  }
  cluster_sync();  // every CTA has read the counters
  if (rank == 0 && tid == 0) {
    p.free_state_out[0] = head + min(static_cast<long long>(page0), avail);
    p.free_state_out[1] = tail;
  }
}

__global__ void __launch_bounds__(kPlanMaxThreads) page_release_kernel(const PageReleaseParams p) {
  __shared__ unsigned long long warp_sums[33];
  __shared__ uint32_t s_page[kPlanMaxThreads];
  pdl_wait();  // no early trigger: like kv_advance, this kernel may write cache_seqlens
  const int tid = threadIdx.x, nthr = blockDim.x;
  const int rank = blockIdx.x, nc = gridDim.x;
  const long long head = p.free_state[0], tail = p.free_state[1];
  const long long room = min(max(p.n_pages - (tail - head), 0ll), static_cast<long long>(p.n_pages));
  const int tail0 = static_cast<int>(((tail % p.n_pages) + p.n_pages) % p.n_pages);
  uint32_t page0 = 0;
  for (int base = 0; base < p.R; base += nthr) {
    const int r = base + tid, rows = min(nthr, p.R - base);
    int len = 0, held = 0;
    bool gone = false;
    if (r < p.R) {
      len = p.seqlens[r];
      gone = p.done[r] != 0;
      if (gone) held = pages_of(max(len, 0), p.page_shift, p.max_pages);
    }
    const unsigned long long incl = block_scan(static_cast<unsigned long long>(held), warp_sums);
    const uint32_t page1 = page0 + static_cast<uint32_t>(warp_sums[32]);
    s_page[tid] = page0 + static_cast<uint32_t>(incl) - held;
    __syncthreads();
    for (uint32_t k = page0 + rank * nthr + tid; k < page1; k += nc * nthr) {
      const int i = row_of(s_page, rows, k);
      const int page = p.block_table[(base + i) * p.table_stride + (k - s_page[i])];
      if (page < 0 || page >= p.n_pages) record_error(kErrPageOutOfRange);
      if (k >= room) {
        record_error(kErrPagesExhausted);  // more pages than the pool has: a row released twice
        continue;
      }
      p.free_pages[wrap(static_cast<long long>(tail0) + k, p.n_pages)] = page;
    }
    page0 = page1;
    cluster_sync();  // every CTA has read this chunk's lengths (and s_page is free again)
    if (rank == 0 && r < p.R) p.seqlens_out[r] = gone ? 0 : len;
  }
  cluster_sync();
  if (rank == 0 && tid == 0) {
    p.free_state_out[0] = head;
    p.free_state_out[1] = tail + min(static_cast<long long>(page0), room);
  }
}

}  // namespace mcb
