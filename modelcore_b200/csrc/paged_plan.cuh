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
// Every CTA scans the lengths itself (1,024 rows at a time, two saturating sums in one scan) and expands
// its share of the tokens and pages, a thread four (plan) or eight (release) of them with their
// searches and loads side by side: integers only, a few KB to a few MB, so launch and dependent
// latencies bound it, not bytes.  free_state_out (and seqlens_out) may be the inputs: the CTA that
// arrives last, all having read them, writes them.
#pragma once

#include "common.cuh"

namespace mcb {

constexpr int kPlanMaxThreads = 1024;

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
  int* counter;         // arrivals, zero on entry and left zero
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
  const int32_t* keep_lens;  // positions that a done request keeps, or null: none
  int* counter;
  int R, n_pages, max_pages, page_shift;
};

// Whether this CTA is the last of the grid to arrive; all threads' reads and writes before are then done
// in every CTA, and `flag` becomes whether any thread of the grid came with it set.  `counter` is zero
// again after the last.
__device__ __forceinline__ bool last_cta(int* counter, bool& flag) {
  __shared__ int s_last;  // 0: not the last, 1: the last, 3: the last and a flag
  constexpr int kFlag = 1 << 16;  // (a grid has fewer CTAs)
  const int mine = __syncthreads_or(flag) ? kFlag + 1 : 1;
  if (threadIdx.x == 0) {
    const int all = atom_add_acq_rel_gpu(counter, mine) + mine;
    s_last = (all & (kFlag - 1)) == static_cast<int>(gridDim.x) ? (all >= kFlag ? 3 : 1) : 0;
    if (s_last) *counter = 0;
  }
  __syncthreads();
  flag = (s_last & 2) != 0;
  return s_last != 0;
}

// Counts of tokens and pages stop at 2^31, above every N and n_pages: lengths may be anything, and the
// sum of a few is past 32 bits.  (The saturating sum is associative, so it can be scanned.)
constexpr uint32_t kCountEnd = 1u << 31;
__device__ __forceinline__ uint32_t count_add(uint32_t a, uint32_t b) {  // both at most kCountEnd
  const uint32_t s = a + b;
  return s < a || s > kCountEnd ? kCountEnd : s;
}
__device__ __forceinline__ uint32_t count_of(unsigned long long n) {
  return static_cast<uint32_t>(n < kCountEnd ? n : kCountEnd);
}

struct SumAdd {
  __device__ __forceinline__ unsigned long long operator()(unsigned long long a, unsigned long long b) const {
    return a + b;
  }
};
struct CountPairAdd {  // two counts in one word
  __device__ __forceinline__ unsigned long long operator()(unsigned long long a, unsigned long long b) const {
    const uint32_t lo = count_add(static_cast<uint32_t>(a), static_cast<uint32_t>(b));
    const uint32_t hi = count_add(static_cast<uint32_t>(a >> 32), static_cast<uint32_t>(b >> 32));
    return static_cast<unsigned long long>(hi) << 32 | lo;
  }
};

// Inclusive scan of one 64-bit value a thread over the block; `warp_sums` is 33 shared words, the
// last of them the block's total.
template <typename Add = SumAdd>
__device__ __forceinline__ unsigned long long block_scan(unsigned long long v, unsigned long long* warp_sums) {
  const Add add;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const unsigned long long o = __shfl_up_sync(0xffffffffu, v, m);
    if (lane >= m) v = add(o, v);
  }
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  if (warp == 0) {
    unsigned long long w = lane < warps ? warp_sums[lane] : 0;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const unsigned long long o = __shfl_up_sync(0xffffffffu, w, m);
      if (lane >= m) w = add(o, w);
    }
    warp_sums[lane] = w;
    if (lane == 31) warp_sums[32] = w;
  }
  __syncthreads();
  return warp > 0 ? add(warp_sums[warp - 1], v) : v;
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

// The same for U values at once, in step.
template <int U>
__device__ __forceinline__ void rows_of(const uint32_t* start, int n, const uint32_t (&x)[U], int (&row)[U]) {
#pragma unroll
  for (int u = 0; u < U; ++u) row[u] = 0;
  int step = 1;
  while (step < n) step <<= 1;
  for (step >>= 1; step > 0; step >>= 1)
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = row[u] + step;
      if (r < n && start[r] <= x[u]) row[u] = r;
    }
}

// x mod n for 0 <= x < 2 n.
__device__ __forceinline__ int wrap(long long x, int n) { return static_cast<int>(x >= n ? x - n : x); }

__device__ __forceinline__ int pages_of(long long len, int shift, int max_pages) {
  const long long n = (len + (1ll << shift) - 1) >> shift;
  return static_cast<int>(n < max_pages ? n : max_pages);
}

__global__ void __launch_bounds__(kPlanMaxThreads) page_plan_kernel(const PagePlanParams p) {
  __shared__ unsigned long long warp_sums[33];
  __shared__ uint32_t s_tok[kPlanMaxThreads + 1], s_page[kPlanMaxThreads + 1];  // (row + 1: its end)
  __shared__ int s_len[kPlanMaxThreads];
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, nthr = blockDim.x;
  const int rank = blockIdx.x, nc = gridDim.x;
  const long long head = p.free_state[0], tail = p.free_state[1];
  const long long avail = min(max(tail - head, 0ll), static_cast<long long>(p.n_pages));
  __shared__ int s_head;  // (one thread's division: the first scan's barriers publish it)
  if (tid == 0) s_head = static_cast<int>(((head % p.n_pages) + p.n_pages) % p.n_pages);
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
    const unsigned long long incl = block_scan<CountPairAdd>(mine, warp_sums);
    const unsigned long long total = warp_sums[32];
    const uint32_t row_tok1 = count_add(tok0, static_cast<uint32_t>(incl));
    if (tid == 0) {
      s_tok[0] = tok0;
      s_page[0] = page0;
    }
    s_tok[tid + 1] = row_tok1;
    s_page[tid + 1] = count_add(page0, static_cast<uint32_t>(incl >> 32));
    s_len[tid] = len;
    if (rank == 0 && r < p.R) p.cu_new[r + 1] = static_cast<int>(min(row_tok1, kCountEnd - 1));
    __syncthreads();
    const uint32_t tok1 = count_add(tok0, static_cast<uint32_t>(total));
    const uint32_t page1 = count_add(page0, static_cast<uint32_t>(total >> 32));
    // new table entries
    for (uint32_t k = page0 + rank * nthr + tid; k < page1; k += nc * nthr) {
      const int i = row_of(s_page, rows, k);
      const int j = pages_of(s_len[i], p.page_shift, p.max_pages) + static_cast<int>(k - s_page[i]);
      int page = -1;
      if (k < avail) page = p.free_pages[wrap(static_cast<long long>(s_head) + k, p.n_pages)];
      else record_error(kErrPagesExhausted);
      p.block_table[(base + i) * p.table_stride + j] = page;
    }
    // positions and slots
    constexpr int U = 4;
    const uint32_t tok_end = min(tok1, static_cast<uint32_t>(p.N)), hop = nc * nthr;
    for (uint32_t t0 = tok0 + rank * nthr + tid; t0 < tok_end; t0 += U * hop) {
      uint32_t t[U];
      int i[U], page[U];
      long long pos[U];
#pragma unroll
      for (int u = 0; u < U; ++u) t[u] = min(t0 + u * hop, tok_end - 1);
      rows_of<U>(s_tok, rows, t, i);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int row_len = s_len[i[u]];
        pos[u] = static_cast<long long>(row_len) + (t[u] - s_tok[i[u]]);
        const long long j = pos[u] >> p.page_shift;
        page[u] = -1;  // none: past the table or the queue, which the rows and the table entries report
        if (j < p.max_pages) {
          const int first = pages_of(row_len, p.page_shift, p.max_pages);
          const uint32_t k = s_page[i[u]] + static_cast<uint32_t>(j - first);
          if (j < first || k < avail) {
            page[u] = j < first ? p.block_table[(base + i[u]) * p.table_stride + j]
                                : p.free_pages[wrap(static_cast<long long>(s_head) + k, p.n_pages)];
            if (page[u] < 0) page[u] = p.n_pages;  // no page number: reported below
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (t0 + u * hop >= tok_end) break;
        const bool in = page[u] >= 0 && page[u] < p.n_pages;
        if (page[u] >= p.n_pages) record_error(kErrPageOutOfRange);
        p.positions[t[u]] = static_cast<int>(pos[u]);
        p.slot_map[t[u]] = in ? (static_cast<long long>(page[u]) << p.page_shift) +
                                    (pos[u] & ((1ll << p.page_shift) - 1))
                              : -1;
      }
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
  bool unused = false;
  if (last_cta(p.counter, unused) && tid == 0) {
    p.free_state_out[0] = head + min(static_cast<long long>(page0), avail);
    p.free_state_out[1] = tail;
  }
}

__global__ void __launch_bounds__(kPlanMaxThreads) page_release_kernel(const PageReleaseParams p) {
  __shared__ unsigned long long warp_sums[33];
  __shared__ uint32_t s_page[kPlanMaxThreads];
  __shared__ int s_first[kPlanMaxThreads];  // the row's first returned table entry
  pdl_wait();  // no early trigger: like kv_advance, this kernel may write cache_seqlens
  const int tid = threadIdx.x, nthr = blockDim.x;
  const int rank = blockIdx.x, nc = gridDim.x;
  const long long head = p.free_state[0], tail = p.free_state[1];
  const uint32_t room =
      static_cast<uint32_t>(min(max(p.n_pages - (tail - head), 0ll), static_cast<long long>(p.n_pages)));
  __shared__ int s_tail;  // (one thread's division: the first scan's barriers publish it)
  if (tid == 0) s_tail = static_cast<int>(((tail % p.n_pages) + p.n_pages) % p.n_pages);
  auto kept_len = [&](int r, int len) {  // of a done request
    return p.keep_lens == nullptr ? 0 : min(max(p.keep_lens[r], 0), max(len, 0));
  };
  // The rows from `base` on: s_page, where each one's pages start in the sequence of all returned ones;
  // returns where the block's end.
  auto rows_pages = [&](int base, uint32_t page0) -> uint32_t {
    const int r = base + tid;
    int held = 0, first = 0;
    if (r < p.R) {
      const int len = p.seqlens[r];
      if (p.done[r] != 0) {
        first = pages_of(kept_len(r, len), p.page_shift, p.max_pages);
        held = pages_of(max(len, 0), p.page_shift, p.max_pages) - first;
      }
    }
    const unsigned long long incl = block_scan(static_cast<unsigned long long>(held), warp_sums);
    s_page[tid] = count_of(page0 + incl - held);
    s_first[tid] = first;
    const uint32_t page1 = count_of(page0 + warp_sums[32]);
    __syncthreads();
    return page1;
  };
  auto no_page = [&](int page) { return static_cast<uint32_t>(page) >= static_cast<uint32_t>(p.n_pages); };
  auto store = [&](uint32_t k, int page) {  // the k-th returned page, k < room
    const uint32_t at = s_tail + k;         // below 2 n_pages
    p.free_pages[at >= static_cast<uint32_t>(p.n_pages) ? at - p.n_pages : at] = page;
  };
  uint32_t page0 = 0;
  bool holes = false;  // entries that name no page
  for (int base = 0; base < p.R; base += nthr) {
    const int rows = min(nthr, p.R - base);
    const uint32_t page1 = rows_pages(base, page0);
    // A warp takes 256 consecutive pages at a time.  Where they are one request's -- long requests --
    // one search finds it, and the entries are a copy; else every lane searches for its own.
    constexpr int U = 8;
    const int lane = tid & 31;
    const uint32_t hop = nc * (nthr >> 5) * 32 * U;
    for (uint32_t w0 = page0 + (rank * (nthr >> 5) + (tid >> 5)) * 32 * U; w0 < page1; w0 += hop) {
      const uint32_t k0 = w0 + lane;
      int page[U];
      const int row = row_of(s_page, rows, w0);
      const uint32_t row_end = row + 1 < rows ? s_page[row + 1] : page1;
      if (row_end - w0 >= 32 * U) {
        const int32_t* src = p.block_table + (base + row) * p.table_stride + s_first[row] + (k0 - s_page[row]);
#pragma unroll
        for (int u = 0; u < U; ++u) page[u] = src[32 * u];
      } else {
        uint32_t k[U];
        int i[U];
#pragma unroll
        for (int u = 0; u < U; ++u) k[u] = min(k0 + 32 * u, page1 - 1);
        rows_of<U>(s_page, rows, k, i);
#pragma unroll
        for (int u = 0; u < U; ++u)
          page[u] = p.block_table[(base + i[u]) * p.table_stride + s_first[i[u]] + (k[u] - s_page[i[u]])];
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t k = k0 + 32 * u;
        if (k >= page1) break;
        holes |= no_page(page[u]);
        if (k < room) store(k, page[u]);
      }
    }
    page0 = page1;
    __syncthreads();  // s_page is free again
  }
  if (!last_cta(p.counter, holes)) return;
  if (holes) {
    // Entries that plan left at -1 when the queue ran out, or worse: they are no pages to hand on.  Rare,
    // so this CTA writes the whole sequence again without them, over what all have written.
    if (tid == 0) record_error(kErrPageOutOfRange);
    uint32_t kept = 0;
    page0 = 0;
    for (int base = 0; base < p.R; base += nthr) {
      const int rows = min(nthr, p.R - base);
      const uint32_t page1 = rows_pages(base, page0);
      for (uint32_t k0 = page0; k0 < page1; k0 += nthr) {
        const uint32_t k = k0 + tid;
        int page = -1;
        if (k < page1) {
          const int i = row_of(s_page, rows, k);
          page = p.block_table[(base + i) * p.table_stride + s_first[i] + (k - s_page[i])];
        }
        const bool is_page = !no_page(page);
        const unsigned long long incl = block_scan(is_page ? 1ull : 0ull, warp_sums);
        if (is_page && kept + incl <= room) store(kept + static_cast<uint32_t>(incl) - 1, page);
        kept += static_cast<uint32_t>(warp_sums[32]);
        __syncthreads();  // warp_sums is free again
      }
      page0 = page1;
      __syncthreads();  // s_page is free again
    }
    page0 = kept;
  }
  for (int r = tid; r < p.R; r += nthr) {
    const int len = p.seqlens[r];
    p.seqlens_out[r] = p.done[r] != 0 ? kept_len(r, len) : len;
  }
  if (tid == 0) {
    if (page0 > room) record_error(kErrPagesExhausted);  // more pages than the pool has: a row released twice
    p.free_state_out[0] = head;
    p.free_state_out[1] = tail + min(page0, room);
  }
}

}  // namespace mcb
