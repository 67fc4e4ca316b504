// Pages of the paged cache copied, shared, moved together and given back.
//
// page_fork: row r's new contents are row source_r's old ones (-1: none), all rows at once.  A page that is
// full is shared: no later token is written to it.  shares = the rows that hold a page, less one; with h_s
// heirs of an old row s it grows by h_s - 1 for each of the row's full pages, and a page whose shares fall to
// -1 is free.  The last page, where it is not full, belongs to the row alone: its first heir keeps it, each
// other one gets a fresh page, in row order, and a copy of the positions in use in every slot.
//   new pages: queue[(head + k) mod n_pages] for the k-th row that needs one
//   freed:     page x with shares_x + change_x < 0, in page order, to queue[(tail + rank) mod n_pages]
// (Counts, not an order of arrival, decide: the same call gives the same queue.)
//
// Three or four launches, each needing the whole of the one before: the plan (one CTA; the others zero the
// changes), then the tables, the changes and the copies, then, in large pools, the freed pages of every 1,024
// counted, then all placed.
// All reads of what may be written in place come before the last.  The copies are bound by HBM (a page's
// positions of one head are contiguous), all else by launches: 16 rows of 12 slots 17 us as called, a beam search's
// step of 256 rows of 12 slots (105 MB) 30 us, 16 at HBM's rate.
//
// paged_keep: the tokens path_0 < path_1 < ... of a row's new ones are kept: position L + i of every slot
// and head gets what L + path_i holds, the row is L + kept long, and the pages behind it that the step
// took are free again.  path_i >= i, so moves in the order of i never overwrite one still to be read, and a
// thread that carries 16 bytes of one head through all of a row's moves needs no other.  kept < 0: the whole step
// as it is.  8 requests of 12 slots 8.8 us as called, 128 of 24 slots (56 MB in rows of 256 bytes) 19 us, 8.6 at HBM's rate:
// four dependent loads a CTA (lengths, path, table, rows).  With the lengths in place, which the last of all CTAs writes,
// 7.0 (no outputs to allocate) and 25 us.
#pragma once

#include "paged_plan.cuh"

namespace mcb {

constexpr int kForkBlock = 1024;  // pages counted together

struct PageForkParams {
  const int32_t* source;       // (R,)
  const int32_t* seqlens;      // (R,)
  const int32_t* table;        // (R, max_pages)
  const int32_t* shares;       // (n_pages,)
  int32_t* queue;              // (n_pages,)
  const long long* state;      // (2,)
  uint16_t* k_pages;           // (slots, n_pages, Hkv, page, D)
  uint16_t* v_pages;
  int32_t* table_out;          // may be table, and so on
  int32_t* shares_out;
  int32_t* seqlens_out;
  long long* state_out;
  long long table_stride, out_stride;
  int R, n_pages, max_pages, page_shift, slots, Hkv, D;
  int table_in_place;
  // workspace
  long long* meta;             // head, head mod n, tail mod n, fresh pages wanted, room
  int32_t* heirs;              // (R,)
  int32_t* first;              // (R,)
  int32_t* new_len;            // (R,)
  int32_t* fresh;              // (R,) the fresh page of a row, -1 (none left) or -2 (none needed)
  int32_t* jobs;               // (R,) the rows that copy
  int32_t* counts;             // freed pages of every block
  int32_t* change;             // (n_pages,)
  int32_t* table_tmp;          // (R, max_pages), with table_in_place
};

__device__ __forceinline__ int fork_len(const PageForkParams& p, int s) {
  const long long cap = static_cast<long long>(p.max_pages) << p.page_shift;
  return static_cast<int>(min(static_cast<long long>(max(p.seqlens[s], 0)), cap));
}

__global__ void __launch_bounds__(1024) page_fork_plan_kernel(const PageForkParams p) {
  __shared__ unsigned long long warp_sums[33];
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x;
  if (blockIdx.x > 0) {
    for (long long i = (blockIdx.x - 1ll) * 1024 + tid; i < p.n_pages; i += (gridDim.x - 1ll) * 1024) p.change[i] = 0;
    return;
  }
  const long long head = p.state[0], tail = p.state[1];
  const long long n = p.n_pages, avail = min(max(tail - head, 0ll), n);
  const int head_at = static_cast<int>(((head % n) + n) % n);
  for (int r = tid; r < p.R; r += 1024) {
    p.heirs[r] = 0;
    p.first[r] = 0x7fffffff;
  }
  __syncthreads();
  auto source_of = [&](int r) {
    const int s = p.source[r];
    if (s >= p.R) record_error(kErrDraftOutOfRange);
    return s >= p.R ? -1 : s;
  };
  for (int r = tid; r < p.R; r += 1024) {
    const int s = source_of(r);
    if (p.seqlens[r] < 0 || p.seqlens[r] != fork_len(p, r)) record_error(kErrPositionBeyondCache);
    if (s < 0) continue;
    atomicAdd(p.heirs + s, 1);
    atomicMin(p.first + s, r);
  }
  __syncthreads();
  long long taken = 0;  // rows that want a fresh page, then those that get one
  for (int base = 0; base < p.R; base += 1024) {
    const int r = base + tid;
    bool want = false;
    int len = 0;
    if (r < p.R) {
      const int s = source_of(r);
      if (s >= 0) {
        len = fork_len(p, s);
        want = (len & ((1 << p.page_shift) - 1)) != 0 && __ldcg(p.first + s) != r;
      }
    }
    const long long k = taken + static_cast<long long>(block_scan(want ? 1ull : 0ull, warp_sums)) - 1;
    taken += static_cast<long long>(warp_sums[32]);
    if (r < p.R) {
      int page = -2;
      if (want) {
        page = k < avail ? p.queue[wrap(static_cast<long long>(head_at) + k, p.n_pages)] : -1;
        if (k >= avail) record_error(kErrPagesExhausted);
        else if (page < 0 || page >= p.n_pages) {
          record_error(kErrPageOutOfRange);
          page = -1;
        }
        p.jobs[k] = r;
      }
      p.fresh[r] = page;
      p.new_len[r] = len;
    }
    __syncthreads();  // warp_sums is free again
  }
  if (tid == 0) {
    const long long got = min(taken, avail);
    p.meta[0] = head + got;
    p.meta[1] = tail;
    p.meta[2] = taken;
    p.meta[3] = min(max(n - (tail - (head + got)), 0ll), n);  // room for freed pages
    p.meta[4] = ((tail % n) + n) % n;
  }
}

__global__ void __launch_bounds__(256) page_fork_apply_kernel(const PageForkParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, page_len = 1 << p.page_shift;
  const long long thr = static_cast<long long>(gridDim.x) * 256, me = static_cast<long long>(blockIdx.x) * 256 + tid;
  int32_t* out = p.table_in_place ? p.table_tmp : p.table_out;
  const long long out_stride = p.table_in_place ? p.max_pages : p.out_stride;
  const long long entries = static_cast<long long>(p.R) * p.max_pages;
  for (long long i = me; i < entries; i += thr) {
    const int r = static_cast<int>(i / p.max_pages), col = static_cast<int>(i % p.max_pages);
    // the row's new entry
    const int len = p.new_len[r], full = len >> p.page_shift, part = len & (page_len - 1);
    int page = -1;
    if (col < full + (part != 0)) {
      const int fresh = p.fresh[r];
      page = col == full && fresh != -2 ? fresh : p.table[p.source[r] * p.table_stride + col];
    }
    out[r * out_stride + col] = page;
    // and what its old one's page loses or gains
    const int old = fork_len(p, r), heirs = p.heirs[r];
    if (col < (old >> p.page_shift) + ((old & (page_len - 1)) != 0)) {
      const int change = col < (old >> p.page_shift) ? heirs - 1 : heirs == 0 ? -1 : 0;
      const int pg = p.table[r * p.table_stride + col];
      if (pg < 0 || pg >= p.n_pages) record_error(kErrPageOutOfRange);
      else if (change != 0) atomicAdd(p.change + pg, change);
    }
  }
  // copies: one head's positions in use of one slot's K or V at a time, a warp each
  const long long jobs = p.meta[2], per = 2ll * p.slots * p.Hkv;
  const int lane = tid & 31;
  for (long long c = me >> 5; c < jobs * per; c += thr >> 5) {
    const int r = p.jobs[c / per], x = static_cast<int>(c % per);
    const int dst = p.fresh[r], len = p.new_len[r];
    const int src = p.table[p.source[r] * p.table_stride + (len >> p.page_shift)];
    if (dst < 0 || src < 0 || src >= p.n_pages) continue;
    uint16_t* pool = x & 1 ? p.v_pages : p.k_pages;
    const int h = (x >> 1) % p.Hkv;
    const long long slot = (x >> 1) / p.Hkv;
    const long long block = static_cast<long long>(page_len) * p.D;
    const uint4* from = reinterpret_cast<const uint4*>(pool + ((slot * p.n_pages + src) * p.Hkv + h) * block);
    uint4* to = reinterpret_cast<uint4*>(pool + ((slot * p.n_pages + dst) * p.Hkv + h) * block);
    const int words = (len & (page_len - 1)) * (p.D / 8);
    constexpr int U = 8;
    for (int i0 = lane; i0 < words; i0 += 32 * U) {
      uint4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + 32 * u < words) v[u] = from[i0 + 32 * u];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + 32 * u < words) to[i0 + 32 * u] = v[u];
    }
  }
}

__device__ __forceinline__ bool fork_freed(const PageForkParams& p, long long page) {
  return page < p.n_pages && p.shares[page] + p.change[page] < 0;
}

__global__ void __launch_bounds__(kForkBlock) page_fork_count_kernel(const PageForkParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int n = __syncthreads_count(fork_freed(p, static_cast<long long>(blockIdx.x) * kForkBlock + threadIdx.x));
  if (threadIdx.x == 0) p.counts[blockIdx.x] = n;
}

// A CTA a block; with one CTA for all blocks, in turn.
__global__ void __launch_bounds__(kForkBlock) page_fork_place_kernel(const PageForkParams p) {
  __shared__ unsigned long long warp_sums[33];
  pdl_wait();  // no early trigger: this kernel may write cache_seqlens
  const int tid = threadIdx.x;
  const int blocks = (p.n_pages + kForkBlock - 1) / kForkBlock;
  const bool alone = gridDim.x == 1;
  unsigned long long before = 0;
  if (!alone) {
    for (int b = tid; b < static_cast<int>(blockIdx.x); b += kForkBlock) before += p.counts[b];
    block_scan(before, warp_sums);
    before = warp_sums[32];
    __syncthreads();
  }
  const unsigned long long room = p.meta[3];
  const long long tail_at = p.meta[4];
  for (int b = blockIdx.x; b < blocks; b += gridDim.x) {
    const long long page = static_cast<long long>(b) * kForkBlock + tid;
    const bool freed = fork_freed(p, page);
    const unsigned long long k = before + block_scan(freed ? 1ull : 0ull, warp_sums) - 1;
    before += warp_sums[32];
    if (freed && k < room) p.queue[wrap(tail_at + static_cast<long long>(k), p.n_pages)] = static_cast<int>(page);
    if (page < p.n_pages) p.shares_out[page] = max(p.shares[page] + p.change[page], 0);
    if (b == blocks - 1 && tid == 0) {
      if (before > room) record_error(kErrPagesExhausted);
      p.state_out[0] = p.meta[0];
      p.state_out[1] = p.meta[1] + static_cast<long long>(min(before, room));
    }
    __syncthreads();  // warp_sums is free again
  }
  const long long me = static_cast<long long>(blockIdx.x) * kForkBlock + tid;
  const long long thr = static_cast<long long>(gridDim.x) * kForkBlock;
  for (long long i = me; i < p.R; i += thr) p.seqlens_out[i] = p.new_len[i];
  if (p.table_in_place) {
    const long long entries = static_cast<long long>(p.R) * p.max_pages;
    for (long long i = me; i < entries; i += thr)
      p.table_out[i / p.max_pages * p.out_stride + i % p.max_pages] = p.table_tmp[i];
  }
}

struct PagedKeepParams {
  const int32_t* path;         // (R, P)
  const int32_t* kept;         // (R,)
  const int32_t* seqlens;      // (R,)
  const int32_t* new_lens;     // (R,)
  const int32_t* table;        // (R, max_pages)
  int32_t* queue;              // (n_pages,)
  const long long* state;      // (2,)
  uint16_t* k_pages;           // (slots, n_pages, Hkv, page, D)
  uint16_t* v_pages;
  long long* state_out;        // may be state
  int32_t* seqlens_out;        // may be seqlens
  int* counter;
  long long table_stride, path_stride;
  int R, P, n_pages, max_pages, page_shift, slots, Hkv, D;
  int in_place;  // seqlens_out is seqlens
};

constexpr int kKeepThreads = 256;

__device__ __forceinline__ int keep_len(const PagedKeepParams& p, int r) {
  const long long cap = static_cast<long long>(p.max_pages) << p.page_shift;
  return static_cast<int>(min(static_cast<long long>(max(p.seqlens[r], 0)), cap));
}
__device__ __forceinline__ int keep_kept(const PagedKeepParams& p, int r, int fresh) {  // (below 0: the whole step as it is)
  const int kept = p.kept[r];
  return kept < 0 ? fresh : min(kept, min(fresh, p.P));
}

// The rows' lengths, and the pages behind them to the queue; one CTA.
__device__ __noinline__ void keep_books(const PagedKeepParams& p, unsigned long long* warp_sums) {
  const int tid = threadIdx.x;
  const long long head = p.state[0], tail = p.state[1], n = p.n_pages;
  const long long room = min(max(n - (tail - head), 0ll), n);
  const int tail_at = static_cast<int>(((tail % n) + n) % n);
  long long back = 0;
  for (int b0 = 0; b0 < p.R; b0 += kKeepThreads) {
    const int row = b0 + tid;
    int c0 = 0, c1 = 0, pages = 0;
    if (row < p.R) {
      const int l = keep_len(p, row), f = max(p.new_lens[row], 0), k = keep_kept(p, row, f);
      c0 = pages_of(static_cast<long long>(l) + k, p.page_shift, p.max_pages);
      c1 = pages_of(static_cast<long long>(l) + f, p.page_shift, p.max_pages);
      for (int c = c0; c < c1; ++c) {
        const int pg = p.table[row * p.table_stride + c];
        if (pg >= 0 && pg < p.n_pages) ++pages;
        else record_error(kErrPageOutOfRange);
      }
      p.seqlens_out[row] = static_cast<int>(min(static_cast<long long>(l) + k, 2147483647ll));
    }
    long long at = back + static_cast<long long>(block_scan(static_cast<unsigned long long>(pages), warp_sums)) - pages;
    back += static_cast<long long>(warp_sums[32]);
    for (int c = c0; c < c1; ++c) {
      const int pg = p.table[row * p.table_stride + c];
      if (pg < 0 || pg >= p.n_pages) continue;
      if (at < room) p.queue[wrap(tail_at + at, p.n_pages)] = pg;
      ++at;
    }
    __syncthreads();  // warp_sums is free again
  }
  if (tid == 0) {
    if (back > room) record_error(kErrPagesExhausted);
    p.state_out[0] = head;
    p.state_out[1] = tail + min(back, room);
  }
}

__global__ void __launch_bounds__(kKeepThreads) paged_keep_kernel(const PagedKeepParams p) {
  __shared__ unsigned long long warp_sums[33];
  __shared__ long long s_src[kKeepThreads], s_dst[kKeepThreads];  // the moves' offsets in a slot, in order
  pdl_wait();  // no early trigger: this kernel may write cache_seqlens
  const int tid = threadIdx.x, page_len = 1 << p.page_shift;
  const int r = blockIdx.y;
  const bool row = r < p.R;  // (no rows: one block row for the counters alone)
  const int len = row ? keep_len(p, r) : 0, fresh = row ? max(p.new_lens[r], 0) : 0, kept = row ? keep_kept(p, r, fresh) : 0;
  if (row && blockIdx.x == 0 && tid == 0) {
    if (p.kept[r] > kept) record_error(kErrDraftOutOfRange);
    if (p.seqlens[r] != len || ((static_cast<long long>(len) + fresh + page_len - 1) >> p.page_shift) > p.max_pages)
      record_error(kErrPositionBeyondCache);
  }
  // this thread's 16 bytes of one head of one slot's K or V
  const int per_vec = p.D / 8;
  const long long column = static_cast<long long>(blockIdx.x) * kKeepThreads + tid;
  const long long vec = column / per_vec;
  const bool active = vec < 2ll * p.slots * p.Hkv;
  uint16_t* base = nullptr;
  if (active) {
    const long long h = (vec >> 1) % p.Hkv, slot = (vec >> 1) / p.Hkv;
    base = (vec & 1 ? p.v_pages : p.k_pages) + ((slot * p.n_pages * p.Hkv + h) << p.page_shift) * p.D +
           column % per_vec * 8;
  }
  const int moving = row && p.kept[r] >= 0 ? kept : 0;
  // Where the lengths' outputs are no inputs, one CTA more writes them beside the others' moves; else the last to
  // arrive, all having read them.  (All arriving before their moves, 1,500 atomics on one word in the way: 19 ->
  // 23 us for 128 requests of 24 slots.)
  if (!p.in_place && r >= p.R) {
    if (blockIdx.x == 0) keep_books(p, warp_sums);
    return;
  }
  for (int i0 = 0; i0 < moving; i0 += kKeepThreads) {
    const int i = i0 + tid;
    bool move = false;
    long long src = 0, dst = 0;
    if (i < moving) {
      const int from = p.path[r * p.path_stride + i];
      if (from < i || from >= fresh) record_error(kErrDraftOutOfRange);
      else if (from > i) {
        const long long a = static_cast<long long>(len) + from, b = static_cast<long long>(len) + i;
        if ((a >> p.page_shift) < p.max_pages) {
          const int pa = p.table[r * p.table_stride + (a >> p.page_shift)];
          const int pb = p.table[r * p.table_stride + (b >> p.page_shift)];
          move = pa >= 0 && pa < p.n_pages && pb >= 0 && pb < p.n_pages;
          if (!move) record_error(kErrPageOutOfRange);
          src = ((static_cast<long long>(pa) * p.Hkv << p.page_shift) + (a & (page_len - 1))) * p.D;
          dst = ((static_cast<long long>(pb) * p.Hkv << p.page_shift) + (b & (page_len - 1))) * p.D;
        }
      }
    }
    const int at = static_cast<int>(block_scan(move ? 1ull : 0ull, warp_sums)) - 1;
    const int moves = static_cast<int>(warp_sums[32]);
    if (move) {
      s_src[at] = src;
      s_dst[at] = dst;
    }
    __syncthreads();
    if (active) {
      constexpr int U = 4;
      for (int m = 0; m < moves; m += U) {
        uint4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (m + u < moves) v[u] = *reinterpret_cast<const uint4*>(base + s_src[m + u]);
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (m + u < moves) *reinterpret_cast<uint4*>(base + s_dst[m + u]) = v[u];
      }
    }
    __syncthreads();
  }
  if (p.in_place && last_cta(p.counter)) keep_books(p, warp_sums);
}

}  // namespace mcb
