// Attention over a paged cache for requests with few new tokens (T * G <= 8 NQT query rows a kv
// head): a flash-decode bound by HBM, every visible key and value read once.
//
//   out[t, h] = sum_c softmax_c(q[t, h] . K[c, h / G] * softmax_scale) V[c, h / G]
// over the keys c of the token's request with c <= pos and (window < 0 or pos - c <= window).
//
// A *unit* is (request, block of ROWS = 8 NQT flattened query rows r = t G + g, kv head).  Its key
// range -- the union of its rows' visible ranges, [lo, hi] -- is cut into 64-key tiles; all units'
// tiles in (request, block, head) order are one sequence of S tiles, and CTA c of the ng that work
// takes [c S / ng, (c + 1) S / ng).  Every CTA computes S from the lengths itself (one block scan),
// so the split is even for any batch and needs no host copy of the lengths.  A unit cut between
// CTAs leaves partials (O / l, log2 sum) in workspace; the contributor that arrives last merges
// them.  A unit is cut only at a CTA's end, so CTA c's counter serves the one unit that starts in c
// and ends after it.
//
// Per CTA a producer warp streams K and V tiles by TMA into a ring that is never drained between
// units: one 4-D box {64 columns, box positions, D / 64 panels, 1} a page chunk, box = min(page, 64),
// from the maps {64, page, D / 64, n_pages Hkv} over the pool -- a contiguous block, since a head's
// page is one.  The warp's lanes hold the next 32 chunks' page numbers.  Two groups of four consumer
// warps take turns at the tiles (a tile is a chain of dependent steps: 16 SMs reach 56 GB/s each
// with one group, 76 with two; one where registers would spill, 16 rows of 128, and at 64, where
// three CTAs share an SM), 16 keys a warp, on the tensor cores with keys on the M side (mma.sync m16n8k16):
//   S^T(16 keys x 8 rows) = K(16 x D) Q^T,  O^T(D x 8 rows) += V^T(D x 16 keys) P^T
// with an online softmax in fp32 a warp, P rounded to bf16 for the product (its sum l is of the
// unrounded values), and a merge of the eight through shared memory after each unit.
//
// Measured as called (and back to back in a graph): 128 requests at 1,024 to 8,192 positions, 16/4 heads of
// 128 (1.27 GB) 199 us (193), 6.4 TB/s; 13 of 4 tokens at 8,192 to 32,700, 32/8 heads (0.97 GB) 167 us (160);
// 64 of 12/12 heads of 64 at 1,024 to 8,192 (0.97 GB) 149 in a graph, 16 query rows a kv head (16/1 heads of
// 128, 128 requests, 0.32 GB) 72; 3 requests of 12 heads of 64 at 500 to 1,023 8.4 us (6.6), all of it
// latency (launch, lengths, page numbers, keys, merge: a chain of loads).
//
// Positions of a tile outside [lo, hi] may hold anything (another request's old values, NaN): their
// scores are replaced by -inf and their value rows are zeroed in shared memory, since 0 * NaN is NaN.
#pragma once

#include <math_constants.h>

#include "common.cuh"
#include "paged_plan.cuh"

namespace mcb {

struct PagedAttnParams {
  const uint16_t* q;
  long long qs[2];             // element strides: token, head
  const int32_t* block_table;  // (R, max_pages)
  long long table_stride;
  const int32_t* seqlens;      // (R,)
  const int32_t* cu_new;       // (R + 1,)
  uint16_t* out;               // (N, Hq, D) contiguous
  float* part_o;               // [(cta * 2 + slot) * rows + n][D]
  float* part_lse;             // [(cta * 2 + slot) * rows + n]
  int* counters;               // [cta], zero on entry, left zero
  int R, N, Hq, Hkv, G, n_pages, max_pages, page_shift, window;
  int few_rows;                // requests of at most this many query rows a kv head go to the decode kernel
  int all;                     // decode kernel: take every request (the chunk kernel is not launched)
  int fill;                    // this launch zeroes the padding tokens' output
  int tpb;                     // chunk kernel: tokens a query tile
  float scale_log2;            // softmax_scale * log2(e)
};

// A request's new tokens: first packed index, count, cached positions.
struct PagedRow {
  int tok0, T, L;
};

__device__ __forceinline__ PagedRow paged_row(const PagedAttnParams& p, int r) {
  PagedRow x;
  x.tok0 = min(max(p.cu_new[r], 0), p.N);
  x.T = min(max(p.cu_new[r + 1], x.tok0), p.N) - x.tok0;
  // a request that does not fit its table (reported by paged_row_fits) stays inside it
  const long long cap = static_cast<long long>(p.max_pages) << p.page_shift;
  x.L = static_cast<int>(min(static_cast<long long>(max(p.seqlens[r], 0)), max(cap - x.T, 0ll)));
  return x;
}

// Whether a request's lengths fit the table (the caller reports once).
__device__ __forceinline__ bool paged_row_fits(const PagedAttnParams& p, int r, const PagedRow& x) {
  return p.seqlens[r] >= 0 &&
         static_cast<long long>(p.seqlens[r]) + x.T <= (static_cast<long long>(p.max_pages) << p.page_shift);
}

constexpr int kPdTile = 64;  // keys a tile
template <int D, int NQT, int STAGES, int GROUPS>
struct PagedDecodeConfig {
  static constexpr int WARPS = 4 * GROUPS;           // consumer warps
  static constexpr int THREADS = (WARPS + 1) * 32;   // and the producer's
  static constexpr int kRows = 8 * NQT;
  static constexpr int NPANEL = D / 64;
  static constexpr int TILE_BYTES = kPdTile * D * 2;
  static constexpr int STAGE_BYTES = 2 * TILE_BYTES;
  static constexpr int RING_BYTES = STAGES * STAGE_BYTES;
  static constexpr int OPITCH = D + 4;
  static constexpr int MERGE_OFFSET = RING_BYTES;
  static constexpr int MERGE_BYTES = WARPS * kRows * OPITCH * 4;
  static constexpr int STAT_OFFSET = MERGE_OFFSET + MERGE_BYTES;
  static constexpr int STAT_BYTES = 2 * WARPS * kRows * 4;
  static constexpr int BAR_OFFSET = STAT_OFFSET + STAT_BYTES;
  static constexpr int SCAN_OFFSET = BAR_OFFSET + 2 * STAGES * 8;
  static constexpr int CTL_OFFSET = SCAN_OFFSET + 33 * 8;
  static constexpr int SMEM_BYTES = CTL_OFFSET + 64 + 1024;
  // a stage always holds the same group's tiles: its phases are then all waited for by that group
  static_assert(STAGES % GROUPS == 0, "whole turns");
  static_assert(BAR_OFFSET % 8 == 0 && SCAN_OFFSET % 8 == 0, "alignment");
};

// One unit of a request (kv head aside): its query rows [r0, r1), visible key range and tiles.
struct PagedUnit {
  PagedRow row;
  int r, qb, nqb, r0, r1, lo, hi, kb, n;
};

template <int ROWS>
__device__ __forceinline__ int paged_blocks(const PagedAttnParams& p, const PagedRow& x) {
  const long long rows = static_cast<long long>(x.T) * p.G;
  return rows <= p.few_rows || p.all ? static_cast<int>((rows + ROWS - 1) / ROWS) : 0;
}

template <int ROWS>
__device__ __forceinline__ PagedUnit paged_unit(const PagedAttnParams& p, const PagedRow& x, int r, int qb, int nqb) {
  PagedUnit u;
  u.row = x;
  u.r = r;
  u.qb = qb;
  u.nqb = nqb;
  u.r0 = qb * ROWS;
  u.r1 = min(u.r0 + ROWS, x.T * p.G);
  const int cap = static_cast<int>((static_cast<long long>(p.max_pages) << p.page_shift) - 1);
  u.hi = static_cast<int>(min(static_cast<long long>(x.L) + (u.r1 - 1) / p.G, static_cast<long long>(cap)));
  u.lo = p.window >= 0 ? max(0, x.L + u.r0 / p.G - p.window) : 0;
  u.kb = min(u.lo, u.hi) / kPdTile * kPdTile;
  u.n = (u.hi - u.kb) / kPdTile + 1;
  return u;
}

// CTA c's share of `total` tiles among ng <= 1,024 CTAs begins at c total / ng; the CTA whose share
// holds tile t.  (In 32 bits where they do: a 64-bit division is a hundred dependent instructions.)
__device__ __forceinline__ long long share_begin(int c, long long total, int ng) {
  if (total < (1 << 21)) return static_cast<uint32_t>(c) * static_cast<uint32_t>(total) / static_cast<uint32_t>(ng);
  return c * total / ng;
}
__device__ __forceinline__ int share_owner(long long t, long long total, int ng) {
  if (total < (1 << 21))
    return static_cast<int>((static_cast<uint32_t>(t + 1) * static_cast<uint32_t>(ng) - 1) / static_cast<uint32_t>(total));
  return static_cast<int>(((t + 1) * ng - 1) / total);
}

// A CTA's place in the tile sequence.
struct PagedWalk {
  PagedUnit u;
  int h, local;
  long long t;
};

// The next unit (the caller knows that one follows).
template <int ROWS>
__device__ __forceinline__ void paged_next(const PagedAttnParams& p, PagedWalk& w) {
  w.local = 0;
  if (++w.h < p.Hkv) return;
  w.h = 0;
  if (w.u.qb + 1 < w.u.nqb) {
    w.u = paged_unit<ROWS>(p, w.u.row, w.u.r, w.u.qb + 1, w.u.nqb);
    return;
  }
  for (int r = w.u.r + 1; r < p.R; ++r) {
    const PagedRow x = paged_row(p, r);
    const int nqb = paged_blocks<ROWS>(p, x);
    if (nqb > 0) {
      w.u = paged_unit<ROWS>(p, x, r, 0, nqb);
      return;
    }
  }
}

// Zeroes the output of the tokens that no request has, [0, cu_new[0]) and [cu_new[R], N): threads 0 ..
// threads - 1 of every CTA.
__device__ __forceinline__ void paged_fill(const PagedAttnParams& p, int D, int threads) {
  const long long per = static_cast<long long>(p.Hq) * D / 8;  // 16-byte words a token
  const int first = min(max(p.cu_new[0], 0), p.N), last = max(min(p.cu_new[p.R], p.N), first);
  const long long lead = first * per, gap = (last - first) * per, end = p.N * per;
  uint4* out = reinterpret_cast<uint4*>(p.out);
  for (long long i = static_cast<long long>(blockIdx.x) * threads + threadIdx.x; i < end - gap;
       i += static_cast<long long>(gridDim.x) * threads)
    out[i < lead ? i : i + gap] = make_uint4(0, 0, 0, 0);
}

// Merges the partials of a cut unit into its output rows, one warp a row: contributors g_first ..
// g_last (the first one's partial is its last unit's, slot 1 unless the unit began its share).  Online
// over 16 contributors at a time, their sums and values all loaded before the first is used: one trip
// to L2 where a pass for the maximum and four values in flight made five of it (7,000 -> 1,900 cycles; the
// 3 requests below 9.7 -> 7.2 us).
template <int D, int ROWS, typename RowOut>
__device__ __forceinline__ void paged_merge(const float* part_o, const float* part_lse, int g_first, int g_last,
                                            bool first_in_slot1, int n, RowOut row_out) {
  constexpr int PER_LANE = D / 32;
  constexpr int AHEAD = 16;
  const int lane = threadIdx.x & 31;
  const int cnt = g_last - g_first + 1;
  auto at = [&](int k) {
    return (static_cast<long long>(g_first + k) * 2 + (k == 0 && first_in_slot1 ? 1 : 0)) * ROWS + n;
  };
  float acc[PER_LANE], wsum = 0.f, mx = -CUDART_INF_F;
#pragma unroll
  for (int e = 0; e < PER_LANE; ++e) acc[e] = 0.f;
  for (int k0 = 0; k0 < cnt; k0 += AHEAD) {
    const float ls = lane < AHEAD && k0 + lane < cnt ? __ldcg(part_lse + at(k0 + lane)) : -CUDART_INF_F;
    float v[AHEAD][PER_LANE];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const float* src = part_o + at(min(k0 + j, cnt - 1)) * D + lane * PER_LANE;  // (a weight of 0 beyond cnt)
      if constexpr (PER_LANE == 4) {
        const float4 x = __ldcg(reinterpret_cast<const float4*>(src));
        v[j][0] = x.x, v[j][1] = x.y, v[j][2] = x.z, v[j][3] = x.w;
      } else {
        const float2 x = __ldcg(reinterpret_cast<const float2*>(src));
        v[j][0] = x.x, v[j][1] = x.y;
      }
    }
    float m_new = fmaxf(mx, ls);
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) m_new = fmaxf(m_new, __shfl_xor_sync(0xffffffffu, m_new, m));
    const float alpha = mx == -CUDART_INF_F ? 1.f : fast_exp2(mx - m_new);  // (nothing summed yet)
    const float wk = ls == -CUDART_INF_F ? 0.f : fast_exp2(ls - m_new);
    mx = m_new;
    wsum *= alpha;
#pragma unroll
    for (int e = 0; e < PER_LANE; ++e) acc[e] *= alpha;
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const float w = __shfl_sync(0xffffffffu, wk, j);
      wsum += w;
      if (w != 0.f)
#pragma unroll
        for (int e = 0; e < PER_LANE; ++e) acc[e] = fmaf(w, v[j][e], acc[e]);
    }
  }
  const float inv = wsum == 0.f ? 0.f : 1.f / wsum;
  uint16_t* dst = row_out(n) + lane * PER_LANE;
  if constexpr (PER_LANE == 4)
    *reinterpret_cast<uint2*>(dst) =
        make_uint2(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv));
  else
    *reinterpret_cast<uint32_t*>(dst) = pack_bf16x2(acc[0] * inv, acc[1] * inv);
}

template <int D, int NQT, int STAGES, int GROUPS>
__global__ void __launch_bounds__(PagedDecodeConfig<D, NQT, STAGES, GROUPS>::THREADS)
    paged_decode_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                        const PagedAttnParams p) {
  using C = PagedDecodeConfig<D, NQT, STAGES, GROUPS>;
  constexpr int WARPS = C::WARPS;
  constexpr int ROWS = C::kRows;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  float* merge = reinterpret_cast<float*>(smem + C::MERGE_OFFSET);
  float* stat = reinterpret_cast<float*>(smem + C::STAT_OFFSET);
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + C::BAR_OFFSET);
  uint64_t* empty_bar = full_bar + STAGES;
  unsigned long long* scan = reinterpret_cast<unsigned long long*>(smem + C::SCAN_OFFSET);
  int* ctl = reinterpret_cast<int*>(smem + C::CTL_OFFSET);  // abort; start r, qb, h, local, tok0, T, L; last
  volatile int* abort_flag = ctl;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 4);
    }
    ctl[0] = 0;
    fence_mbarrier_init();
    prefetch_tensormap(&kmap);
    prefetch_tensormap(&vmap);
  }
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();

  // ---- the sequence's length, and the unit holding this CTA's first tile ----
  // Up to 32 requests every warp does it alone, a request a lane: no barrier, nothing through shared
  // memory (3 requests of 12 heads of 64 at 500 to 1,023: 7.2 -> 6.6 us; 24 of 32/8 heads of 128: 33.0 ->
  // 32.2); more, the CTA together.
  PagedWalk w;
  long long t_end;
  int ng;
  long long total;
  if (p.R <= 32) {
    PagedRow x = {0, 0, 0};
    long long mine = 0;
    if (lane < p.R) {
      x = paged_row(p, lane);
      if (blockIdx.x == 0 && warp == 0 && !paged_row_fits(p, lane, x)) record_error(kErrPositionBeyondCache);
      const int nqb = paged_blocks<ROWS>(p, x);
      for (int qb = 0; qb < nqb; ++qb) mine += paged_unit<ROWS>(p, x, lane, qb, nqb).n;
      mine *= p.Hkv;
    }
    long long incl = mine;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const long long o = __shfl_up_sync(0xffffffffu, incl, m);
      if (lane >= m) incl += o;
    }
    total = __shfl_sync(0xffffffffu, incl, 31);
    ng = static_cast<int>(min(static_cast<long long>(gridDim.x), total));
    if (static_cast<int>(blockIdx.x) < ng) {
      w.t = share_begin(blockIdx.x, total, ng);
      t_end = share_begin(blockIdx.x + 1, total, ng);
      const int r = __ffs(__ballot_sync(0xffffffffu, w.t < incl)) - 1;  // (w.t < total: some lane's)
      long long left = w.t - __shfl_sync(0xffffffffu, incl - mine, r);
      x.tok0 = __shfl_sync(0xffffffffu, x.tok0, r);
      x.T = __shfl_sync(0xffffffffu, x.T, r);
      x.L = __shfl_sync(0xffffffffu, x.L, r);
      const int nqb = paged_blocks<ROWS>(p, x);
      w.u = paged_unit<ROWS>(p, x, r, 0, nqb);
      while (left >= static_cast<long long>(w.u.n) * p.Hkv) {
        left -= static_cast<long long>(w.u.n) * p.Hkv;
        w.u = paged_unit<ROWS>(p, x, r, w.u.qb + 1, nqb);
      }
      const uint32_t at = static_cast<uint32_t>(left);  // < n Hkv
      w.h = static_cast<int>(at / static_cast<uint32_t>(w.u.n));
      w.local = static_cast<int>(at % static_cast<uint32_t>(w.u.n));
    }
  } else {
    const int per = (p.R + C::THREADS - 1) / C::THREADS;
    const int row_a = min(static_cast<int>(threadIdx.x) * per, p.R), row_b = min(row_a + per, p.R);
    long long mine = 0;
    for (int r = row_a; r < row_b; ++r) {
      const PagedRow x = paged_row(p, r);
      if (blockIdx.x == 0 && !paged_row_fits(p, r, x)) record_error(kErrPositionBeyondCache);
      const int nqb = paged_blocks<ROWS>(p, x);
      for (int qb = 0; qb < nqb; ++qb) mine += paged_unit<ROWS>(p, x, r, qb, nqb).n;
    }
    mine *= p.Hkv;
    const long long incl = static_cast<long long>(block_scan(static_cast<unsigned long long>(mine), scan));
    total = static_cast<long long>(scan[32]);
    ng = static_cast<int>(min(static_cast<long long>(gridDim.x), total));
    if (static_cast<int>(blockIdx.x) < ng) {
      w.t = share_begin(blockIdx.x, total, ng);
      t_end = share_begin(blockIdx.x + 1, total, ng);
      if (incl - mine <= w.t && w.t < incl) {
        long long left = w.t - (incl - mine);
        bool found = false;
        for (int r = row_a; r < row_b && !found; ++r) {
          const PagedRow x = paged_row(p, r);
          const int nqb = paged_blocks<ROWS>(p, x);
          for (int qb = 0; qb < nqb; ++qb) {
            const int n = paged_unit<ROWS>(p, x, r, qb, nqb).n;
            if (left < static_cast<long long>(n) * p.Hkv) {
              const int at = static_cast<int>(left);  // < n * Hkv
              ctl[1] = r;
              ctl[2] = qb;
              ctl[3] = at / n;
              ctl[4] = at % n;
              ctl[5] = x.tok0;
              ctl[6] = x.T;
              ctl[7] = x.L;
              found = true;
              break;
            }
            left -= static_cast<long long>(n) * p.Hkv;
          }
        }
      }
      __syncthreads();
      const PagedRow x = {ctl[5], ctl[6], ctl[7]};
      w.u = paged_unit<ROWS>(p, x, ctl[1], ctl[2], paged_blocks<ROWS>(p, x));
      w.h = ctl[3];
      w.local = ctl[4];
    }
  }
  if (p.fill && warp < WARPS) paged_fill(p, D, WARPS * 32);
  if (static_cast<int>(blockIdx.x) >= ng) return;
  const int box_shift = min(p.page_shift, 6);  // positions a TMA box: min(page, 64)
  const int box = 1 << box_shift;
  const uint32_t panel_bytes = static_cast<uint32_t>(box) * 128u;

  if (warp == WARPS) {
    // ---------------- producer warp ----------------
    const uint64_t policy = l2_policy_evict_first();
    const int nch = kPdTile >> box_shift;  // chunks a tile
    const uint32_t chunk_bytes = panel_bytes * C::NPANEL;
    uint32_t g = 0;
    while (w.t < t_end) {
      const int seg = static_cast<int>(min(static_cast<long long>(w.u.n - w.local), t_end - w.t));
      const int32_t* table = p.block_table + w.u.r * p.table_stride;
      int base = -1, pg = 0;  // lane l holds the page of chunk base + l
      for (int i = 0; i < seg; ++i, ++g) {
        const int s = g % STAGES;
        const int c0 = (w.u.kb + (w.local + i) * kPdTile) >> box_shift;
        if (base < 0 || c0 + nch > base + 32) {
          base = c0;
          const long long key = static_cast<long long>(c0 + lane) << box_shift;
          pg = p.n_pages;  // outside the pool: a box there reads zeros
          if (key <= w.u.hi && key + box > w.u.lo) {
            pg = table[key >> p.page_shift];
            if (pg < 0 || pg >= p.n_pages) {
              record_error(kErrPageOutOfRange);
              pg = p.n_pages;
            }
          }
        }
        const int page = __shfl_sync(0xffffffffu, pg, (c0 - base + lane) & 31);
        const int key0 = (c0 + lane) << box_shift;
        const bool load = lane < nch && key0 <= w.u.hi && key0 + box > w.u.lo;
        const int loads = __popc(__ballot_sync(0xffffffffu, load));
        if (g >= STAGES) {
          const bool ok = mbar_wait_or_abort(&empty_bar[s], ((g / STAGES) - 1) & 1, abort_flag);
          if (!__all_sync(0xffffffffu, ok)) {  // a wait ran out: let the copies in flight land first
            for (uint32_t f = g - STAGES; f < g; ++f) mbar_wait(&full_bar[f % STAGES], (f / STAGES) & 1);
            return;
          }
        }
        if (lane == 0) mbar_arrive_expect_tx(&full_bar[s], static_cast<uint32_t>(loads) * 2 * chunk_bytes);
        __syncwarp();
        if (load) {
          uint8_t* kdst = smem + s * C::STAGE_BYTES + lane * chunk_bytes;
          const int pos = key0 & ((1 << p.page_shift) - 1);
          tma_load_4d(kdst, &kmap, &full_bar[s], 0, pos, 0, page * p.Hkv + w.h, policy);
          tma_load_4d(kdst + C::TILE_BYTES, &vmap, &full_bar[s], 0, pos, 0, page * p.Hkv + w.h, policy);
        }
      }
      w.t += seg;
      w.local += seg;
      if (w.local == w.u.n && w.t < t_end) paged_next<ROWS>(p, w);
    }
    return;
  }

  // ---------------- consumer warps ----------------
  // this lane's rows of the tile for the K (ldmatrix) and V (ldmatrix.trans) fragments
  auto row_offset = [&](int row) {
    return static_cast<uint32_t>(row >> box_shift) * panel_bytes * C::NPANEL +
           static_cast<uint32_t>(row & (box - 1)) * 128u;
  };
  const int part = warp & 3;  // of the tile: keys part * 16 .. +15
  const int krow = part * 16 + (lane & 7) + ((lane >> 3) & 1) * 8;
  const int vrow = part * 16 + (lane & 7) + (lane >> 4) * 8;
  const uint32_t koff = row_offset(krow), voff = row_offset(vrow);
  const uint32_t swz = static_cast<uint32_t>(lane & 7) << 4;
  uint32_t g = 0;
  int seg_index = 0;

  auto load_q = [&](const PagedWalk& x, uint32_t(&qf)[NQT][D / 16][2]) {
#pragma unroll
    for (int j = 0; j < NQT; ++j) {
      const int r = x.u.r0 + j * 8 + (lane >> 2);
      const uint16_t* src = nullptr;
      if (r < x.u.r1)
        src = p.q + (x.u.row.tok0 + r / p.G) * p.qs[0] + (x.h * p.G + r % p.G) * p.qs[1];
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const int d0 = kk * 16 + 2 * (lane & 3);
        qf[j][kk][0] = src ? *reinterpret_cast<const uint32_t*>(src + d0) : 0u;
        qf[j][kk][1] = src ? *reinterpret_cast<const uint32_t*>(src + d0 + 8) : 0u;
      }
    }
  };
  uint32_t qf[NQT][D / 16][2];
  load_q(w, qf);
  while (w.t < t_end) {
    const PagedUnit& u = w.u;
    const int seg = static_cast<int>(min(static_cast<long long>(u.n - w.local), t_end - w.t));
    const bool complete = w.local == 0 && seg == u.n;
    const int slot = seg_index == 0 ? 0 : 1;
    const int nvalid = u.r1 - u.r0;
    const long long start = w.t - w.local;  // the unit's first tile, and who has its tiles
    int g_first = 0, g_last = 0;
    if (!complete) {
      g_first = share_owner(start, total, ng);
      g_last = share_owner(start + u.n - 1, total, ng);
    }

    float m_run[NQT][2], l_run[NQT][2], o_acc[NQT][D / 16][4];
    int row_hi[NQT][2], row_lo[NQT][2];
#pragma unroll
    for (int j = 0; j < NQT; ++j) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int rr = u.r0 + j * 8 + 2 * (lane & 3) + e;
        m_run[j][e] = -CUDART_INF_F;
        l_run[j][e] = 0.f;
        const int qpos = u.row.L + rr / p.G;
        row_hi[j][e] = rr < u.r1 ? min(qpos, u.hi) : -1;  // a padding row sees nothing
        row_lo[j][e] = p.window >= 0 ? qpos - p.window : 0;
      }
#pragma unroll
      for (int db = 0; db < D / 16; ++db)
#pragma unroll
        for (int c = 0; c < 4; ++c) o_acc[j][db][c] = 0.f;
    }

    for (int i = 0; i < seg; ++i, ++g) {
      if ((g & (GROUPS - 1)) != static_cast<uint32_t>(warp >> 2)) continue;  // the other group's tile
      const int s = g % STAGES;
      if (mbar_wait_or_abort(&full_bar[s], (g / STAGES) & 1, abort_flag)) {
        const uint32_t kbase = smem_u32(smem + s * C::STAGE_BYTES);
        const uint32_t vbase = kbase + C::TILE_BYTES;
        const int tile0 = u.kb + (w.local + i) * kPdTile;
        const bool edge = tile0 < u.lo || tile0 + kPdTile - 1 > u.hi;
        if (edge) {
          // value rows outside [lo, hi] to zero (this warp's 16 rows; two lanes a row)
          const int row = part * 16 + (lane >> 1);
          if (tile0 + row < u.lo || tile0 + row > u.hi) {
            const uint32_t at = vbase + row_offset(row);
#pragma unroll
            for (int c = 0; c < D / 16; ++c)
              sts128(at + (c >> 2) * panel_bytes + ((c & 3) * 2 + (lane & 1)) * 16, make_uint4(0, 0, 0, 0));
          }
          fence_proxy_async_shared();  // TMA refills this stage later
          __syncwarp();
        }
        float sc[NQT][4], sd[NQT][4];  // even and odd steps: two dependent chains instead of one
#pragma unroll
        for (int j = 0; j < NQT; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) sc[j][c] = sd[j][c] = 0.f;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t chunk = ((kk & 3) * 2 + (lane >> 4)) << 4;
          uint32_t a0, a1, a2, a3;
          ldsm_x4(kbase + koff + (kk >> 2) * panel_bytes + (chunk ^ swz), a0, a1, a2, a3);
#pragma unroll
          for (int j = 0; j < NQT; ++j) mma_16816(kk & 1 ? sd[j] : sc[j], a0, a1, a2, a3, qf[j][kk][0], qf[j][kk][1]);
        }
#pragma unroll
        for (int j = 0; j < NQT; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) sc[j][c] += sd[j][c];
        const int key = tile0 + part * 16 + (lane >> 2);
#pragma unroll
        for (int j = 0; j < NQT; ++j) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& s0 = sc[j][e];
            float& s1 = sc[j][e + 2];
            if (key > row_hi[j][e] || key < row_lo[j][e]) s0 = -CUDART_INF_F;
            if (key + 8 > row_hi[j][e] || key + 8 < row_lo[j][e]) s1 = -CUDART_INF_F;
            float mx = fmaxf(s0, s1);
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            const float m_new = fmaxf(m_run[j][e], mx);
            float alpha = 1.f, msub = 0.f;
            if (m_new != -CUDART_INF_F) {
              alpha = fast_exp2((m_run[j][e] - m_new) * p.scale_log2);
              msub = m_new * p.scale_log2;
            }
            m_run[j][e] = m_new;
            s0 = fast_exp2(fmaf(s0, p.scale_log2, -msub));  // exp2(-inf) = 0 for masked keys
            s1 = fast_exp2(fmaf(s1, p.scale_log2, -msub));
            l_run[j][e] = fmaf(l_run[j][e], alpha, s0 + s1);
#pragma unroll
            for (int db = 0; db < D / 16; ++db) {
              o_acc[j][db][e] *= alpha;
              o_acc[j][db][e + 2] *= alpha;
            }
          }
        }
        uint32_t pb[NQT][2];
#pragma unroll
        for (int j = 0; j < NQT; ++j) {
          pb[j][0] = movmatrix_trans(pack_bf16x2(sc[j][0], sc[j][1]));
          pb[j][1] = movmatrix_trans(pack_bf16x2(sc[j][2], sc[j][3]));
        }
#pragma unroll
        for (int db = 0; db < D / 16; ++db) {
          const uint32_t chunk = ((db & 3) * 2 + ((lane >> 3) & 1)) << 4;
          uint32_t a0, a1, a2, a3;
          ldsm_x4_trans(vbase + voff + (db >> 2) * panel_bytes + (chunk ^ swz), a0, a1, a2, a3);
#pragma unroll
          for (int j = 0; j < NQT; ++j) mma_16816(o_acc[j][db], a0, a1, a2, a3, pb[j][0], pb[j][1]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty_bar[s]);
    }

    // the next unit's query fragments load while this one merges
    PagedWalk wn = w;
    wn.t += seg;
    wn.local += seg;
    if (wn.t < t_end) {
      if (wn.local == wn.u.n) paged_next<ROWS>(p, wn);
      load_q(wn, qf);
    }

    // ---- merge the warps' states ----
    float* mbuf = merge;
    float* st_m = stat;
    float* st_l = st_m + WARPS * ROWS;
    if (seg_index > 0) named_barrier(1, WARPS * 32);  // the last unit's have been read
#pragma unroll
    for (int j = 0; j < NQT; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float v = l_run[j][e];
        v += __shfl_xor_sync(0xffffffffu, v, 4);
        v += __shfl_xor_sync(0xffffffffu, v, 8);
        v += __shfl_xor_sync(0xffffffffu, v, 16);
        const int n = j * 8 + 2 * (lane & 3) + e;
        if (n >= nvalid) continue;
        if (lane < 4) {
          st_m[warp * ROWS + n] = m_run[j][e];
          st_l[warp * ROWS + n] = v;
        }
        float* dst = mbuf + (warp * ROWS + n) * C::OPITCH;
#pragma unroll
        for (int db = 0; db < D / 16; ++db) {
          const int d = db * 16 + (lane >> 2);
          dst[d] = o_acc[j][db][e];
          dst[d + 8] = o_acc[j][db][e + 2];
        }
      }
    named_barrier(1, WARPS * 32);
    auto row_out = [&](int n) {
      const int r = u.r0 + n;
      return p.out + (static_cast<long long>(u.row.tok0 + r / p.G) * p.Hq + w.h * p.G + r % p.G) * D;
    };
    for (int idx = threadIdx.x; idx < nvalid * D; idx += WARPS * 32) {
      const int n = idx / D, d = idx - n * D;
      float mmax = -CUDART_INF_F;
#pragma unroll
      for (int ww = 0; ww < WARPS; ++ww) mmax = fmaxf(mmax, st_m[ww * ROWS + n]);
      float ltot = 0.f, o = 0.f;
#pragma unroll
      for (int ww = 0; ww < WARPS; ++ww) {
        const float mw = st_m[ww * ROWS + n];
        const float f = mw == -CUDART_INF_F ? 0.f : fast_exp2((mw - mmax) * p.scale_log2);
        ltot = fmaf(st_l[ww * ROWS + n], f, ltot);
        o = fmaf(mbuf[(ww * ROWS + n) * C::OPITCH + d], f, o);
      }
      o = ltot == 0.f ? 0.f : o / ltot;  // (a NaN stays one)
      if (complete) {
        row_out(n)[d] = float_to_bf16_bits(o);
      } else {
        const long long prow = (static_cast<long long>(blockIdx.x) * 2 + slot) * ROWS + n;
        p.part_o[prow * D + d] = o;
        if (d == 0) p.part_lse[prow] = ltot == 0.f ? -CUDART_INF_F : mmax * p.scale_log2 + __log2f(ltot);
      }
    }
    if (!complete) {
      // the barrier orders every thread's stores before thread 0's release of the counter
      named_barrier(1, WARPS * 32);
      if (threadIdx.x == 0) {
        int* counter = p.counters + g_first;
        const bool last = atom_add_acq_rel_gpu(counter, 1) == g_last - g_first;
        if (last) *counter = 0;  // every contributor has arrived: ready for the next call
        ctl[8] = last;
      }
      named_barrier(1, WARPS * 32);
      if (ctl[8])
        for (int n = warp; n < nvalid; n += WARPS)
          paged_merge<D, ROWS>(p.part_o, p.part_lse, g_first, g_last, start != share_begin(g_first, total, ng), n,
                               row_out);
    }
    ++seg_index;
    w = wn;
  }
}

}  // namespace mcb
