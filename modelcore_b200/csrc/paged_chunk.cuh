// Attention over a paged cache for chunks of new tokens (more query rows a kv head than the decode
// kernel takes): tcgen05 products with TMEM accumulators, bound by the tensor cores for long
// chunks and by HBM for short ones.
//
// The query rows of one kv head are packed, row = token * G + head of the group, so a 128-row tile
// is TPB = floor(128 / G) tokens with all G heads: the K/V tiles they share are read once, and a
// short chunk still fills rows.  A *unit* is (request, 2 TPB tokens = two tiles Q0, Q1, kv head);
// its key range -- from the first key its first token sees to its last token's position -- is cut
// into 128-key tiles, each serving both query tiles.  As in the decode kernel, all units' key tiles
// form one sequence that the CTAs (one an SM) share evenly, computed on the device from the
// lengths; a cut unit leaves (O / l, log2 sum) in workspace and paged_combine_kernel, launched
// after, merges them (spread over the GPU: one CTA merging a unit cut eighteen ways would take
// longer than its share of the products).
//
// Roles of a CTA's ten warps:
//   warp 0      TMA producer: Q0, Q1 per unit; K_j, V_j into a two-stage ring that runs on across
//               units, one box a (page chunk, 64-column panel); lanes hold the next page numbers
//   warp 1      allocates TMEM; lane 0 issues the products
//                 S_t = Q_t K_j^T   M=128 N=128 K=D  (both operands from shared memory)
//                 O_t += P_t V_j    M=128 N=D K=128  (P from TMEM)
//   warps 2-5   softmax of Q0, warps 6-9 of Q1: one thread a query row
// TMEM: S0, S1 (128 columns each), O0, O1 (D each).  D = 128 fills the 512 columns, so P (bf16)
// is written over S and the issue order is PV0_j S0_j+1 PV1_j S1_j+1: one tile's products run
// during the other's softmax.  With D = 64 P has columns of its own, and S_j+1 is computed as soon
// as S_j has been read.
//
// Softmax without a maximum on the critical path: the exponent's reference m is a maximum the row
// has really had (its first tile's), moved only when it must be.  A tile in which every row has an m
// and nothing is masked is exponentiated at once; P and l may then exceed 1 -- fp32 and bf16 reach
// 2^127 -- and only when a row's sum over the tile leaves 2^100 is the tile redone with a new m (S is
// still in TMEM) and O and l rescaled.  Other tiles (masked edges, a row's first keys) take the
// maximum first and move m when it grew by 2^8.  Rounding: P to bf16 for the product; l sums the
// unrounded values.
// Some of the exponentials run as a polynomial on the FMA pipe (exp2_poly_pair): the 16 a clock
// an SM of the special function unit would otherwise take as long as the products.
//
// A key tile's positions outside the unit's [lo, hi] may hold anything: scores there are replaced
// by -inf (never computed with), and their rows of V are zeroed in shared memory by the softmax
// threads before the product reads them (0 * NaN is NaN).
// Every wait is bounded; a timeout raises the abort flag, the issuer waits for its products, the
// producer for its copies, and TMEM is freed.
#pragma once

#include "paged_decode.cuh"
#include "prefill_attn.cuh"

namespace mcb {

constexpr int kPcTile = 128;      // query rows a tile, keys a key tile
constexpr int kPcThreads = 320;   // producer, issuer, 2 x 4 softmax warps

// What paged_combine_kernel needs of the unit that starts in a CTA's share and ends after it.
struct PagedCut {
  int tok0, tok1;      // the unit's tokens [tok0, tok1) in the packed batch
  int h, g_last;       // kv head; last contributing CTA (h < 0: no such unit)
  int slot1, pad[3];   // the first contributor's partial is in its slot 1
};

struct PagedChunkParams {
  PagedAttnParams a;
  PagedCut* cuts;      // [grid]
  int tpb;             // tokens a tile
  int wait_last;       // the kernel ahead is this call's decode kernel, whose output this one does
                       // not read: wait for it only before the end
};

template <int D>
struct PagedChunkConfig {
  static constexpr int kPanels = D / 64;
  static constexpr int kTileBytes = kPanels * kPcTile * 128;
  static constexpr bool kSepP = D == 64;                 // P in columns of its own
  static constexpr uint32_t kPCol = 2 * kPcTile;         // (kSepP) P0, P1: 64 columns each
  static constexpr uint32_t kOCol = kSepP ? 3 * kPcTile : 2 * kPcTile;
  static constexpr int kKOff = 2 * kTileBytes;           // Q0, Q1, then K and V, two stages each
  static constexpr int kVOff = kKOff + 2 * kTileBytes;
  static constexpr int kBarOff = kVOff + 2 * kTileBytes;
  static constexpr int kScanOff = kBarOff + 256;
  static constexpr int kBytes = kScanOff + 256 + 1024;
  // above half of an SM's shared memory: two CTAs never meet on one SM, whose TMEM each needs whole
  static constexpr int kSmem = kBytes > 118784 ? kBytes : 118784;
};

__device__ __forceinline__ void tma_load_3d(void* smem_dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1,
                                            int c2, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4, %5}], [%2], %6;" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "l"(policy)
      : "memory");
}

__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float lo_f(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v)); }
__device__ __forceinline__ float hi_f(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v >> 32)); }

__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// (2^a, 2^b) of a pair, each clamped below at 2^-125, as exp2_poly3: x = n + f, n = round(x) by the
// 1.5 * 2^23 constant, a cubic for 2^f, and n added to the exponent (the constant's own bits leave
// the word when shifted by 23).  Packed except the clamp and the exponent.  Above 2^127 the result
// is meaningless: the caller watches the inputs' maximum.  A NaN comes out as 3.4e38, which the
// caller's bound on the sum catches.
__device__ __forceinline__ uint64_t exp2_poly_pair(uint64_t x) {
  const uint64_t xc = pair_f32(max_nan(lo_f(x), -125.f), max_nan(hi_f(x), -125.f));
  const uint64_t magic = pair_f32(12582912.f, 12582912.f), unmagic = pair_f32(-12582912.f, -12582912.f);
  const uint64_t t = add2(xc, magic);
  const uint64_t f = fma2(add2(t, unmagic), pair_f32(-1.f, -1.f), xc);
  uint64_t q = fma2(pair_f32(0.0551716648f, 0.0551716648f), f, pair_f32(0.242611125f, 0.242611125f));
  q = fma2(q, f, pair_f32(0.693260968f, 0.693260968f));
  q = fma2(q, f, pair_f32(0.999928057f, 0.999928057f));
  const uint32_t r0 = static_cast<uint32_t>(q) + (static_cast<uint32_t>(t) << 23);
  const uint32_t r1 = static_cast<uint32_t>(q >> 32) + (static_cast<uint32_t>(t >> 32) << 23);
  return static_cast<uint64_t>(r0) | static_cast<uint64_t>(r1) << 32;
}

// A unit (kv head aside): tiles' first tokens and counts, their key-tile ranges from kb.
struct ChunkUnit {
  PagedRow row;
  int r, qb, nqb;
  int c0, c1;            // tokens in Q0 and Q1 (first tokens: qb * 2 tpb, + tpb)
  int b0, e0, b1, e1;    // key tiles [b, e) each query tile needs, counted from kb
  int lo, hi, kb, n;
};

__device__ __forceinline__ int chunk_blocks(const PagedChunkParams& p, const PagedRow& x) {
  return static_cast<long long>(x.T) * p.a.G > p.a.few_rows ? (x.T + 2 * p.tpb - 1) / (2 * p.tpb) : 0;
}

__device__ __forceinline__ ChunkUnit chunk_unit(const PagedChunkParams& p, const PagedRow& x, int r, int qb, int nqb) {
  ChunkUnit u;
  u.row = x;
  u.r = r;
  u.qb = qb;
  u.nqb = nqb;
  const int first = qb * 2 * p.tpb, left = x.T - first;
  u.c0 = min(left, p.tpb);
  u.c1 = min(max(left - p.tpb, 0), p.tpb);
  const int cap = static_cast<int>((static_cast<long long>(p.a.max_pages) << p.a.page_shift) - 1);
  auto last_key = [&](int tok) { return static_cast<int>(min(static_cast<long long>(x.L) + tok, static_cast<long long>(cap))); };
  auto first_key = [&](int tok) { return p.a.window >= 0 ? max(0, x.L + tok - p.a.window) : 0; };
  u.lo = first_key(first);
  u.hi = last_key(first + u.c0 + u.c1 - 1);
  u.kb = min(u.lo, u.hi) / kPcTile * kPcTile;
  u.n = (u.hi - u.kb) / kPcTile + 1;
  u.b0 = 0;
  u.e0 = (last_key(first + u.c0 - 1) - u.kb) / kPcTile + 1;
  u.b1 = u.e1 = 0;
  if (u.c1 > 0) {
    u.b1 = min((min(first_key(first + p.tpb), u.hi) - u.kb) / kPcTile, u.n - 1);
    u.e1 = u.n;
  }
  return u;
}

struct ChunkWalk {
  ChunkUnit u;
  int h, local;
  long long t;
};

__device__ __forceinline__ void chunk_next(const PagedChunkParams& p, ChunkWalk& w) {
  w.local = 0;
  if (++w.h < p.a.Hkv) return;
  w.h = 0;
  if (w.u.qb + 1 < w.u.nqb) {
    w.u = chunk_unit(p, w.u.row, w.u.r, w.u.qb + 1, w.u.nqb);
    return;
  }
  for (int r = w.u.r + 1; r < p.a.R; ++r) {
    const PagedRow x = paged_row(p.a, r);
    const int nqb = chunk_blocks(p, x);
    if (nqb > 0) {
      w.u = chunk_unit(p, x, r, 0, nqb);
      return;
    }
  }
}

// The rows of one warp's share, 32 at a time (a lane each), the blocks of each row with any in turn
// (a lane each): visit(r, nqb, row, first block of this lane's batch, lane's tile count, valid).
// Stops when visit returns true (uniform).
template <typename F>
__device__ __forceinline__ void chunk_rows(const PagedChunkParams& p, int row_a, int row_b, F visit) {
  const int lane = threadIdx.x & 31;
  for (int base = row_a; base < row_b; base += 32) {
    PagedRow x = {0, 0, 0};
    int nqb = 0;
    if (base + lane < row_b) {
      x = paged_row(p.a, base + lane);
      if (blockIdx.x == 0 && !paged_row_fits(p.a, base + lane, x)) record_error(kErrPositionBeyondCache);
      nqb = chunk_blocks(p, x);
    }
    unsigned have = __ballot_sync(0xffffffffu, nqb > 0);
    while (have) {
      const int src = __ffs(have) - 1;
      have &= have - 1;
      PagedRow y;
      y.tok0 = __shfl_sync(0xffffffffu, x.tok0, src);
      y.T = __shfl_sync(0xffffffffu, x.T, src);
      y.L = __shfl_sync(0xffffffffu, x.L, src);
      const int nb = __shfl_sync(0xffffffffu, nqb, src);
      for (int qb = 0; qb < nb; qb += 32) {
        const int n = qb + lane < nb ? chunk_unit(p, y, base + src, qb + lane, nb).n : 0;
        if (visit(base + src, qb, n)) return;
      }
    }
  }
}

template <int D>
__global__ void __launch_bounds__(kPcThreads, 1)
    paged_chunk_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                       const __grid_constant__ CUtensorMap vmap, const PagedChunkParams p) {
  using Cfg = PagedChunkConfig<D>;
  constexpr bool SEP = Cfg::kSepP;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::kBarOff);
  uint64_t* q_full = bars + 0;
  uint64_t* q_empty = bars + 1;
  uint64_t* k_full = bars + 2;    // [2]
  uint64_t* v_full = bars + 4;    // [2]
  uint64_t* kv_empty = bars + 6;  // [2]
  uint64_t* s_full = bars + 8;    // [2] per query tile
  uint64_t* p_full = bars + 10;   // [2] 128 arrivals
  uint64_t* s_free = bars + 12;   // [2] 128 arrivals (SEP): S has been read
  uint64_t* pv_done = bars + 14;  // [2] (SEP): a P V product has completed
  uint64_t* o_done = bars + 16;
  uint64_t* epi_done = bars + 17; // 256 arrivals, once a unit
  uint64_t* drained = bars + 18;
  constexpr int kNumBars = 19;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kNumBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + kNumBars + 1);
  int* ctl = reinterpret_cast<int*>(bars + kNumBars + 2);  // start: r, qb, h, local
  long long* warp_tot = reinterpret_cast<long long*>(smem + Cfg::kScanOff);  // [10]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kNumBars; ++i) mbar_init(bars + i, i >= 10 && i < 14 ? 128 : i == 17 ? 256 : 1);
    *abort_flag = 0;
    fence_mbarrier_init();
    prefetch_tensormap(&qmap);
    prefetch_tensormap(&kmap);
    prefetch_tensormap(&vmap);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (!p.wait_last) {
    pdl_wait();
    pdl_launch_dependents();
  }

  // ---- the sequence's length and this CTA's first tile ----
  const int per = (p.a.R + 9) / 10;
  const int row_a = min(warp * per, p.a.R), row_b = min(row_a + per, p.a.R);
  long long mine = 0;
  chunk_rows(p, row_a, row_b, [&](int, int, int n) {
    mine += n;
    return false;
  });
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, m);
  mine *= p.a.Hkv;
  if (lane == 0) warp_tot[warp] = mine;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  long long total = 0, before = 0;
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    if (i < warp) before += warp_tot[i];
    total += warp_tot[i];
  }
  if (p.a.fill) paged_fill(p.a, D);
  const int ng = static_cast<int>(min(static_cast<long long>(gridDim.x), total));
  const bool active = static_cast<int>(blockIdx.x) < ng;
  const long long t_begin = active ? share_begin(blockIdx.x, total, ng) : 0;
  const long long t_end = active ? share_begin(blockIdx.x + 1, total, ng) : 0;
  if (active && before <= t_begin && t_begin < before + mine) {
    long long left = t_begin - before;
    chunk_rows(p, row_a, row_b, [&](int r, int qb, int n) {
      int incl = n;
#pragma unroll
      for (int m = 1; m < 32; m <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, incl, m);
        if (lane >= m) incl += o;
      }
      const long long all = static_cast<long long>(__shfl_sync(0xffffffffu, incl, 31)) * p.a.Hkv;
      if (left >= all) {
        left -= all;
        return false;
      }
      const long long mine0 = static_cast<long long>(incl - n) * p.a.Hkv;
      if (n > 0 && mine0 <= left && left < mine0 + static_cast<long long>(n) * p.a.Hkv) {
        ctl[0] = r;
        ctl[1] = qb + lane;
        ctl[2] = static_cast<int>((left - mine0) / n);
        ctl[3] = static_cast<int>((left - mine0) % n);
      }
      return true;
    });
  }
  if (threadIdx.x == 0) p.cuts[blockIdx.x].h = -1;
  __syncthreads();
  const uint32_t tmem = *tmem_slot;
  const uint32_t base = smem_u32(smem);
  ChunkWalk w;
  w.t = t_begin;
  if (active) {
    const PagedRow x = paged_row(p.a, ctl[0]);
    w.u = chunk_unit(p, x, ctl[0], ctl[1], chunk_blocks(p, x));
    w.h = ctl[2];
    w.local = ctl[3];
  }

  if (warp == 0) {
    // ---------------- producer warp ----------------
    const uint64_t pol = l2_policy_evict_first();
    const int box_shift = min(p.a.page_shift, 7);  // positions a box: min(page, 128)
    const int box = 1 << box_shift, nch = kPcTile >> box_shift;
    const uint32_t box_bytes = static_cast<uint32_t>(box) * 128u;
    const uint32_t q_bytes = static_cast<uint32_t>(p.tpb * p.a.G) * 128u;
    int g = 0, k = 0;
    bool ok = true;
    while (ok && w.t < t_end) {
      const int seg = static_cast<int>(min(static_cast<long long>(w.u.n - w.local), t_end - w.t));
      if (k > 0) ok = __all_sync(0xffffffffu, mbar_wait_or_abort(q_empty, (k - 1) & 1, abort_flag));
      if (!ok) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(q_full, (w.u.c1 > 0 ? 2 : 1) * Cfg::kPanels * q_bytes);
        for (int t = 0; t < (w.u.c1 > 0 ? 2 : 1); ++t)
#pragma unroll
          for (int pn = 0; pn < Cfg::kPanels; ++pn)
            tma_load_3d(smem + t * Cfg::kTileBytes + pn * kPcTile * 128, &qmap, q_full, pn * 64, w.h * p.a.G,
                        w.u.row.tok0 + (w.u.qb * 2 + t) * p.tpb, pol);
      }
      ++k;
      const int32_t* table = p.a.block_table + w.u.r * p.a.table_stride;
      int pbase = -1, pg = 0;  // lane l holds the page of chunk pbase + l
      for (int i = 0; i < seg; ++i, ++g) {
        const int st = g & 1;
        const int c0 = (w.u.kb + (w.local + i) * kPcTile) >> box_shift;
        if (pbase < 0 || c0 + nch > pbase + 32) {
          pbase = c0;
          const long long key = static_cast<long long>(c0 + lane) << box_shift;
          pg = p.a.n_pages;  // outside the pool: a box there reads zeros
          if (key <= w.u.hi && key + box > w.u.lo) {
            pg = table[key >> p.a.page_shift];
            if (pg < 0 || pg >= p.a.n_pages) {
              record_error(kErrPageOutOfRange);
              pg = p.a.n_pages;
            }
          }
        }
        // lane l: chunk l / panels, panel l % panels
        const int ch = lane / Cfg::kPanels, pn = lane % Cfg::kPanels;
        const int page = __shfl_sync(0xffffffffu, pg, (c0 - pbase + ch) & 31);
        const int key0 = (c0 + ch) << box_shift;
        const bool load = ch < nch && key0 <= w.u.hi && key0 + box > w.u.lo;
        const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, load)) * box_bytes;
        if (g >= 2) {
          ok = __all_sync(0xffffffffu, mbar_wait_or_abort(&kv_empty[st], ((g >> 1) - 1) & 1, abort_flag));
          if (!ok) break;
        }
        if (lane == 0) {
          mbar_arrive_expect_tx(&k_full[st], bytes);
          mbar_arrive_expect_tx(&v_full[st], bytes);
        }
        __syncwarp();
        if (load) {
          const int pos = key0 & ((1 << p.a.page_shift) - 1);
          uint8_t* dst = smem + st * Cfg::kTileBytes + pn * kPcTile * 128 + ch * box_bytes;
          tma_load_4d(dst + Cfg::kKOff, &kmap, &k_full[st], 0, pos, pn, page * p.a.Hkv + w.h, pol);
          tma_load_4d(dst + Cfg::kVOff, &vmap, &v_full[st], 0, pos, pn, page * p.a.Hkv + w.h, pol);
        }
      }
      if (!ok) break;
      w.t += seg;
      w.local += seg;
      if (w.local == w.u.n && w.t < t_end) chunk_next(p, w);
    }
    if (*abort_flag && lane == 0) {  // the copies in flight land before the CTA can exit
      for (int f = max(0, g - 2); f < g; ++f) {
        mbar_wait(&k_full[f & 1], (f >> 1) & 1);
        mbar_wait(&v_full[f & 1], (f >> 1) & 1);
      }
      if (k > 0) mbar_wait(q_full, (k - 1) & 1);
    }
    __syncwarp();
  } else if (warp == 1 && lane == 0) {
    // ---------------- product issuer ----------------
    constexpr uint32_t idesc_s = umma_idesc_bf16(128, kPcTile, 0);
    constexpr uint32_t idesc_o = umma_idesc_bf16(128, D, 1);
    int g = 0, k = 0;
    int pv_total[2] = {0, 0}, s_total[2] = {0, 0};
    bool ok = true;
    while (ok && w.t < t_end) {
      const int seg = static_cast<int>(min(static_cast<long long>(w.u.n - w.local), t_end - w.t));
      // this segment's key tiles [b, e) of each query tile, from w.local
      const int b0 = max(w.u.b0 - w.local, 0), e0 = min(w.u.e0 - w.local, seg);
      const int b1 = max(w.u.b1 - w.local, 0), e1 = min(w.u.e1 - w.local, seg);
      const int s_here = max(e0 - b0, 0) + max(e1 - b1, 0);
      ok = mbar_wait_or_abort(q_full, k & 1, abort_flag);
      int k_waited = -1, v_waited = -1, s_issued = 0;
      int pv_unit[2] = {0, 0};
      auto on = [&](int t, int j) { return t == 0 ? j >= b0 && j < e0 : j >= b1 && j < e1; };
      auto issue_s = [&](int t, int j) -> bool {
        const int gj = g + j;
        if (SEP && s_total[t] > 0 && !mbar_wait_or_abort(&s_free[t], (s_total[t] - 1) & 1, abort_flag)) return false;
        ++s_total[t];
        if (k_waited < j) {
          if (!mbar_wait_or_abort(&k_full[gj & 1], (gj >> 1) & 1, abort_flag)) return false;
          k_waited = j;
        }
        tc_fence_after();
        const uint32_t qa = base + t * Cfg::kTileBytes, ka = base + Cfg::kKOff + (gj & 1) * Cfg::kTileBytes;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (kk >> 2) * (kPcTile * 128) + (kk & 3) * 32;
          umma_ss(tmem + t * kPcTile, smem_desc_sw128(qa + off, 16, 1024), smem_desc_sw128(ka + off, 16, 1024),
                  idesc_s, kk > 0 ? 1u : 0u);
        }
        umma_commit(&s_full[t]);
        if (++s_issued == s_here) umma_commit(q_empty);
        return true;
      };
      auto issue_pv = [&](int t, int j) -> bool {
        const int gj = g + j;
        if (!mbar_wait_or_abort(&p_full[t], pv_total[t] & 1, abort_flag)) return false;
        if (v_waited < j) {
          if (!mbar_wait_or_abort(&v_full[gj & 1], (gj >> 1) & 1, abort_flag)) return false;
          v_waited = j;
        }
        tc_fence_after();
        const uint32_t va = base + Cfg::kVOff + (gj & 1) * Cfg::kTileBytes;
        const uint32_t pa = tmem + (SEP ? Cfg::kPCol + t * (kPcTile / 2) : t * kPcTile);
#pragma unroll
        for (int kk = 0; kk < kPcTile / 16; ++kk)
          umma_ts(tmem + Cfg::kOCol + t * D, pa + kk * 8, smem_desc_sw128(va + kk * 16 * 128, kPcTile * 128, 1024),
                  idesc_o, (pv_unit[t] > 0 || kk > 0) ? 1u : 0u);
        if (SEP) umma_commit(&pv_done[t]);
        ++pv_unit[t];
        ++pv_total[t];
        return true;
      };
      if (ok && on(0, 0)) ok = issue_s(0, 0);
      if (ok && on(1, 0)) ok = issue_s(1, 0);
      for (int j = 0; ok && j < seg; ++j) {
        if constexpr (SEP) {
          if (ok && on(0, j + 1)) ok = issue_s(0, j + 1);
          if (ok && on(0, j)) ok = issue_pv(0, j);
          if (ok && on(1, j + 1)) ok = issue_s(1, j + 1);
          if (ok && on(1, j)) ok = issue_pv(1, j);
          if (ok) umma_commit(&kv_empty[(g + j) & 1]);
        } else {
          if (ok && on(0, j)) ok = issue_pv(0, j);
          if (ok && on(0, j + 1)) ok = issue_s(0, j + 1);
          if (ok && on(1, j)) ok = issue_pv(1, j);
          if (ok) umma_commit(&kv_empty[(g + j) & 1]);
          if (ok && on(1, j + 1)) ok = issue_s(1, j + 1);
        }
      }
      if (ok && k > 0) ok = mbar_wait_or_abort(epi_done, (k - 1) & 1, abort_flag);
      if (ok) umma_commit(o_done);
      g += seg;
      ++k;
      w.t += seg;
      w.local += seg;
      if (w.local == w.u.n && w.t < t_end) chunk_next(p, w);
    }
    umma_commit(drained);  // every product has completed before TMEM is freed
    mbar_wait(drained, 0);
  } else if (warp >= 2) {
    // ---------------- softmax: four warps a query tile, one thread a row ----------------
    const int t = (warp - 2) >> 2;
    const int quarter = warp & 3;         // TMEM lanes 32 * quarter .. +31
    const int row = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_addr = tmem + lane_off + t * kPcTile;
    const uint32_t o_addr = tmem + lane_off + Cfg::kOCol + t * D;
    const uint32_t p_addr = SEP ? tmem + lane_off + Cfg::kPCol + t * (kPcTile / 2) : s_addr;
    const int rt = row / p.a.G, rh = row - rt * p.a.G;  // the row's token in the tile, head in the group
    const float sc = p.a.scale_log2;
    int g = 0, k = 0, s_cnt = 0;
    int seg_index = 0;
    bool ok = true;
    while (ok && w.t < t_end) {
      const int seg = static_cast<int>(min(static_cast<long long>(w.u.n - w.local), t_end - w.t));
      const int cnt_tok = t ? w.u.c1 : w.u.c0;
      const int jb = max((t ? w.u.b1 : w.u.b0) - w.local, 0), je = min((t ? w.u.e1 : w.u.e0) - w.local, seg);
      const int first = (w.u.qb * 2 + t) * p.tpb;  // the tile's first token of the request
      const bool valid = rt < cnt_tok;             // (rows past tpb * G have rt >= tpb)
      const int pos = w.u.row.L + first + rt;
      const int pos0 = w.u.row.L + first, pos1 = pos0 + cnt_tok - 1;  // the tile's positions
      const int see_hi = min(pos, w.u.hi), see_lo = p.a.window >= 0 ? pos - p.a.window : 0;
      const bool warp_rows = __any_sync(0xffffffffu, valid);
      float m_used = -INFINITY, l = 0.f;
      int cnt = 0;
      for (int j = jb; j < je; ++j, ++cnt, ++s_cnt) {
        if (!__all_sync(0xffffffffu, mbar_wait_or_abort(&s_full[t], s_cnt & 1, abort_flag))) {
          ok = false;
          break;
        }
        tc_fence_after();
        const int kt = w.u.kb + (w.local + j) * kPcTile;  // the tile's first key
        if (kt < w.u.lo || kt + kPcTile - 1 > w.u.hi) {
          // rows of V outside [lo, hi] to zero, a thread a row
          const int gj = g + j;
          if (!__all_sync(0xffffffffu, mbar_wait_or_abort(&v_full[gj & 1], (gj >> 1) & 1, abort_flag))) {
            ok = false;
            break;
          }
          if (kt + row < w.u.lo || kt + row > w.u.hi) {
            const uint32_t at = base + Cfg::kVOff + (gj & 1) * Cfg::kTileBytes + row * 128;
#pragma unroll
            for (int c = 0; c < 8 * Cfg::kPanels; ++c)
              sts128(at + (c >> 3) * (kPcTile * 128) + (c & 7) * 16, make_uint4(0, 0, 0, 0));
          }
          fence_proxy_async_shared();
        }
        if (!warp_rows) {  // no query row in this warp's quarter: P may be anything
          if (SEP) mbar_arrive(&s_free[t]);
          if (SEP && cnt > 0 &&
              !__all_sync(0xffffffffu, mbar_wait_or_abort(&pv_done[t], (s_cnt - 1) & 1, abort_flag))) {
            ok = false;
            break;
          }
          tc_fence_before();
          mbar_arrive(&p_full[t]);
          continue;
        }
        const bool full = kt + kPcTile - 1 <= min(pos0, w.u.hi) && (p.a.window < 0 || pos1 - kt <= p.a.window);
        uint32_t sr[128];
        tmem_ld128(s_addr, sr);
        float alpha = 1.f, sum;
        bool redo = !full || __any_sync(0xffffffffu, valid && m_used == -INFINITY);
        if (!redo) {
          const uint64_t sc2 = pair_f32(sc, sc), nm2 = pair_f32(-m_used, -m_used);
          uint64_t acc0 = 0, acc1 = 0;
          float pmax = -INFINITY;  // of the polynomial's inputs
#pragma unroll
          for (int c = 0; c < 8; ++c) {  // 16 keys -> 8 words of P
#pragma unroll
            for (int u = 0; u < 8; ++u) {
              const uint64_t x = fma2(static_cast<uint64_t>(sr[16 * c + 2 * u]) |
                                          static_cast<uint64_t>(sr[16 * c + 2 * u + 1]) << 32,
                                      sc2, nm2);
              uint64_t e;
              if (u == 2 || u == 5 || u == 7) {  // three pairs of eight
                pmax = fmax3(pmax, lo_f(x), hi_f(x));
                e = exp2_poly_pair(x);
              } else {
                e = pair_f32(fast_exp2(lo_f(x)), fast_exp2(hi_f(x)));
              }
              if (u & 1) acc1 = add2(acc1, e);
              else acc0 = add2(acc0, e);
              sr[8 * c + u] = pack_bf16x2_rn(lo_f(e), hi_f(e));  // registers of scores already consumed
            }
          }
          acc0 = add2(acc0, acc1);
          sum = lo_f(acc0) + hi_f(acc0);
          redo = __any_sync(0xffffffffu, valid && !(sum < 1.2676506e30f && pmax < 100.f));  // 2^100
          if (redo) tmem_ld128(s_addr, sr);
        }
        if (redo) {
          if (!full) {
            // this row sees the columns [c_lo, c_hi): one unsigned compare a column
            const int c_hi = valid ? min(kPcTile, see_hi - kt + 1) : 0;
            const int c_lo = max(0, see_lo - kt);
            const uint32_t width = c_hi > c_lo ? static_cast<uint32_t>(c_hi - c_lo) : 0u;
#pragma unroll
            for (int c = 0; c < 128; ++c)
              if (static_cast<uint32_t>(c - c_lo) >= width) sr[c] = __float_as_uint(-INFINITY);
          }
          float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < 16; ++c)
#pragma unroll
            for (int u = 0; u < 4; ++u)
              m4[u] = fmax3(m4[u], __uint_as_float(sr[8 * c + 2 * u]), __uint_as_float(sr[8 * c + 2 * u + 1]));
          const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * sc;
          if (mx > m_used + 8.f) {
            alpha = fast_exp2(m_used - mx);  // 0 when m_used is -inf
            m_used = mx;
            l *= alpha;
          }
          const float neg_m = m_used == -INFINITY ? 0.f : -m_used;
          float s0 = 0.f, s1 = 0.f;
#pragma unroll
          for (int c = 0; c < 64; ++c) {
            const float e0 = fast_exp2(fmaf(__uint_as_float(sr[2 * c]), sc, neg_m));
            const float e1 = fast_exp2(fmaf(__uint_as_float(sr[2 * c + 1]), sc, neg_m));
            s0 += e0;
            s1 += e1;
            sr[c] = pack_bf16x2_rn(e0, e1);
          }
          sum = s0 + s1;
        }
        if constexpr (SEP) {
          // S is read; P's columns and O are free once the last product has completed
          tc_fence_before();
          mbar_arrive(&s_free[t]);
          if (cnt > 0) {
            if (!__all_sync(0xffffffffu, mbar_wait_or_abort(&pv_done[t], (s_cnt - 1) & 1, abort_flag))) {
              ok = false;
              break;
            }
            tc_fence_after();
          }
        }
#pragma unroll
        for (int c = 0; c < 4; ++c)
          tmem_st16_nowait(p_addr + 16 * c, *reinterpret_cast<const uint32_t(*)[16]>(&sr[16 * c]));
        l += sum;
        if (cnt > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld32(o_addr + c * 32, o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st32(o_addr + c * 32, o);
          }
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&p_full[t]);
      }
      if constexpr (SEP) {
        if (ok && cnt > 0 && !__all_sync(0xffffffffu, mbar_wait_or_abort(&pv_done[t], (s_cnt - 1) & 1, abort_flag)))
          ok = false;
      }
      if (ok && !__all_sync(0xffffffffu, mbar_wait_or_abort(o_done, k & 1, abort_flag))) ok = false;
      if (ok) {
        tc_fence_after();
        const bool complete = w.local == 0 && seg == w.u.n;
        const float inv = l == 0.f ? 0.f : 1.f / l;  // (a NaN stays one)
        const int tok = w.u.row.tok0 + first + rt;
        if (complete) {
          if (warp_rows) {
            uint16_t* dst = p.a.out + (static_cast<long long>(tok) * p.a.Hq + w.h * p.a.G + rh) * D;
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              tmem_ld32(o_addr + c * 32, o);
              if (valid)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  uint4 v;
                  v.x = pack_bf16x2(__uint_as_float(o[8 * e + 0]) * inv, __uint_as_float(o[8 * e + 1]) * inv);
                  v.y = pack_bf16x2(__uint_as_float(o[8 * e + 2]) * inv, __uint_as_float(o[8 * e + 3]) * inv);
                  v.z = pack_bf16x2(__uint_as_float(o[8 * e + 4]) * inv, __uint_as_float(o[8 * e + 5]) * inv);
                  v.w = pack_bf16x2(__uint_as_float(o[8 * e + 6]) * inv, __uint_as_float(o[8 * e + 7]) * inv);
                  *reinterpret_cast<uint4*>(dst + c * 32 + 8 * e) = v;
                }
            }
          }
        } else {
          const long long prow = (static_cast<long long>(blockIdx.x) * 2 + (seg_index ? 1 : 0)) * 256 + t * 128 + row;
          if (valid) p.a.part_lse[prow] = l == 0.f ? -INFINITY : m_used + __log2f(l);
          if (warp_rows && cnt > 0) {
            float* dst = p.a.part_o + prow * D;
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              tmem_ld32(o_addr + c * 32, o);
              if (valid)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  *reinterpret_cast<float4*>(dst + c * 32 + 4 * e) =
                      make_float4(__uint_as_float(o[4 * e]) * inv, __uint_as_float(o[4 * e + 1]) * inv,
                                  __uint_as_float(o[4 * e + 2]) * inv, __uint_as_float(o[4 * e + 3]) * inv);
            }
          }
          if (threadIdx.x == 64) {
            const long long start = w.t - w.local;
            if (share_owner(start, total, ng) == static_cast<int>(blockIdx.x)) {
              PagedCut c;
              c.tok0 = w.u.row.tok0 + w.u.qb * 2 * p.tpb;
              c.tok1 = c.tok0 + w.u.c0 + w.u.c1;
              c.h = w.h;
              c.g_last = share_owner(start + w.u.n - 1, total, ng);
              c.slot1 = seg_index ? 1 : 0;
              c.pad[0] = c.pad[1] = c.pad[2] = 0;
              p.cuts[blockIdx.x] = c;
            }
          }
        }
      }
      tc_fence_before();
      mbar_arrive(epi_done);  // O is read: the issuer may let the next unit's o_done complete
      g += seg;
      ++k;
      ++seg_index;
      w.t += seg;
      w.local += seg;
      if (w.local == w.u.n && w.t < t_end) chunk_next(p, w);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (p.wait_last) {  // the decode kernel has completed before anything after this kernel starts
    pdl_wait();
    pdl_launch_dependents();
  }
}

// Merges the units cut between CTAs: blockIdx.x is the CTA whose share the unit starts in,
// blockIdx.y and the warps divide its 256 rows.
template <int D>
__global__ void __launch_bounds__(256) paged_combine_kernel(const PagedChunkParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const PagedCut c = p.cuts[blockIdx.x];
  if (c.h < 0) return;
  const int rows = p.tpb * p.a.G;
  auto row_out = [&](int n) {
    const int rr = n & 127, tok = c.tok0 + (n >> 7) * p.tpb + rr / p.a.G;
    return p.a.out + (static_cast<long long>(tok) * p.a.Hq + c.h * p.a.G + rr % p.a.G) * D;
  };
  for (int n = blockIdx.y * 8 + (threadIdx.x >> 5); n < 256; n += gridDim.y * 8) {
    const int rr = n & 127;
    if (rr >= rows || c.tok0 + (n >> 7) * p.tpb + rr / p.a.G >= c.tok1) continue;
    paged_merge<D, 256>(p.a.part_o, p.a.part_lse, blockIdx.x, c.g_last, c.slot1 != 0, n, row_out);
  }
}

}  // namespace mcb
