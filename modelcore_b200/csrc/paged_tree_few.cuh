// paged_tree_attn for requests of few query rows a kv head (at most 32): the products with the keys on
// the M side of the tensor cores, so that what they and the softmax cost goes with the rows there are.
//
//   S^T (128 keys x R rows) = K_j Q^T          M=128 N=R K=D     (both from shared memory)
//   P^T                      = 2^(S^T scale - m)  a thread a key: R exponentials, stored for the next product
//   O^T (D x R rows) += V_j^T P^T              M=128 N=R K=128   (both from shared memory)
// with R = 16 or 32 rows, token * G + head, of one *unit* (request, R / G tokens, kv head).  The tiles of
// all units are one sequence that the CTAs share evenly, as in the kernel beside this one, whose walk, masks and
// descriptions these are; a cut unit's last contributor merges it.  A tile of K and V, 64 KB at head size 128, has some 2,100 cycles at HBM's rate;
// with the rows on the M side it took 1,280 of the tensor cores whatever the rows, and the exponentials of 16
// rows fell to one warp.
//
// Roles: warps 0 and 3 producers of K (and queries, descriptions) and V; warp 1 issues S^T, warp 2 O^T, in the
// tiles' order; warps 4-7 and 8-11 are two softmax groups that take the tiles in turn, each with its own S^T,
// P^T, O^T, references m and sums, merged at a unit's end.  TMEM: S^T and O^T of both, 4 R columns.
//
// A row's m is what its first tile's maximum was and moves where a score exceeds it by 2^8: the
// threads hold a key each, so a maximum over keys is a reduction over the group (a butterfly that
// leaves each lane one row), taken only then and in a part's first tile.  The group agrees on that in one
// meeting a tile.  l is summed a thread a row and reduced over the keys at the end.
//
// Measured, back to back in a graph: 32 requests of 8,192 with 4 tokens of 16/4 heads of 128 (16 rows) 91 us, 5.9
// TB/s; 32 of 4,096 with one token of 12/12 heads of 64 80 us, 5.0 TB/s, with 16 tokens 84 (the rows on the other
// side of the products: 104 and 117).  3 requests of 8 tokens of 12/12 heads of 64 at 1,000: 15.2 us, latency: launch
// and lengths 4, a tile's maximum and masks 4, sums and way out 3.  With 64 rows the registers for them spill or
// the scores are read twice, and it is no faster than the other kernel (148 against 112 us at head size 64).
#pragma once

#include "paged_tree.cuh"

namespace mcb {

template <int D, int R>
struct TreeFewConfig {
  static constexpr int kPanels = D / 64;
  static constexpr int kTileBytes = kPanels * kPtTile * 128;
  static constexpr int kQBytes = kPanels * R * 128;
  static constexpr int kPBytes = kPtTile * R * 2;
  // what 226 KB hold beside two query tiles and two P^T: 6 tiles at head size 128, 12 at 64
  static constexpr int kK = D == 128 ? 3 : 5, kV = D == 128 ? 3 : 7;
  static constexpr int kStages = kK + kV;
  static constexpr int kRingOff = 0;
  static constexpr int kQOff = kRingOff + kStages * kTileBytes;
  static constexpr int kPOff = kQOff + 2 * kQBytes;
  static constexpr int kBarOff = kPOff + 2 * kPBytes;
  static constexpr int kNumBars = 2 * kStages + 23;
  static constexpr int kSegOff = (kBarOff + kNumBars * 8 + 32 + 63) / 64 * 64;
  static constexpr int kRowOff = kSegOff + 4 * 64;       // R tokens' {see_lo, see_hi, pos}
  static constexpr int kRefOff = kRowOff + R * 12;       // [2][R] -m of either group
  static constexpr int kVoteOff = kRefOff + 2 * R * 4;   // [2][2][4] what a group's warps vote
  static constexpr int kBytes = kVoteOff + 64 + 1024;
  // above half of an SM's shared memory: one CTA an SM
  static_assert(kBytes > 118784 && kBytes <= 232448, "one CTA an SM");
  static constexpr uint32_t kTmemCols = 4 * R;
};

// Shared-memory descriptor of an MN-major tile of R values a row: the swizzle is as wide as the row (64 or 32 bytes).
template <int R>
__device__ __forceinline__ uint64_t smem_desc_rows(uint32_t addr) {
  constexpr uint64_t mode = R == 32 ? 4 : 6;
  return static_cast<uint64_t>((addr >> 4) & 0x3fffu) | (static_cast<uint64_t>((R * 16) >> 4) << 16) |
         (static_cast<uint64_t>((R * 16) >> 4) << 32) | (1ull << 46) | (mode << 61);
}
// The 16-byte chunk's place in such a row.
template <int R>
__device__ __forceinline__ uint32_t row_chunk(int row, int chunk) {
  constexpr int wide = R * 2 / 16;  // chunks a row
  return static_cast<uint32_t>(row * R * 2 + ((chunk ^ (row / (8 / wide) & (wide - 1))) << 4));
}

// The -m of a row that has no m yet: a -0, which leaves scores as they are and which no m's negative is.
constexpr float kNoRef = -0.f;
__device__ __forceinline__ bool no_ref(float neg_m) { return __float_as_uint(neg_m) == 0x80000000u; }

// Over the warp's lanes, of 32 values a lane: lane i gets the reduction of every lane's v[i].
template <typename F>
__device__ __forceinline__ float warp_transpose_reduce(float (&v)[32], F f) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float send = up ? v[i] : v[i + o], keep = up ? v[i + o] : v[i];
      v[i] = f(keep, __shfl_xor_sync(0xffffffffu, send, o));
    }
  }
  return v[0];
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
template <int R>
__device__ __forceinline__ void tmem_ld_rows(uint32_t taddr, uint32_t (&r)[R]) {
  if constexpr (R == 32) tmem_ld32(taddr, r);
  else tmem_ld16(taddr, r);
}

// Which rows see key c, which is in the unit's [lo, hi].  `tokens`: see_lo, see_hi and pos of each of the unit's n,
// of which `tok` is the first; the request's are T from tok0 on, after L cached ones.  (Arguments by value: what
// has an address lives in local memory, and shared memory leaves the L1 cache next to nothing to keep it.)
__device__ __noinline__ uint64_t tree_row_bits(const PagedTreeParams& p, const int* tokens, int n, int tok, int tok0, int L,
                                               int T, int c) {
  const int j = c - L, G = p.a.G;
  const uint64_t heads = ~0ull >> (64 - G);
  uint64_t bits = 0;
  if (j < 0 || T > 32 * p.words) {
    for (int i = 0; i < n; ++i)
      if (c >= tokens[i * 3] && c <= tokens[i * 3 + 1]) bits |= heads << (i * G);
    return bits;
  }
  // a tree's new token: by the masks, eight tokens' words on their way at once
  const int kpos = p.a.window >= 0 ? max(p.positions[tok0 + j], L) : 0;
  const uint32_t* word = p.mask + static_cast<long long>(tok) * p.words + (j >> 5);
  constexpr int U = 8;
  for (int i0 = 0; i0 < n; i0 += U) {
    uint32_t w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = word[min(i0 + u, n - 1) * p.words];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u;
      if (i < n && (w[u] >> (j & 31) & 1) && (p.a.window < 0 || tokens[i * 3 + 2] - kpos <= p.a.window))
        bits |= heads << (i * G);
    }
  }
  return bits;
}

template <int D, int R>
__global__ void __launch_bounds__(kPtThreads, 1)
    paged_tree_few_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                          const __grid_constant__ CUtensorMap vmap, const __grid_constant__ PagedTreeParams p) {
  using Cfg = TreeFewConfig<D, R>;
  constexpr int SK = Cfg::kK, SV = Cfg::kV, ST = SK + SV, C = R;  // C rows at a time
  static_assert(R == 16 || R == 32, "a lane a row");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::kBarOff);
  uint64_t* full = bars;             // [ST] K of key tile g at g mod SK, V at SK + g mod SV
  uint64_t* empty = full + ST;       // [ST]
  uint64_t* q_full = empty + ST;     // [2] part k's queries are in place k mod 2
  uint64_t* q_empty = q_full + 2;    // [2]
  uint64_t* s_full = q_empty + 2;    // [2] a group
  uint64_t* s_free = s_full + 2;     // [2] 4 arrivals: S^T has been read
  uint64_t* p_full = s_free + 2;     // [2] 128 arrivals
  uint64_t* pv_done = p_full + 2;    // [2]
  uint64_t* v_ready = pv_done + 2;   // [2] a tile's values have landed, told for tiles with keys outside [lo, hi]
  uint64_t* epi_done = v_ready + 2;  // 256 arrivals: a part's O^T have been read
  uint64_t* seg_full = epi_done + 1; // [4] a description is there
  uint64_t* meet = seg_full + 4;     // [2] 4 arrivals: a group's warps (an mbarrier's wait is bounded, a barrier's not)
  uint64_t* meet_all = meet + 2;     // 8 arrivals: both groups'
  uint64_t* drained = meet_all + 1;  // 2 arrivals
  static_assert(2 * ST + 23 == Cfg::kNumBars, "the barriers above");
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + Cfg::kNumBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* ctl = reinterpret_cast<int*>(tmem_slot + 2);  // start: r, qb, h, local
  TreeSeg* segs = reinterpret_cast<TreeSeg*>(smem + Cfg::kSegOff);
  int* tokens = reinterpret_cast<int*>(smem + Cfg::kRowOff);
  float* ref = reinterpret_cast<float*>(smem + Cfg::kRefOff);
  long long* warp_tot = reinterpret_cast<long long*>(smem + Cfg::kPOff);  // [12], before the roles begin
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < Cfg::kNumBars; ++i) {
      uint64_t* b = bars + i;
      const bool four = (b >= s_free && b < p_full) || (b >= meet && b < meet_all);
      mbar_init(b, four ? 4 : b >= p_full && b < pv_done ? 128 : b == epi_done ? 256 : b == meet_all ? 8 : b == drained ? 2 : 1);
    }
    *abort_flag = 0;
    fence_mbarrier_init();
    prefetch_tensormap(&qmap);
    prefetch_tensormap(&kmap);
    prefetch_tensormap(&vmap);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, Cfg::kTmemCols);
    tmem_relinquish();
  }
  pdl_wait();
  pdl_launch_dependents();

  // ---- the sequence's length and this CTA's first tile ----
  tc_fence_before();
  TreeWalk w;
  const TreeShare share = tree_place(p, w, warp_tot, ctl);
  tc_fence_after();
  const long long t_begin = share.t_begin, t_end = share.t_end;
  const uint32_t tmem = *tmem_slot;
  const uint32_t base = smem_u32(smem);
  auto wait = [&](uint64_t* bar, uint32_t parity) {  // warp-uniform
    return __all_sync(0xffffffffu, mbar_wait_small(bar, parity, abort_flag)) != 0;
  };
  // the x-th description, once it is there; false on a timeout
  auto next_seg = [&](int x, TreeSeg& d) {
    if (!wait(&seg_full[x & 3], (x >> 2) & 1)) return false;
    const int4* src = reinterpret_cast<const int4*>(&segs[x & 3]);
    int4* dst = reinterpret_cast<int4*>(&d);
#pragma unroll
    for (int i = 0; i < 4; ++i) dst[i] = src[i];
    return true;
  };

  if (warp == 0 || warp == 3) {
    // ---------------- producers: of K, the queries and the descriptions; of V ----------------
    const int kv = warp == 3;
    const CUtensorMap* map = kv ? &vmap : &kmap;
    const uint64_t policy = l2_policy_evict_first();
    const int box_shift = min(p.a.page_shift, 7);  // positions a box: min(page, 128)
    const int box = 1 << box_shift, nch = kPtTile >> box_shift;
    const uint32_t box_bytes = static_cast<uint32_t>(box) * 128u;
    const uint32_t q_bytes = static_cast<uint32_t>(p.a.tpb * p.a.G) * 128u;
    const int lch = lane / Cfg::kPanels, lpn = lane % Cfg::kPanels;
    const uint32_t lane_dst = Cfg::kRingOff + lpn * kPtTile * 128 + lch * box_bytes;
    uint32_t gt = 0;  // key tiles so far
    int k = 0;        // parts so far
    bool ok = true;
    while (ok && w.t < t_end) {
      const int seg = static_cast<int>(min(static_cast<long long>(w.u.n - w.local), t_end - w.t));
      const int32_t* table = p.a.block_table + w.u.r * p.a.table_stride;
      // lane l holds the page of chunk pbase + l; the next 32 are on their way
      int pg = 0, pg_next = 0;
      bool in_next = false;
      auto page_at = [&](int c) {
        const long long key = static_cast<long long>(c + lane) << box_shift;
        in_next = key <= w.u.hi && key + box > w.u.lo;
        return in_next ? table[key >> p.a.page_shift] : 0;
      };
      const int c_first = (w.u.kb + w.local * kPtTile) >> box_shift;
      pg_next = page_at(c_first);
      int pbase = c_first - 32;
      if (!kv) {
        if (k > 1 && !(ok = wait(&q_empty[k & 1], ((k >> 1) - 1) & 1))) break;
        if (lane == 0) {
          const bool whole = w.local == 0 && seg == w.u.n;
          TreeSeg d;
          d.seg = seg;
          d.kt0 = w.u.kb + w.local * kPtTile;
          d.lo = w.u.lo;
          d.hi = w.u.hi;
          d.L = w.u.row.L;
          d.T = w.u.row.T;
          d.tok0 = w.u.row.tok0;
          d.first = w.u.qb * p.a.tpb;
          d.c0 = w.u.c0;
          d.c1 = 0;
          d.h = w.h;
          d.part = whole ? -1 : k > 0 ? 1 : 0;
          d.last = w.t + seg >= t_end;
          d.q = d.pad[0] = d.pad[1] = 0;
          if (!whole) tree_owners(share, w, d.pad[0], d.pad[1], d.q);
          segs[k & 3] = d;
          mbar_arrive(&seg_full[k & 3]);
          mbar_arrive_expect_tx(&q_full[k & 1], Cfg::kPanels * q_bytes);
#pragma unroll
          for (int pn = 0; pn < Cfg::kPanels; ++pn)
            tma_load_3d(smem + Cfg::kQOff + (k & 1) * Cfg::kQBytes + pn * R * 128, &qmap, &q_full[k & 1], pn * 64,
                        w.h * p.a.G, d.tok0 + d.first, policy);
        }
        __syncwarp();
      }
      ++k;
      for (int i = 0; i < seg; ++i, ++gt) {
        const int c0 = c_first + i * nch;
        if (c0 + nch > pbase + 32) {
          pbase = c0;
          pg = pg_next;
          if (pg < 0 || pg >= p.a.n_pages) {
            if (in_next) record_error(kErrPageOutOfRange);
            pg = p.a.n_pages;  // outside the pool: a box there reads zeros
          }
          pg_next = page_at(c0 + 32);
        }
        // a lane a box: chunk lch, panel lpn of the tile's, those with visible keys
        const int key0 = (c0 + lch) << box_shift;
        const bool load = lch < nch && key0 <= w.u.hi && key0 > w.u.lo - box;
        const int row = __shfl_sync(0xffffffffu, pg, (c0 - pbase + lch) & 31) * p.a.Hkv + w.h;
        const int pos = key0 & ((1 << p.a.page_shift) - 1);
        const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, load)) * box_bytes;
        const uint32_t st = kv ? SK + gt % SV : gt % SK, turn = kv ? gt / SV : gt / SK;
        if (turn > 0 && !(ok = wait(&empty[st], (turn - 1) & 1))) break;
        if (lane == 0) mbar_arrive_expect_tx(&full[st], bytes);
        __syncwarp();
        if (load) tma_load_4d(smem + lane_dst + st * Cfg::kTileBytes, map, &full[st], 0, pos, lpn, row, policy);
        __syncwarp();
      }
      if (!ok) break;
      w.t += seg;
      w.local += seg;
      if (w.local == w.u.n && w.t < t_end) tree_next(p, w);
    }
    if (*abort_flag && lane == 0) {  // the copies in flight land before the CTA can exit
      const uint32_t n = kv ? SV : SK;
      for (uint32_t f = gt > n ? gt - n : 0; f < gt; ++f) mbar_wait(&full[(kv ? SK : 0) + f % n], (f / n) & 1);
      for (int x = kv ? k : max(k - 2, 0); x < k; ++x) mbar_wait(&q_full[x & 1], (x >> 1) & 1);
    }
    __syncwarp();
  } else if (warp < 3) {
    // ---------------- product issuers: S^T, O^T ----------------
    constexpr uint32_t idesc_s = umma_idesc_bf16(128, R, 0);
    constexpr uint32_t idesc_o = umma_idesc_bf16(128, R, 1) | 1u << 15;  // A and B both MN-major
    tree_fill(p.a, D, threadIdx.x - 32, 64);
    const bool pv = __shfl_sync(0xffffffffu, warp, 0) == 2;
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const uint64_t q0_desc = smem_desc_sw128(base + Cfg::kQOff, 16, 1024);
    const uint64_t k0_desc = smem_desc_sw128(base + Cfg::kRingOff, 16, 1024);
    // (head size 64: the M side's upper 64 rows are other keys' values, into lanes that nothing reads)
    const uint64_t v0_desc = smem_desc_sw128(base + Cfg::kRingOff, D == 128 ? kPtTile * 128 : 64 * 128, 1024);
    const uint64_t p0_desc = smem_desc_rows<R>(base + Cfg::kPOff);
    uint32_t g = 0, uses[2] = {0, 0};  // key tiles so far; the groups'
    bool ok = true;
    TreeSeg d;
    d.last = t_begin >= t_end;
    for (int k = 0; ok && !d.last; ++k) {
      if (!(ok = next_seg(k, d))) break;
      if (!pv) ok = wait(&q_full[k & 1], (k >> 1) & 1);
#pragma unroll 1
      for (int j = 0; ok && j < d.seg; ++j, ++g) {
        const int t = __shfl_sync(0xffffffffu, j & 1, 0);
        const uint32_t n = t ? uses[1] : uses[0];  // the group's tiles before
        if (!pv) {
          const uint32_t st = __shfl_sync(0xffffffffu, g % SK, 0);
          if (!(ok = wait(&full[st], (g / SK) & 1))) break;
          if (n > 0 && !(ok = wait(&s_free[t], (n - 1) & 1))) break;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t ka = k0_desc + st * (Cfg::kTileBytes >> 4), qa = q0_desc + (k & 1) * (Cfg::kQBytes >> 4);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
              umma_ss(tm + t * R, ka + (kk >> 2) * ((kPtTile * 128) >> 4) + (kk & 3) * (32 >> 4),
                      qa + (kk >> 2) * ((R * 128) >> 4) + (kk & 3) * (32 >> 4), idesc_s, kk > 0 ? 1u : 0u);
            umma_commit(&s_full[t]);
            umma_commit(&empty[st]);
            if (j == d.seg - 1) umma_commit(&q_empty[k & 1]);
          }
        } else {
          const uint32_t st = __shfl_sync(0xffffffffu, SK + g % SV, 0);
          if (!(ok = wait(&full[st], (g / SV) & 1))) break;
          const int kt = d.kt0 + j * kPtTile;
          if ((kt < d.lo || kt + kPtTile - 1 > d.hi) && lane == 0) mbar_arrive(&v_ready[t]);
          if (!(ok = wait(&p_full[t], n & 1))) break;
          // (a part's first products overwrite O^T: the last part's have been read)
          if (j < 2 && k > 0 && !(ok = wait(epi_done, (k - 1) & 1))) break;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t va = v0_desc + st * (Cfg::kTileBytes >> 4), pa = p0_desc + t * (Cfg::kPBytes >> 4);
#pragma unroll
            for (int kk = 0; kk < kPtTile / 16; ++kk)
              umma_ss(tm + (2 + t) * R, va + kk * ((16 * 128) >> 4), pa + kk * ((16 * R * 2) >> 4), idesc_o,
                      kk > 0 || j > 1 ? 1u : 0u);
            umma_commit(&empty[st]);
            umma_commit(&pv_done[t]);
          }
        }
        __syncwarp();
        uses[0] += t == 0;
        uses[1] += t;
      }
    }
    if (elect_one()) umma_commit(drained);  // every product has completed before TMEM is freed
    __syncwarp();
    mbar_wait(drained, 0);
    __syncwarp();
  } else {
    // ---------------- softmax: two groups of four warps, a thread a key ----------------
    const int t = (warp - 4) >> 2, quarter = warp & 3;  // group; TMEM lanes 32 * quarter .. +31
    const int key = quarter * 32 + lane;                // of the tile; and at the end the row of O^T
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_addr = tmem + lane_off + t * R, o_addr = tmem + lane_off + 2 * R;
    const float sc = p.a.scale_log2;
    int* votes = reinterpret_cast<int*>(smem + Cfg::kVoteOff) + t * 8;
    volatile int* merge = ctl;                          // whether this CTA merges a cut unit
    uint8_t* p_tile = smem + Cfg::kPOff + t * Cfg::kPBytes;
    float* wred = reinterpret_cast<float*>(p_tile);     // [4][R] while no product reads P^T
    float* delta = wred + 4 * R;                        // [R]
    float* neg_m = ref + t * R;
    uint32_t g = 0, n = 0, edges = 0;                   // key tiles so far, this group's, those at an edge
    uint32_t met = 0, met_all = 0;
    bool ok = true;
    // The group meets, and learns whether any of its threads has v set.  (Two slots of votes: one is written
    // again when all have passed the next meeting, so have read it.)
    auto group_any = [&](bool v) {
      const bool any = __any_sync(0xffffffffu, v);
      __syncwarp();  // (a vote orders no memory: lane 0's arrival is to release all lanes' stores)
      if (lane == 0) {
        votes[(met & 1) * 4 + quarter] = any;
        mbar_arrive(&meet[t]);
      }
      ok = wait(&meet[t], met & 1) && ok;
      const uint4 all = lds128(smem_u32(votes + (met & 1) * 4));
      ++met;
      return (all.x | all.y | all.z | all.w) != 0;
    };
    auto all_meet = [&] {
      __syncwarp();
      if (lane == 0) mbar_arrive(meet_all);
      ok = wait(meet_all, met_all++ & 1) && ok;
    };
    TreeSeg d;
    d.last = t_begin >= t_end;
    for (int k = 0; ok && !d.last; ++k) {
      if (!(ok = next_seg(k, d))) break;
      const bool causal = d.T > 32 * p.words;
      // what the tokens see of the cached keys (a chunk's: of all)
      const int i = threadIdx.x - 128;
      if (i < d.c0) {
        const int pos = causal ? d.L + d.first + i : max(p.positions[d.tok0 + d.first + i], d.L);
        tokens[i * 3] = p.a.window >= 0 ? max(pos - p.a.window, 0) : 0;
        tokens[i * 3 + 1] = min(causal ? pos : d.L - 1, d.hi);
        tokens[i * 3 + 2] = pos;
      }
      all_meet();
      if (!ok) break;
      // keys in [all_lo, all_hi] are seen by every row that there is
      int all_lo = 0, all_hi = d.hi;
      for (int x = lane; x < d.c0; x += 32) {
        all_lo = max(all_lo, tokens[x * 3]);
        all_hi = min(all_hi, tokens[x * 3 + 1]);
      }
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) {
        all_lo = max(all_lo, __shfl_xor_sync(0xffffffffu, all_lo, o));
        all_hi = min(all_hi, __shfl_xor_sync(0xffffffffu, all_hi, o));
      }
      float l[R];
#pragma unroll
      for (int r = 0; r < R; ++r) l[r] = 0.f;
      bool unsettled = true;  // some row has no m yet
      int tiles = 0;          // this group's, of the part
      for (int j = t; j < d.seg; j += 2, ++tiles, ++n) {
        const int kt = d.kt0 + j * kPtTile, c = kt + key;
        const bool plain = kt >= all_lo && kt + kPtTile - 1 <= all_hi;
        uint64_t bits = 0;
        if (!plain) {
          if (kt < d.lo || kt + kPtTile - 1 > d.hi) {
            // rows of V outside [lo, hi] to zero, a thread a row
            if (!(ok = wait(&v_ready[t], edges++ & 1))) break;
            if (c < d.lo || c > d.hi) {
              const uint32_t at = base + Cfg::kRingOff + (SK + (g + j) % SV) * Cfg::kTileBytes + key * 128;
#pragma unroll
              for (int x = 0; x < 8 * Cfg::kPanels; ++x)
                sts128(at + (x >> 3) * (kPtTile * 128) + (x & 7) * 16, make_uint4(0, 0, 0, 0));
            }
            fence_proxy_async_shared();
          }
          if (c >= d.lo && c <= d.hi) bits = tree_row_bits(p, tokens, d.c0, d.tok0 + d.first, d.tok0, d.L, d.T, c);
        }
        if (!(ok = wait(&s_full[t], n & 1))) break;
        tc_fence_after();
        // C rows' scores, less their m: -inf where the row does not see the key
        auto scores = [&](int r0, bool bare, float(&x)[C]) {
          uint32_t s[C];
          tmem_ld_rows<C>(s_addr + r0, s);
#pragma unroll
          for (int r = 0; r < C; r += 4) {
            const float4 m4 = bare ? make_float4(0.f, 0.f, 0.f, 0.f) : *reinterpret_cast<const float4*>(neg_m + r0 + r);
            x[r] = fmaf(__uint_as_float(s[r]), sc, m4.x);
            x[r + 1] = fmaf(__uint_as_float(s[r + 1]), sc, m4.y);
            x[r + 2] = fmaf(__uint_as_float(s[r + 2]), sc, m4.z);
            x[r + 3] = fmaf(__uint_as_float(s[r + 3]), sc, m4.w);
          }
          if (!plain) {
            const uint32_t seen = static_cast<uint32_t>(bits >> r0);
#pragma unroll
            for (int r = 0; r < C; ++r)
              if (!(seen >> r & 1)) x[r] = -INFINITY;
          }
        };
        bool far = false;
        if (!unsettled) {
          float top = -INFINITY;
#pragma unroll
          for (int r0 = 0; r0 < R; r0 += C) {
            float x[C];
            scores(r0, false, x);
#pragma unroll
            for (int r = 0; r < C; r += 2) top = fmax3(top, x[r], x[r + 1]);
          }
          far = top > 8.f;
        }
        // P^T of this group's last tile has been read: the meeting tells the group
        if (n > 0 && !(ok = wait(&pv_done[t], (n - 1) & 1))) break;
        tc_fence_after();
        if (!unsettled) far = group_any(far);  // (unsettled is the group's)
        if (!ok) break;
        if (__builtin_expect(far || unsettled, 0)) {
          // the rows' maxima over the tile, less their m
#pragma unroll 1
          for (int r0 = 0; r0 < R; r0 += C) {
            float x[C], v[32];
            scores(r0, tiles == 0, x);
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = i < C ? x[i % C] : -INFINITY;
            const float mx = warp_transpose_reduce(v, [](float a, float b) { return fmaxf(a, b); });
            if (lane < C) wred[quarter * R + r0 + lane] = mx;
          }
          group_any(false);
          if (key < R) {
            const float mx = fmaxf(fmaxf(wred[key], wred[R + key]), fmaxf(wred[2 * R + key], wred[3 * R + key]));
            const float old = tiles == 0 ? kNoRef : neg_m[key];
            float move = 0.f, to = old;
            if (mx > -INFINITY && (no_ref(old) || mx > 8.f)) {
              move = mx;
              to = (no_ref(old) ? 0.f : old) - mx;  // (never -0)
            } else if (key >= d.c0 * p.a.G) {
              to = 0.f;  // no row: it waits for none
            }
            delta[key] = move;
            neg_m[key] = to;
          }
          group_any(false);
          if (!ok) break;
          bool none = false, scale = false;
#pragma unroll
          for (int r = 0; r < R; ++r) {
            none |= no_ref(neg_m[r]);  // a row that has seen nothing, or nothing but NaN
            const float by = delta[r];
            if (by != 0.f && tiles > 0) {
              scale = true;
              if (l[r] != 0.f) l[r] *= fast_exp2(-by);  // (0: nothing seen so far, and by may be anything)
            }
          }
          unsettled = none;
          if (scale) {  // (by the same numbers in all threads: converged)
#pragma unroll 1
            for (int r0 = 0; r0 < R; r0 += 16) {
              uint32_t o[16];
              tmem_ld16(o_addr + t * R + r0, o);
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float by = delta[r0 + i], v = __uint_as_float(o[i]);
                if (by != 0.f && v != 0.f) o[i] = __float_as_uint(v * fast_exp2(-by));
              }
              tmem_st16_nowait(o_addr + t * R + r0, o);
            }
            tmem_st_wait();
          }
          group_any(false);  // wred and delta are P^T again
          if (!ok) break;
        }
#pragma unroll
        for (int r0 = 0; r0 < R; r0 += C) {
          float x[C];
          scores(r0, false, x);
#pragma unroll
          for (int r = 0; r < C; r += 8) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float e0 = fast_exp2(x[r + 2 * i]), e1 = fast_exp2(x[r + 2 * i + 1]);
              l[r0 + r + 2 * i] += e0;
              l[r0 + r + 2 * i + 1] += e1;
              w[i] = pack_bf16x2_rn(e0, e1);
            }
            *reinterpret_cast<uint4*>(p_tile + row_chunk<R>(key, (r0 + r) >> 3)) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free[t]);  // S^T may be overwritten
        fence_proxy_async_shared();
        tc_fence_before();
        mbar_arrive(&p_full[t]);
      }
      if (!ok) break;
      if (tiles > 0 && !(ok = wait(&pv_done[t], (n - 1) & 1))) break;
      tc_fence_after();
      // ---- the sums over the keys, the weights of both groups' O^T, and out ----
      group_any(false);  // (every warp has seen the last product: wred is free)
      if (!ok) break;
#pragma unroll
      for (int r0 = 0; r0 < R; r0 += 32) {
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = i < R ? l[(r0 + i) % R] : 0.f;
        const float sum = warp_transpose_reduce(v, [](float a, float b) { return a + b; });
        if (lane < R) wred[quarter * R + r0 + lane] = sum;
      }
      tc_fence_before();
      all_meet();
      if (!ok) break;
      tc_fence_after();
      const long long slot = static_cast<long long>(blockIdx.x) * 2 + d.part;
      const bool two = d.seg > 1;
      const int rows = d.c0 * p.a.G;
      // a lane a row: both groups' sums and weights, by every warp for itself
      float w0 = 0.f, w1 = 0.f;
      {
        const int r = lane < R ? lane : 0;
        const float* red0 = reinterpret_cast<const float*>(smem + Cfg::kPOff);
        const float* red1 = reinterpret_cast<const float*>(smem + Cfg::kPOff + Cfg::kPBytes);
        const float l0 = (red0[r] + red0[R + r]) + (red0[2 * R + r] + red0[3 * R + r]);
        const float l1 = two ? (red1[r] + red1[R + r]) + (red1[2 * R + r] + red1[3 * R + r]) : 0.f;
        const float m0 = no_ref(ref[r]) ? -INFINITY : -ref[r];
        const float m1 = !two || no_ref(ref[R + r]) ? -INFINITY : -ref[R + r], m = fmaxf(m0, m1);
        // (no m: nothing seen, or NaN alone, and then l is one)
        const float f0 = m0 == -INFINITY ? (l0 == 0.f ? 0.f : l0) : fast_exp2(m0 - m);
        const float f1 = m1 == -INFINITY ? (l1 == 0.f ? 0.f : l1) : fast_exp2(m1 - m);
        const float all = (f0 == 0.f ? 0.f : l0 * f0) + (f1 == 0.f ? 0.f : l1 * f1);
        const float inv = all == 0.f ? 0.f : 1.f / all;
        w0 = all != all ? all : f0 * inv;
        w1 = all != all ? all : f1 * inv;
        if (d.part >= 0 && warp == 4 && lane < rows)
          p.a.part_lse[slot * R + lane] = all == 0.f ? -INFINITY : all != all ? all : m + __log2f(all);
      }
      if (quarter * 32 < D) {  // a group half of the rows, a thread a column of the output
        const int half = t * (R / 2);
        int head = half % p.a.G;  // of the group
        uint16_t* out = p.a.out + (static_cast<long long>(d.tok0 + d.first + half / p.a.G) * p.a.Hq + d.h * p.a.G + head) * D + key;
        float* part = p.a.part_o + (slot * R + half) * D + key;
        const long long next_token = static_cast<long long>(p.a.Hq - p.a.G) * D;
#pragma unroll 1
        for (int r0 = half; r0 < half + R / 2 && r0 < rows; r0 += 8) {
          uint32_t a[16], b[16];  // (16 columns, 8 of them for this turn)
          tmem_ld16(o_addr + (r0 & ~15), a);
          if (two) tmem_ld16(o_addr + R + (r0 & ~15), b);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = r0 + i;
            const float u0 = __shfl_sync(0xffffffffu, w0, r), u1 = __shfl_sync(0xffffffffu, w1, r);
            const uint32_t av = r0 & 8 ? a[i + 8] : a[i], bv = r0 & 8 ? b[i + 8] : b[i];
            float o = u0 == 0.f ? 0.f : __uint_as_float(av) * u0;
            if (two && u1 != 0.f) o = fmaf(__uint_as_float(bv), u1, o);
            if (r < rows) {
              if (d.part >= 0) *part = o;
              else *out = float_to_bf16_bits(o);
            }
            part += D;
            out += D;
            if (++head == p.a.G) {
              head = 0;
              out += next_token;
            }
          }
        }
      }
      tc_fence_before();
      mbar_arrive(epi_done);  // O^T are read: they may be overwritten
      g += d.seg;
      if (d.part >= 0) {
        // The contributor that arrives last merges all partials, a warp a row (a kernel after this one for it cost
        // a small call 4 us of 19).  The meeting orders every thread's stores before the counter's release.
        all_meet();
        if (!ok) break;
        if (warp == 4 && lane == 0) {
          int* counter = p.a.counters + d.pad[0];
          const bool last = atom_add_acq_rel_gpu(counter, 1) == d.pad[1] - d.pad[0];
          if (last) *counter = 0;  // every contributor has arrived: ready for the next call
          *merge = last;
        }
        all_meet();
        if (!ok) break;
        if (*merge)
          for (int n = warp - 4; n < rows; n += 8)
            paged_merge<D, R>(p.a.part_o, p.a.part_lse, d.pad[0], d.pad[1], d.q, n, [&](int r) {
              return p.a.out +
                     (static_cast<long long>(d.tok0 + d.first + r / p.a.G) * p.a.Hq + d.h * p.a.G + r % p.a.G) * D;
            });
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, Cfg::kTmemCols);
  }
}

}  // namespace mcb
