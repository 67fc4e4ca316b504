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
// Roles of a CTA's warps:
//   warp 0      TMA producer and walker: describes each unit (or the part of one in this CTA's share)
//               in shared memory for the other roles, loads Q0, Q1, then K_j and V_j into rings of
//               two that run on across units, one box a (page chunk, 64-column panel)
//   warps 1, 2  (warp 1 allocates TMEM) products of Q0, of Q1, by halves h of a key tile
//                 S_th = Q_t K_jh^T     M=128 N=64 K=D   (both operands from shared memory)
//                 O_t += P_th V_jh      M=128 N=D K=64   (P from TMEM)
//   warps 4-11  softmax of Q0, warps 12-19 of Q1: two threads a query row, one a half of the keys
// TMEM: four S_th of 64 columns (the bf16 P_th is written over its S_th), O0, O1 (D columns each): all
// 512 columns at D = 128.  A half is a chain of its own, S -> softmax -> P V -> next S, and the four
// chains take turns on the tensor cores, so the softmax of three runs while a fourth's products do.
// With whole tiles (N = 128, two chains) a chain's softmax had to fit beside one other chain's
// products, which it does not (1,600 cycles against 1,024), and both then waited: 3,700 cycles a key
// tile where the products take 2,048.  N = 64 costs the tensor cores a quarter more (S reads Q from
// shared memory once for 64 keys: 384 cycles for 256 worth) and the rest overlaps: 2,560 of some 3,300.
// Measured, 16/4 heads of 128, as called (and back to back in a graph): 8,192 tokens after 8,192 766 us
// (741), 1,077 TFLOP/s at the 1.45 GHz that the power limit leaves; five chunks of 2,041 under a window of
// 1,024 124 us (118), 574 TFLOP/s -- nine key tiles a unit there, and a unit costs some 12,000 cycles beside
// its tiles: the first tile's maximum and the masks at both ends (5,500), the last product and O's way out
// (6,000).  96 registers a thread, the most that 640 threads allow, with 48 bytes spilled (44 at head size
// 64) around the rare branches.
//
// Softmax without a maximum on the critical path: the exponent's reference m is the row's maximum over
// the first tile in which it sees a key, and stays.  P and l may then exceed 1 -- fp32 and bf16
// reach 2^127 -- and only when a row's sum over 64 keys leaves 2^32 is m moved (see `over` below).
// O stays below 2^32 (keys / 64) max|V|: values up to 2^78 for 2^20 keys and more, where a running maximum
// would carry 2^107.  (At 2^100 it overflowed for values of 2^27.  2^32 is 22 units of score above the first
// tile's maximum; normed queries and keys of rms 1.2 and head size 128 score within +-16.3.)
// The two threads of a row thus need not meet in a tile.  Rounding: P to bf16 for the product; l sums
// the unrounded values.
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
constexpr int kPcThreads = 640;   // producer, two issuers, an idle warp, 2 x 8 softmax warps
constexpr int kPcWarps = kPcThreads / 32;

// What paged_combine_kernel needs of the unit that starts in a CTA's share and ends after it.
struct PagedCut {
  int tok0, tok1;      // the unit's tokens [tok0, tok1) in the packed batch
  int h, g_last;       // kv head; last contributing CTA (h < 0: no such unit)
  int slot1, pad[3];   // the first contributor's partial is in its slot 1
};

struct PagedChunkParams {
  PagedAttnParams a;
  PagedCut* cuts;      // [grid]
  int wait_last;       // the kernel ahead is this call's decode kernel, whose output this one does
                       // not read: wait for it only before the end
};

template <int D>
struct PagedChunkConfig {
  static constexpr int kPanels = D / 64;
  static constexpr int kTileBytes = kPanels * kPcTile * 128;
  static constexpr uint32_t kOCol = 2 * kPcTile;         // TMEM: S (and P) below, O0, O1 above
  static constexpr int kKOff = 2 * kTileBytes;           // Q0, Q1, then K and V, two stages each
  static constexpr int kVOff = kKOff + 2 * kTileBytes;
  static constexpr int kBarOff = kVOff + 2 * kTileBytes;
  static constexpr int kScanOff = kBarOff + 336;
  static constexpr int kSegOff = kScanOff + 256;
  // per query tile and row quarter: what the two warps exchange (PagedPair)
  static constexpr int kPairOff = kSegOff + 4 * 64;
  static constexpr int kBytes = kPairOff + 2 * 4 * 1024 + 1024;
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

// The keys and values of a request are read by all its units, most of them through L2: as evict_first,
// the right policy for data read once, 8,192 tokens after 8,192 took 856 us against 769 (window chunks
// 129 against 121).
__device__ __forceinline__ uint64_t l2_policy_evict_normal() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(p));
  return p;
}

// A bounded wait that polls rarely: try_wait suspends the warp for up to 20 us at a time (a plain one
// returns after a fraction of that, and the polls of sixteen waiting warps took a third of the
// schedulers' issue slots from the warps at work).
__device__ __forceinline__ bool mbar_try_wait_long(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "r"(20000)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool mbar_test_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool mbar_wait_small(uint64_t* bar, uint32_t parity, volatile int* abort) {
  if (mbar_test_wait(bar, parity) || mbar_try_wait_long(bar, parity)) return true;
  const uint64_t t0 = global_timer_ns();
#pragma unroll 1
  while (!mbar_try_wait_long(bar, parity)) {
    if (*abort) return false;
    if (global_timer_ns() - t0 > kWaitLimitNs) {
      record_error(kErrWaitTimeout);
      *abort = 1;
      return false;
    }
  }
  return true;
}

// True in one lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
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

// A unit (kv head aside): tiles' first tokens and counts, their key-tile ranges from kb.
struct ChunkUnit {
  PagedRow row;
  int r, qb, nqb;
  int c0, c1;            // tokens in Q0 and Q1 (first tokens: qb * 2 tpb, + tpb)
  int b0, e0, b1, e1;    // key tiles [b, e) each query tile needs, counted from kb
  int lo, hi, kb, n;
};

__device__ __forceinline__ int chunk_blocks(const PagedChunkParams& p, const PagedRow& x) {
  return static_cast<long long>(x.T) * p.a.G > p.a.few_rows ? (x.T + 2 * p.a.tpb - 1) / (2 * p.a.tpb) : 0;
}

__device__ __forceinline__ ChunkUnit chunk_unit(const PagedChunkParams& p, const PagedRow& x, int r, int qb, int nqb) {
  ChunkUnit u;
  u.row = x;
  u.r = r;
  u.qb = qb;
  u.nqb = nqb;
  const int first = qb * 2 * p.a.tpb, left = x.T - first;
  u.c0 = min(left, p.a.tpb);
  u.c1 = min(max(left - p.a.tpb, 0), p.a.tpb);
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
    u.b1 = min((min(first_key(first + p.a.tpb), u.hi) - u.kb) / kPcTile, u.n - 1);
    u.e1 = u.n;
  }
  return u;
}

// What the two warps of a row quarter share: per-row values they exchange (two slots), the rows' m
// after an overflow and how many there were, and each warp's progress -- 2 n + 1: it waits in the
// handshake over an overflow in its n-th tile, 2 n: that handshake is over and its P not yet stored, 2 n +
// 2: its P of the n-th tile is stored (or, the first half's warp, a part of a unit ended before its n-th
// tile and the products of all its P are complete).
struct PagedPair {
  float xch[2][2][32];
  float m[32];
  int events;
  int progress[2];
  int pad[93];
};
static_assert(sizeof(PagedPair) == 1024, "eight of 1 KB");

// The part of a unit in one CTA's share, as the producer describes it to the other roles.
struct ChunkSeg {
  int seg;             // key tiles (0: no more parts)
  int kt0;             // the first one's first key
  int lo, hi;          // the unit's visible keys
  int b0, e0, b1, e1;  // the tiles [b, e) of each query tile, counted from the first here
  int pos0;            // position of the unit's first token
  int c0, c1;          // tokens in Q0, Q1
  int tok;             // the unit's first token in the packed batch
  int h;               // kv head
  int part;            // -1: the whole unit; else the slot of the partial result
  int pad[2];
};
static_assert(sizeof(ChunkSeg) == 64, "four descriptions of 64 bytes");

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

// 32 TMEM columns of this warp's lanes, not waited for; tmem_ld_wait32 orders every use after it.
__device__ __forceinline__ void tmem_ld32_nowait(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_wait32(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

// 32 TMEM columns of this warp's lanes to zero.
__device__ __noinline__ void tmem_zero32(uint32_t taddr) {
  const uint32_t z[32] = {};
  tmem_st32(taddr, z);
}

// The maximum of this thread's 64 scores; with mask, columns outside [lo, hi) are first set to -inf in
// TMEM.  Out of line, as all that a tile in a row's interior does not run: see mbar_wait_small.
__device__ __noinline__ float tmem_prep(uint32_t addr, bool mask, int lo, int hi) {
  const uint32_t width = hi > lo ? static_cast<uint32_t>(hi - lo) : 0u;
  float mx = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < 64; c += 32) {
    uint32_t a[32];
    tmem_ld32(addr + c, a);
    if (mask) {
#pragma unroll
      for (int e = 0; e < 32; ++e)
        if (static_cast<uint32_t>(c + e - lo) >= width) a[e] = __float_as_uint(-INFINITY);
      tmem_st32(addr + c, a);
    }
#pragma unroll
    for (int e = 0; e < 32; e += 2) mx = fmax3(mx, __uint_as_float(a[e]), __uint_as_float(a[e + 1]));
  }
  return mx;
}

// 32 of a row's weights, 2^(s * scale - m): packed bf16 into w, the unrounded ones added to acc.  (A
// polynomial on the FMA pipe for some of them, to spare the special function unit's 16 a clock, lost: it
// costs the issue slots that the four chains' warps share.  8,192 after 8,192, in one run back to back in
// a graph: 748 us without, 750, 760, 789 and 818 with one pair of sixteen, one, two and three of eight.)
__device__ __forceinline__ void exp32(const uint32_t (&s)[32], uint64_t sc2, uint64_t nm2, uint32_t (&w)[16],
                                      uint64_t& acc0, uint64_t& acc1) {
#pragma unroll
  for (int c = 0; c < 16; ++c) {
    const uint64_t x = fma2(static_cast<uint64_t>(s[2 * c]) | static_cast<uint64_t>(s[2 * c + 1]) << 32, sc2, nm2);
    const float e0 = fast_exp2(lo_f(x)), e1 = fast_exp2(hi_f(x));
    if (c & 1) acc1 = add2(acc1, pair_f32(e0, e1));
    else acc0 = add2(acc0, pair_f32(e0, e1));
    w[c] = pack_bf16x2_rn(e0, e1);
  }
}

// `cols` accumulator columns of this warp's rows times alpha; 32 packed columns of P times alpha.
__device__ __noinline__ void tmem_scale(uint32_t addr, int cols, float alpha) {
#pragma unroll 1
  for (int c = 0; c < cols; c += 32) {
    uint32_t o[32];
    tmem_ld32(addr + c, o);
#pragma unroll
    for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
    tmem_st32(addr + c, o);
  }
}
__device__ __noinline__ void tmem_scale_bf16(uint32_t addr, float alpha) {
  uint32_t o[32];
  tmem_ld32(addr, o);
#pragma unroll
  for (int e = 0; e < 32; ++e)
    o[e] = pack_bf16x2_rn(__uint_as_float(o[e] << 16) * alpha, __uint_as_float(o[e] & 0xffff0000u) * alpha);
  tmem_st32(addr, o);
}

// COLS columns of this warp's rows of O times inv: as bf16 to out at row `orow` (-1: no such row), or as
// fp32 to part, whose layout is [4 columns][row] so that the lanes' stores join.  For out four lanes
// transpose 4 x 16 bytes by shuffles and write 64 contiguous bytes of a row together (a store of 32
// rows' separate 16 bytes takes the LSU 32 cycles, these 8).
template <int COLS>
__device__ __noinline__ void chunk_store(uint32_t o_addr, float inv, int orow, uint16_t* out, long long pitch,
                                         float* part) {
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (int c = 0; c < COLS; c += 32) {
    uint32_t o[32];
    tmem_ld32(o_addr + c, o);
#pragma unroll
    for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * inv);
    if (part != nullptr) {
      if (orow >= 0)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          *reinterpret_cast<uint4*>(part + (c / 4 + e) * (256 * 4)) =
              make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
      continue;
    }
    uint32_t v[4][4];  // four 16-byte chunks of this lane's row
#pragma unroll
    for (int e = 0; e < 16; ++e)
      v[e >> 2][e & 3] = pack_bf16x2_rn(__uint_as_float(o[2 * e]), __uint_as_float(o[2 * e + 1]));
#pragma unroll
    for (int b = 1; b < 4; b <<= 1)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i & b) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t got = __shfl_xor_sync(0xffffffffu, (lane & b) ? v[i][e] : v[i | b][e], b);
          if (lane & b) v[i][e] = got;
          else v[i | b][e] = got;
        }
      }
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // now v[i]: this lane's chunk of the group's i-th row
      const int ri = __shfl_sync(0xffffffffu, orow, (lane & ~3) + i);
      if (ri >= 0)
        *reinterpret_cast<uint4*>(out + ri * pitch + c + (lane & 3) * 8) = make_uint4(v[i][0], v[i][1], v[i][2], v[i][3]);
    }
  }
}

template <int D>
__global__ void __launch_bounds__(kPcThreads, 1)
    paged_chunk_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                       const __grid_constant__ CUtensorMap vmap, const PagedChunkParams p) {
  using Cfg = PagedChunkConfig<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::kBarOff);
  uint64_t* q_full = bars + 0;
  uint64_t* q_empty = bars + 1;
  uint64_t* k_full = bars + 2;     // [2]
  uint64_t* v_full = bars + 4;     // [2]
  uint64_t* k_empty = bars + 6;    // [2]
  uint64_t* v_empty = bars + 8;    // [2]
  uint64_t* s_full = bars + 10;    // [4] chain (query tile) * 2 + half
  uint64_t* p_full = bars + 14;    // [4] 128 arrivals
  uint64_t* o_done = bars + 18;    // [2] per query tile: a part's products are complete
  uint64_t* epi_done = bars + 35;  // [2] 256 arrivals: ... and its O has been read
  uint64_t* drained = bars + 20;
  uint64_t* pv_end = bars + 33;    // [2] per query tile: a part's last product of the first half is complete
  // [4] a description is there.  The producer writes description x after q_empty(x - 1), so after
  // epi_done(x - 3): every softmax thread is past x - 3, and the four in the ring are never behind
  uint64_t* seg_full = bars + 21;
  uint64_t* pairs = bars + 25;     // [2][4] 2 arrivals: the two warps of a tile's row quarter
  constexpr int kNumBars = 37;
  static_assert((kNumBars + 4) * 8 <= 336, "barriers, TMEM slot, abort flag and start in 336 bytes");
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kNumBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + kNumBars + 1);
  int* ctl = reinterpret_cast<int*>(bars + kNumBars + 2);  // start: r, qb, h, local
  long long* warp_tot = reinterpret_cast<long long*>(smem + Cfg::kScanOff);  // [20]
  ChunkSeg* segs = reinterpret_cast<ChunkSeg*>(smem + Cfg::kSegOff);         // [4]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kNumBars; ++i) {
      // two arrivals: what both issuers hand back or end with, and the pairs
      const bool two = i == 1 || (i >= 6 && i < 10) || i == 20 || (i >= 25 && i < 33);
      mbar_init(bars + i, i >= 14 && i < 18 ? 128 : i >= 35 ? 256 : two ? 2 : 1);
    }
    *abort_flag = 0;
    for (int i = 0; i < 8; ++i) {
      PagedPair* pr = reinterpret_cast<PagedPair*>(smem + Cfg::kPairOff) + i;
      pr->events = pr->progress[0] = pr->progress[1] = 0;
    }
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
  const int per = (p.a.R + kPcWarps - 1) / kPcWarps;
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
  for (int i = 0; i < kPcWarps; ++i) {
    if (i < warp) before += warp_tot[i];
    total += warp_tot[i];
  }
  if (p.a.fill) paged_fill(p.a, D, blockDim.x);
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
  auto wait = [&](uint64_t* bar, uint32_t parity) {  // warp-uniform
    return __all_sync(0xffffffffu, mbar_wait_small(bar, parity, abort_flag)) != 0;
  };
  // the x-th description, once it is there; false on a timeout
  auto next_seg = [&](int x, ChunkSeg& d) {
    if (!wait(&seg_full[x & 3], (x >> 2) & 1)) return false;
    const int4* src = reinterpret_cast<const int4*>(&segs[x & 3]);
    int4* dst = reinterpret_cast<int4*>(&d);
#pragma unroll
    for (int i = 0; i < 4; ++i) dst[i] = src[i];
    return true;
  };

  if (warp < 4) {
    if (warp == 0) {
      // ---------------- producer and walker ----------------
      const uint64_t q_pol = l2_policy_evict_first(), kv_pol = l2_policy_evict_normal();
      const int box_shift = min(p.a.page_shift, 7);  // positions a box: min(page, 128)
      const int box = 1 << box_shift, nch = kPcTile >> box_shift;
      const uint32_t box_bytes = static_cast<uint32_t>(box) * 128u;
      const uint32_t q_bytes = static_cast<uint32_t>(p.a.tpb * p.a.G) * 128u;
      const int lch = lane / Cfg::kPanels, lpn = lane % Cfg::kPanels;
      ChunkWalk w;
      w.t = t_begin;
      if (active) {
        const PagedRow x = paged_row(p.a, ctl[0]);
        w.u = chunk_unit(p, x, ctl[0], ctl[1], chunk_blocks(p, x));
        w.h = ctl[2];
        w.local = ctl[3];
      }
      int g = 0, k = 0;
      bool ok = true;
      while (ok && w.t < t_end) {
        const int seg = static_cast<int>(min(static_cast<long long>(w.u.n - w.local), t_end - w.t));
        if (k > 0 && !(ok = wait(q_empty, (k - 1) & 1))) break;
        if (lane == 0) {
          const bool whole = w.local == 0 && seg == w.u.n;
          ChunkSeg d;
          d.seg = seg;
          d.kt0 = w.u.kb + w.local * kPcTile;
          d.lo = w.u.lo;
          d.hi = w.u.hi;
          d.b0 = max(w.u.b0 - w.local, 0);
          d.e0 = min(w.u.e0 - w.local, seg);
          d.b1 = max(w.u.b1 - w.local, 0);
          d.e1 = min(w.u.e1 - w.local, seg);
          d.pos0 = w.u.row.L + w.u.qb * 2 * p.a.tpb;
          d.c0 = w.u.c0;
          d.c1 = w.u.c1;
          d.tok = w.u.row.tok0 + w.u.qb * 2 * p.a.tpb;
          d.h = w.h;
          d.part = whole ? -1 : k > 0 ? 1 : 0;
          d.pad[0] = d.pad[1] = 0;
          segs[k & 3] = d;
          mbar_arrive(&seg_full[k & 3]);
          const long long start = w.t - w.local;
          if (!whole && w.local == 0) {  // it starts here and ends in another CTA's share
            PagedCut c;
            c.tok0 = d.tok;
            c.tok1 = d.tok + d.c0 + d.c1;
            c.h = w.h;
            c.g_last = share_owner(start + w.u.n - 1, total, ng);
            c.slot1 = d.part;
            c.pad[0] = c.pad[1] = c.pad[2] = 0;
            p.cuts[blockIdx.x] = c;
          }
          mbar_arrive_expect_tx(q_full, (w.u.c1 > 0 ? 2 : 1) * Cfg::kPanels * q_bytes);
          for (int t = 0; t < (w.u.c1 > 0 ? 2 : 1); ++t)
#pragma unroll
            for (int pn = 0; pn < Cfg::kPanels; ++pn)
              tma_load_3d(smem + t * Cfg::kTileBytes + pn * kPcTile * 128, &qmap, q_full, pn * 64, w.h * p.a.G,
                          d.tok + t * p.a.tpb, q_pol);
        }
        __syncwarp();
        ++k;
        const int32_t* table = p.a.block_table + w.u.r * p.a.table_stride;
        int pbase = 0, pg = 0;  // lane l holds the page of chunk pbase + l
        auto pages_from = [&](int c) {
          pbase = c;
          const long long key = static_cast<long long>(c + lane) << box_shift;
          pg = p.a.n_pages;  // outside the pool: a box there reads zeros
          if (key <= w.u.hi && key + box > w.u.lo) {
            pg = table[key >> p.a.page_shift];
            if (pg < 0 || pg >= p.a.n_pages) {
              record_error(kErrPageOutOfRange);
              pg = p.a.n_pages;
            }
          }
        };
        pages_from((w.u.kb + w.local * kPcTile) >> box_shift);
        for (int i = 0; ok && i < seg; ++i, ++g) {
          const int st = __shfl_sync(0xffffffffu, g & 1, 0);
          const int c0 = (w.u.kb + (w.local + i) * kPcTile) >> box_shift;
          if (c0 + nch > pbase + 32) pages_from(c0);
          // a lane a box: chunk lch, panel lpn of the tile's, those with visible keys (a loop over the boxes
          // held the products up where they are many, pages of 16: 385 -> 372 us for 4 chunks of 1,500)
          const int key0 = (c0 + lch) << box_shift;
          const bool load = lch < nch && key0 <= w.u.hi && key0 + box > w.u.lo;
          const int row = __shfl_sync(0xffffffffu, pg, (c0 - pbase + lch) & 31) * p.a.Hkv + w.h;
          const int pos = key0 & ((1 << p.a.page_shift) - 1);
          const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, load)) * box_bytes;
#pragma unroll 1
          for (int kv = 0; kv < 2; ++kv) {
            uint64_t* full = kv ? &v_full[st] : &k_full[st];
            if (g >= 2 && !(ok = wait(kv ? &v_empty[st] : &k_empty[st], ((g >> 1) - 1) & 1))) break;
            if (lane == 0) mbar_arrive_expect_tx(full, bytes);
            __syncwarp();
            uint8_t* dst = smem + (kv ? Cfg::kVOff : Cfg::kKOff) + st * Cfg::kTileBytes;
            if (load)
              tma_load_4d(dst + lpn * kPcTile * 128 + lch * box_bytes, kv ? &vmap : &kmap, full, 0, pos, lpn, row, kv_pol);
            __syncwarp();
          }
        }
        if (!ok) break;
        w.t += seg;
        w.local += seg;
        if (w.local == w.u.n && w.t < t_end) chunk_next(p, w);
      }
      if (ok && lane == 0) {
        segs[k & 3].seg = 0;
        mbar_arrive(&seg_full[k & 3]);
      }
      if (*abort_flag && lane == 0) {  // the copies in flight land before the CTA can exit
        for (int f = max(0, g - 2); f <= g; ++f) {
          if (f < g) mbar_wait(&k_full[f & 1], (f >> 1) & 1);
          if (f < g) mbar_wait(&v_full[f & 1], (f >> 1) & 1);
        }
        if (k > 0) mbar_wait(q_full, (k - 1) & 1);
      }
      __syncwarp();
    } else if (warp < 3) {
      // ---------------- product issuers, one a query tile ----------------
      // The whole warp waits, converged, and one elected lane issues: the descriptors are then
      // warp-uniform (a base and constants) and an MMA costs the warp an instruction or two.  Issued
      // from a lane-0 branch each took a dozen, and with two busy softmax warps on the same scheduler
      // the tensor cores starved: 2,400 FLOP a clock an SM against 8,000 in this form (both products
      // back to back beside fp32 work; 8,192 at most).  A warp a tile, because issuing blocks until
      // the tensor cores are nearly done: with one warp they idled while it went through its waits.
      constexpr uint32_t idesc_s = umma_idesc_bf16(128, 64, 0);
      constexpr uint32_t idesc_o = umma_idesc_bf16(128, D, 1);
      const int t = __shfl_sync(0xffffffffu, warp - 1, 0);
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      const uint64_t q_desc = smem_desc_sw128(base + t * Cfg::kTileBytes, 16, 1024);
      const uint64_t k_desc = smem_desc_sw128(base + Cfg::kKOff, 16, 1024);
      const uint64_t v_desc = smem_desc_sw128(base + Cfg::kVOff, kPcTile * 128, 1024);
      int g = 0;
      uint32_t parity = 0;  // of this tile's P so far
      bool ok = true;
      ChunkSeg d;
      for (int k = 0; ok; ++k) {
        if (!(ok = next_seg(k, d)) || d.seg == 0) break;
        ok = wait(q_full, k & 1);
        const int b = t ? d.b1 : d.b0, e = t ? d.e1 : d.e0;  // this tile's key tiles
        if (b >= e && lane == 0) mbar_arrive(q_empty);
        bool o_read = k == 0;  // the part before has been read out of O_t
        // Step j, half by half: P V of key tile j and S of j + 1 (j = -1: the first S).  Every key tile
        // is waited for and handed back by both issuers, used or not: each stage's phases stay in step.
#pragma unroll 1
        for (int j = -1; ok && j < d.seg; ++j) {
          const bool pv = j >= b && j < e, sn = j + 1 >= b && j + 1 < e, next = j + 1 < d.seg;
          const int gj = g + j, st = __shfl_sync(0xffffffffu, gj & 1, 0), st1 = st ^ 1;
          if (j >= 0) ok = wait(&v_full[st], (gj >> 1) & 1);
          if (ok && next) ok = wait(&k_full[st1], ((gj + 1) >> 1) & 1);
#pragma unroll 1
          for (int h = 0; ok && h < 2; ++h) {
            if (pv && !(ok = wait(&p_full[t * 2 + h], parity))) break;
            // A part's first product overwrites O_t.  Its P says that the warps with rows are past the last
            // part's end (they meet in the first tile), but a quarter without rows here hands its P over at
            // once, one of its warps possibly still at the last part's columns.
            if (pv && !o_read) {
              if (!(ok = wait(&epi_done[t], (k - 1) & 1))) break;
              o_read = true;
            }
            tc_fence_after();
            const uint32_t s_col = tm + t * kPcTile + h * 64;
            if (elect_one()) {
              if (pv) {
                const uint64_t va = v_desc + st * (Cfg::kTileBytes >> 4) + h * ((64 * 128) >> 4);
                const uint32_t more = j > b || h ? 1u : 0u;
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
                  umma_ts(tm + Cfg::kOCol + t * D, s_col + kk * 8, va + kk * ((16 * 128) >> 4), idesc_o,
                          kk > 0 ? 1u : more);
                if (!h && j == e - 1) umma_commit(&pv_end[t]);
                if (h) umma_commit(&v_empty[st]);
              }
              if (sn) {
                const uint64_t ka = k_desc + st1 * (Cfg::kTileBytes >> 4) + h * ((64 * 128) >> 4);
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                  const int off = (kk >> 2) * ((kPcTile * 128) >> 4) + (kk & 3) * (32 >> 4);
                  umma_ss(s_col, q_desc + off, ka + off, idesc_s, kk > 0 ? 1u : 0u);
                }
                umma_commit(&s_full[t * 2 + h]);
                if (h) umma_commit(&k_empty[st1]);
                if (h && j + 1 == e - 1) umma_commit(q_empty);
              }
            }
            __syncwarp();
          }
          if (lane == 0) {
            if (!pv && j >= 0) mbar_arrive(&v_empty[st]);
            if (!sn && next) mbar_arrive(&k_empty[st1]);
          }
          parity ^= pv ? 1u : 0u;
        }
        if (ok && !o_read) ok = wait(&epi_done[t], (k - 1) & 1);
        if (ok && elect_one()) umma_commit(&o_done[t]);
        __syncwarp();
        g += d.seg;
      }
      if (elect_one()) umma_commit(drained);  // every product has completed before TMEM is freed
      __syncwarp();
      mbar_wait(drained, 0);
      __syncwarp();
    }
  } else {
    // ---------------- softmax: eight warps a query tile, two threads a row ----------------
    const int t = (warp - 4) >> 3, hh = ((warp - 4) >> 2) & 1;  // query tile; half of the keys
    const int quarter = warp & 3;         // TMEM lanes 32 * quarter .. +31
    const int row = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_addr = tmem + lane_off + t * kPcTile + hh * 64;  // S, and P over it
    const uint32_t o_addr = tmem + lane_off + Cfg::kOCol + t * D;
    const int rt = row / p.a.G;           // the row's token in the tile
    const float sc = p.a.scale_log2;
    const uint64_t sc2 = pair_f32(sc, sc);
    uint64_t* pair = pairs + t * 4 + quarter;
    uint64_t* my_s = &s_full[t * 2 + hh];
    uint64_t* my_p = &p_full[t * 2 + hh];
    PagedPair* pr = reinterpret_cast<PagedPair*>(smem + Cfg::kPairOff) + t * 4 + quarter;
    volatile int* progress = pr->progress;
    volatile int* events = &pr->events;
    int g = 0, s_cnt = 0, ex = 0, seen = 0, ends = 0;
    bool ok = true;
    // The other thread's v (of this row): written to slot ex % 2 and read after both warps have
    // arrived; a slot is written again two exchanges later, when both have read it.
    auto exchange = [&](float v) -> float {
      pr->xch[ex & 1][hh][lane] = v;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(pair);
      if (!wait(pair, ex & 1)) ok = false;
      tc_fence_after();
      return pr->xch[ex++ & 1][hh ^ 1][lane];
    };
    for (int k = 0; ok; ++k) {
      ChunkSeg d;
      if (!(ok = next_seg(k, d)) || d.seg == 0) break;
      const int cnt_tok = t ? d.c1 : d.c0;
      const int jb = t ? d.b1 : d.b0, je = t ? d.e1 : d.e0;
      const bool valid = rt < cnt_tok;             // (rows past tpb * G have rt >= tpb)
      const int pos0 = d.pos0 + t * p.a.tpb, pos1 = pos0 + cnt_tok - 1;  // the tile's positions
      const int see_hi = min(pos0 + rt, d.hi), see_lo = p.a.window >= 0 ? pos0 + rt - p.a.window : 0;
      // 64 keys starting in [full_lo, full_hi] are seen whole by every row
      const int full_hi = min(pos0, d.hi) - 63, full_lo = p.a.window >= 0 ? pos1 - p.a.window : 0;
      // ... and 64 keys starting outside [some_lo, some_hi] by none (no window takes that below 32 bits)
      const int some_hi = min(pos1, d.hi), some_lo = p.a.window >= 0 ? max(pos0 - p.a.window, 0) - 63 : 0;
      const bool warp_rows = __any_sync(0xffffffffu, valid);
      float m_used = -INFINITY, l = 0.f;
      bool all_m = !warp_rows;  // every row here has an m
      int kt = d.kt0 + jb * kPcTile + hh * 64;  // the first of this half's keys
      auto new_m = [&] {  // the other warp moved m after an overflow
        seen = *events;
        const float m = pr->m[lane];
        if (m != m_used) l *= fast_exp2(m_used - m);
        m_used = m;
      };
      int cnt = 0;
      for (int j = jb; j < je; ++j, ++cnt, ++s_cnt, kt += kPcTile) {
        const bool plain = kt >= full_lo && kt <= full_hi && all_m && warp_rows;
        if (!(ok = wait(my_s, s_cnt & 1))) break;
        tc_fence_after();
        uint32_t a[32];
        tmem_ld32_nowait(s_addr, a);  // on its way during the checks
        if (__builtin_expect(*events != seen, 0)) new_m();
        if (__builtin_expect(!plain, 0)) {
          tmem_ld_wait32(a);
          if (kt < d.lo || kt + 63 > d.hi) {
            // rows of V outside [lo, hi] to zero: 64 rows, two threads a row
            const int st = (g + j) & 1;
            if (!(ok = wait(&v_full[st], ((g + j) >> 1) & 1))) break;
            const int vr = row >> 1;
            if (kt + vr < d.lo || kt + vr > d.hi) {
              const uint32_t at = base + Cfg::kVOff + st * Cfg::kTileBytes + (hh * 64 + vr) * 128;
#pragma unroll
              for (int c = 0; c < 4 * Cfg::kPanels; ++c)
                sts128(at + (Cfg::kPanels == 2 ? (row & 1) * (kPcTile * 128) + c * 16 : ((row & 1) * 4 + c) * 16),
                       make_uint4(0, 0, 0, 0));
            }
            fence_proxy_async_shared();
          }
          if (!warp_rows) {  // no query row in this quarter: P may be anything
            tc_fence_before();
            mbar_arrive(my_p);
            continue;
          }
          const bool full = kt >= full_lo && kt <= full_hi, none = kt < some_lo || kt > some_hi;
          float mx = -INFINITY;
          if (!none) mx = tmem_prep(s_addr, !full, max(0, see_lo - kt), valid ? min(64, see_hi - kt + 1) : 0) * sc;
          if (!all_m) {
            // (the same in both warps, which are both at their tile j: no product of O is in flight)
            mx = fmaxf(mx, exchange(mx));
            float alpha = 1.f;
            if (mx > m_used + 24.f) {  // a row's first keys, or far above its m (64 of 2^24 stay below `over`)
              alpha = fast_exp2(m_used - mx);  // 0 when m was -inf
              m_used = mx;
              l *= alpha;
            }
            all_m = !__any_sync(0xffffffffu, valid && m_used == -INFINITY);
            if (cnt > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
              tmem_scale(o_addr + hh * (D / 2), D / 2, alpha);
              exchange(0.f);  // both halves of O are scaled before either P can be used
            }
            if (!ok) break;
          }
          if (none) {
            tmem_zero32(s_addr);
            tc_fence_before();
            mbar_arrive(my_p);
            __syncwarp();
            if (lane == 0) progress[hh] = 2 * s_cnt + 2;
            continue;
          }
          tmem_ld32_nowait(s_addr, a);  // (masked)
        }
        uint32_t w0[16], w1[16];  // P of the first and the second 32 columns
        float sum;
        bool redone = false;
        while (true) {
          const float neg_m = m_used == -INFINITY ? 0.f : -m_used;
          const uint64_t nm2 = pair_f32(neg_m, neg_m);
          uint64_t acc0 = 0, acc1 = 0;
          tmem_ld_wait32(a);
          exp32(a, sc2, nm2, w0, acc0, acc1);
          tmem_ld32(s_addr + 32, a);
          exp32(a, sc2, nm2, w1, acc0, acc1);
          acc0 = add2(acc0, acc1);
          sum = lo_f(acc0) + hi_f(acc0);
          const bool over = valid && sum >= 4294967296.f;  // 2^32 (not a NaN)
          if (__builtin_expect(redone || !__any_sync(0xffffffffu, over), 1)) break;
          // Overflow (never where the maximum has just been exchanged, so all_m holds for both warps
          // from here on and they meet only below).  m moves to the maximum of the rows that need it, and
          // what was computed with the old one is rescaled.  The products of a query tile are issued
          // first half, second half, first half, ..., and this warp holds up its own: the other warp
          //   - has overflowed too (odd progress): both take the rows' common maximum and redo theirs; or
          //   - has stored the P whose product comes after this one's -- the first half's warp (hh = 0)
          //     in tile n waits for the second's tile n, the second's for the first's tile n + 1 -- so
          //     every product of O before is complete (its S was), and it waits for a next S that
          //     cannot come: this warp rescales that P and O, and the other finds the new m (events)
          //     before its next tile.
          redone = true;
          __syncwarp();
          if (lane == 0) progress[hh] = 2 * s_cnt + 1;
          const int need = 2 * (s_cnt + hh) + 1, low = 2 * (s_cnt - 1 + hh) + 1;
          int other = 0;
          bool there = false;
          const uint64_t t0 = global_timer_ns();
#pragma unroll 1
          while (!there && !*abort_flag && global_timer_ns() - t0 < kWaitLimitNs) {
            other = __shfl_sync(0xffffffffu, progress[hh ^ 1], 0);
            there = other >= need || other == low;
            __syncwarp();
          }
          if (__any_sync(0xffffffffu, !there)) {
            if (lane == 0 && !*abort_flag) record_error(kErrWaitTimeout);
            *abort_flag = 1;
            ok = false;
            break;
          }
          tc_fence_after();
          const bool both = other & 1;
          float mx = tmem_prep(s_addr, false, 0, 0) * sc;
          bool move = over;
          if (both) {
            mx = fmaxf(mx, exchange(mx));
            move = exchange(move ? 1.f : 0.f) != 0.f || move;
          }
          float alpha = 1.f;
          if (move && mx > m_used) {
            alpha = fast_exp2(m_used - mx);
            m_used = mx;
            l *= alpha;
          }
          if (both) {
            tmem_scale(o_addr + hh * (D / 2), D / 2, alpha);
            // No longer waiting, and the other is to know before it can look again: it may reach its next
            // tile and overflow there before this one's P is stored, would take an odd progress left
            // standing for this warp at the handshake, and wait for it in an exchange that it has left.
            // (The exchange publishes it.  A warp that goes on alone, below, may leave its odd progress:
            // that is below the other's `low` from the other's next tile on.)
            if (lane == 0) progress[hh] = 2 * s_cnt;
            exchange(0.f);  // both halves of O are scaled before either P can be used
            if (!ok) break;
          } else {
            tmem_scale(o_addr, D, alpha);
            tmem_scale_bf16(s_addr + (hh ? -64 : 64), alpha);
            pr->m[lane] = m_used;
            __syncwarp();
            seen = __shfl_sync(0xffffffffu, *events, 0) + 1;
            __syncwarp();
            if (lane == 0) *events = seen;
          }
          tmem_ld32_nowait(s_addr, a);
        }
        if (!ok) break;
        l += sum;
        tmem_st16_nowait(s_addr, w0);
        tmem_st16_nowait(s_addr + 16, w1);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(my_p);
        __syncwarp();
        if (lane == 0) progress[hh] = 2 * s_cnt + 2;
      }
      if (ok && cnt > 0) {
        ok = wait(&pv_end[t], ends & 1);
        ++ends;
        if (hh == 0 && lane == 0) progress[0] = 2 * s_cnt + 2;
      }
      if (ok) ok = wait(&o_done[t], k & 1);
      if (ok && warp_rows) {
        tc_fence_after();
        if (*events != seen) new_m();
        const float other = exchange(l);
        l = hh ? other + l : l + other;              // one order for both
        const float inv = l == 0.f ? 0.f : 1.f / l;  // (a NaN stays one)
        const long long slot = static_cast<long long>(blockIdx.x) * 2 + d.part;
        if (d.part >= 0 && valid && hh == 0)
          p.a.part_lse[slot * 256 + t * 128 + row] = l == 0.f ? -INFINITY : m_used + __log2f(l);
        if (cnt > 0) {
          const int orow = valid ? (d.tok + t * p.a.tpb + rt) * p.a.Hq + d.h * p.a.G + (row - rt * p.a.G) : -1;
          float* part = d.part < 0 ? nullptr
                                   : p.a.part_o + ((slot * (D / 4) + hh * (D / 8)) * 256 + t * 128 + row) * 4;
          chunk_store<D / 2>(o_addr + hh * (D / 2), inv, orow, p.a.out + hh * (D / 2), D, part);
        }
      }
      tc_fence_before();
      mbar_arrive(&epi_done[t]);  // O is read: the issuer may let the next unit's o_done complete
      g += d.seg;
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

// Merges the units cut between CTAs: blockIdx.x is the CTA whose share the unit starts in, blockIdx.y
// 32 of its rows.  A lane is a row, a warp takes every eighth group of four columns (the partials'
// layout: a load is 512 contiguous bytes); the rows leave through shared memory, whole.
template <int D>
__global__ void __launch_bounds__(256) paged_combine_kernel(const PagedChunkParams p) {
  __shared__ uint2 rows[32][D / 4 + 1];
  __shared__ int out_row[32];
  pdl_wait();
  pdl_launch_dependents();
  const PagedCut c = p.cuts[blockIdx.x];
  if (c.h < 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n = blockIdx.y * 32 + lane, rr = n & 127;
  const int rt = rr / p.a.G, tok = c.tok0 + (n >> 7) * p.a.tpb + rt;
  const bool valid = rt < p.a.tpb && tok < c.tok1;
  if (!__syncthreads_or(valid)) return;
  const int cnt = c.g_last - static_cast<int>(blockIdx.x) + 1;
  auto slot = [&](int k) { return (static_cast<long long>(blockIdx.x) + k) * 2 + (k == 0 && c.slot1 ? 1 : 0); };
  float mx = -CUDART_INF_F, wsum = 0.f;
  if (valid) {
    for (int k = 0; k < cnt; ++k) mx = fmaxf(mx, __ldcg(p.a.part_lse + slot(k) * 256 + n));
    for (int k = 0; k < cnt; ++k) {
      const float ls = __ldcg(p.a.part_lse + slot(k) * 256 + n);
      wsum += ls == -CUDART_INF_F ? 0.f : fast_exp2(ls - mx);
    }
  }
  const float inv = wsum == 0.f ? 0.f : 1.f / wsum;
  if (warp == 0) out_row[lane] = valid ? tok * p.a.Hq + c.h * p.a.G + (rr - rt * p.a.G) : -1;
#pragma unroll 1
  for (int q = warp; q < D / 4; q += 8) {
    float a[4] = {0.f, 0.f, 0.f, 0.f};
    if (valid) {
#pragma unroll 4
      for (int k = 0; k < cnt; ++k) {
        const float ls = __ldcg(p.a.part_lse + slot(k) * 256 + n);
        if (ls == -CUDART_INF_F) continue;  // (its partial was not written)
        const float w = fast_exp2(ls - mx);
        const float4 v =
            __ldcg(reinterpret_cast<const float4*>(p.a.part_o) + (slot(k) * (D / 4) + q) * 256 + n);
        a[0] = fmaf(w, v.x, a[0]);
        a[1] = fmaf(w, v.y, a[1]);
        a[2] = fmaf(w, v.z, a[2]);
        a[3] = fmaf(w, v.w, a[3]);
      }
    }
    rows[lane][q] = make_uint2(pack_bf16x2(a[0] * inv, a[1] * inv), pack_bf16x2(a[2] * inv, a[3] * inv));
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * (D / 4); i += 256) {
    const int r = i / (D / 4), q = i % (D / 4);
    if (out_row[r] >= 0)
      *reinterpret_cast<uint2*>(p.a.out + static_cast<long long>(out_row[r]) * D + 4 * q) = rows[r][q];
  }
}

}  // namespace mcb
