// Attention of trees of drafted tokens over a paged cache.
//
//   out[t, h] = sum_c softmax_c(q[t, h] . K[c, h / G] * softmax_scale) V[c, h / G]
// over the cached keys c < L with position_t - c <= window, and the request's new tokens j with mask
// bit j of t and position_t - position_j <= window (window < 0: all).  A request of more new tokens
// than the mask has bits is a chunk of a prompt, the chunk kernel's where that is launched.
//
// A tree has few query rows for many keys (16 tokens of 4 heads a kv head over 8,000 keys: 64 rows, 64
// FLOP a byte): bound by HBM, if products and softmax keep up with 44 GB/s an SM, a 128-key tile of K and V
// in 2,800 cycles at head size 128 and in 1,400 at 64.  The query rows of a kv head are packed as in the
// chunk kernel, row = token * G + head, 128 a tile; a *unit* is (request, two tiles Q0, Q1, kv head), its
// keys from the first that any of its rows may see to the request's last.  All units' 128-key tiles form one
// sequence that the CTAs (one an SM) share evenly, computed on the device from the lengths; a cut unit leaves
// (O / l, log2 sum) in workspace and tree_combine_kernel, launched after, merges them.
//
// Roles of a CTA's warps:
//   warp 0      TMA producer and walker: describes each part of a unit in shared memory, loads its queries,
//               and K tiles into a ring that runs on across units
//   warp 3      the same walk, V tiles
//   warps 1, 2  (warp 1 allocates TMEM) products of group 0, of group 1:
//                 S_th = Q K_jh^T    M=128 N=64 K=D   (both operands from shared memory; h: half of a key tile)
//                 O_t += P_th V_jh   M=128 N=D K=64   (P from TMEM, over its S)
//   warps 4-7   softmax of group 0, warps 8-11 of group 1: a thread a query row
// Two groups, each with its own S, running maximum, sum and accumulator, so that one group's products run
// beside the other's softmax.  Where a unit has one query tile -- up to 128 rows, most trees -- the groups
// take its key tiles in turn, each key tile read once, and merge their two results in TMEM at the
// unit's end; with two tiles each group has one and both read every key tile.
// TMEM: S_0, S_1 of 128 columns, O_0, O_1 of D: all 512 at D = 128.
//
// A group's key tile goes half by half (64 keys), S -> softmax -> P V -> the next tile's S, so that the products of one half
// run beside the softmax of the other.  The running maximum m moves only when a row's scores exceed it by 2^8 (P and l
// stay far below 2^127): then the row's O, in TMEM, is rescaled, after the half's before P V, the one product that may
// still be at it.  P is rounded to bf16 for the product; l sums the unrounded values.
//
// Masks: only the tiles with new tokens, at a window's start or at the unit's end look at them; a row's
// 32 bits at a time are made from its interval of cached keys and its mask words, shifted to the
// tile.  A key tile's positions outside the unit's [lo, hi] may hold anything: scores there are replaced by
// -inf, and their rows of V are zeroed in shared memory before the product reads them (0 * NaN is NaN).
// Every wait is bounded; a timeout raises the abort flag, the issuers wait for their products, the
// producers for their copies, and TMEM is freed.
//
// Measured, back to back in a graph with the combine (16/4 heads of 128, pages of 64): 32 requests of 8,192 with 16
// tokens each (64 rows) 97 us, 5.6 TB/s; with 64 tokens (256 rows) 157 us, 3.5 TB/s and 880 TFLOP/s -- two tiles a
// key tile are 2,560 cycles of products at N = 64 and 2,048 of exponentials, and take some 4,000 at the 1.45 GHz
// that the power limit leaves: the tensor cores 42% busy, the special function unit 44%.  12/12 heads of 64, 64
// tokens at 4,096: 112 us.  Whole key tiles (one chain a group) were slower, 206 us for the 256 rows, and one
// producer warp for both K and V (127 against 117 us at head size 64, one row).
#pragma once

#include "paged_chunk.cuh"

namespace mcb {

struct PagedTreeParams {
  PagedAttnParams a;
  PagedCut* cuts;            // [grid]
  const int32_t* positions;  // (N,)
  const uint32_t* mask;      // (N, words)
  int words;
  int unit_tok;              // new tokens a unit: a tile's or two tiles'
};

constexpr int kPtTile = 128;      // query rows a tile, keys a key tile
constexpr int kPtThreads = 384;   // two producers, two issuers, 2 x 4 softmax warps
constexpr int kPtWarps = kPtThreads / 32;

template <int D>
struct PagedTreeConfig {
  static constexpr int kPanels = D / 64;
  static constexpr int kTileBytes = kPanels * kPtTile * 128;
  static constexpr int kK = D == 128 ? 2 : 5, kV = D == 128 ? 3 : 7;  // (V's wait for the softmax)
  static constexpr int kStages = kK + kV;                // K's ring, then V's
  static constexpr uint32_t kOCol = 2 * kPtTile;         // TMEM: S (and P) below, O_0, O_1 above
  static constexpr int kRingOff = 2 * kTileBytes;        // Q0, Q1, then the ring
  static constexpr int kBarOff = kRingOff + kStages * kTileBytes;
  static constexpr int kNumBars = 4 * kStages + 29;
  static constexpr int kSegOff = (kBarOff + kNumBars * 8 + 32 + 63) / 64 * 64;
  static constexpr int kXchOff = kSegOff + 4 * 64;       // a float a row of either group
  static constexpr int kBytes = kXchOff + 2 * kPtTile * 4 + 1024;
  // above half of an SM's shared memory: two CTAs never meet on one SM, whose TMEM each needs whole
  static_assert(kBytes > 118784 && kBytes <= 232448, "one CTA an SM");
};

// A unit (kv head aside).
struct TreeUnit {
  PagedRow row;
  int r, qb, nqb;
  int c0, c1;       // tokens in Q0 and Q1 (first tokens: qb * unit_tok, + tpb)
  int lo, hi, kb, n;
};

__device__ __forceinline__ bool tree_causal(const PagedTreeParams& p, const PagedRow& x) {
  return x.T > 32 * p.words;
}

__device__ __forceinline__ int tree_blocks(const PagedTreeParams& p, const PagedRow& x) {
  return p.a.all || !tree_causal(p, x) ? (x.T + p.unit_tok - 1) / p.unit_tok : 0;
}

__device__ __forceinline__ TreeUnit tree_unit(const PagedTreeParams& p, const PagedRow& x, int r, int qb, int nqb) {
  TreeUnit u;
  u.row = x;
  u.r = r;
  u.qb = qb;
  u.nqb = nqb;
  const int first = qb * p.unit_tok, left = min(x.T - first, p.unit_tok);
  u.c0 = min(left, p.a.tpb);
  u.c1 = left - u.c0;
  const bool causal = tree_causal(p, x);
  const long long cap = (static_cast<long long>(p.a.max_pages) << p.a.page_shift) - 1;
  const int last = causal ? first + u.c0 + u.c1 - 1 : x.T - 1;  // a tree's token may see any other
  u.lo = p.a.window >= 0 ? max(0, x.L + (causal ? first : 0) - p.a.window) : 0;
  u.hi = static_cast<int>(min(static_cast<long long>(x.L) + last, cap));
  u.kb = min(u.lo, u.hi) / kPtTile * kPtTile;
  u.n = (u.hi - u.kb) / kPtTile + 1;
  return u;
}

// The part of a unit in one CTA's share, as the producer describes it to the other roles.
struct TreeSeg {
  int seg;             // key tiles
  int kt0;             // the first one's first key
  int lo, hi;          // the unit's keys
  int L, T, tok0;      // the request's
  int first;           // the unit's first token, counted from the request's first
  int c0, c1;          // tokens in Q0, Q1
  int h;               // kv head
  int part;            // -1: the whole unit; else the slot of the partial result
  int q;               // one tile: which of the two places its queries have; parities of q_full << 1, << 2
                       // (the kernel for few rows: whether the first contributor's partial is in its slot 1)
  int last;            // no more parts
  int pad[2];          // (the kernel for few rows: a cut unit's first and last contributors)
};
static_assert(sizeof(TreeSeg) == 64, "four descriptions of 64 bytes");

struct TreeWalk {
  TreeUnit u;
  int h, local;
  long long t;
};

__device__ __forceinline__ void tree_next(const PagedTreeParams& p, TreeWalk& w) {
  w.local = 0;
  if (++w.h < p.a.Hkv) return;
  w.h = 0;
  if (w.u.qb + 1 < w.u.nqb) {
    w.u = tree_unit(p, w.u.row, w.u.r, w.u.qb + 1, w.u.nqb);
    return;
  }
  for (int r = w.u.r + 1; r < p.a.R; ++r) {
    const PagedRow x = paged_row(p.a, r);
    const int nqb = tree_blocks(p, x);
    if (nqb > 0) {
      w.u = tree_unit(p, x, r, 0, nqb);
      return;
    }
  }
}

// chunk_rows for this kernel's units: rows [row_a, row_b) 32 at a time (a lane each), the blocks of each row
// in turn (a lane each).  Stops when visit(request, first block, this lane's tiles) returns true (uniform).
template <typename F>
__device__ __forceinline__ void tree_rows(const PagedTreeParams& p, int row_a, int row_b, F visit) {
  const int lane = threadIdx.x & 31;
  for (int base = row_a; base < row_b; base += 32) {
    PagedRow x = {0, 0, 0};
    int nqb = 0;
    if (base + lane < row_b) {
      x = paged_row(p.a, base + lane);
      if (blockIdx.x == 0 && !paged_row_fits(p.a, base + lane, x)) record_error(kErrPositionBeyondCache);
      nqb = tree_blocks(p, x);
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
        const int n = qb + lane < nb ? tree_unit(p, y, base + src, qb + lane, nb).n : 0;
        if (visit(base + src, qb, n)) return;
      }
    }
  }
}

// Where a CTA's share of the tiles begins and ends, and the walk at its start: every warp's own when all requests
// fit its lanes (no barrier, nothing through shared memory, which a step of few requests is made of), else the
// CTA's together through `tot` (kPtWarps words) and `ctl` (4).  Ends with all threads past one __syncthreads.
struct TreeShare {
  long long total, t_begin, t_end;
  int ng;
  int g_first, g_last;  // the one unit's contributors, where a CTA's share is one unit's (else g_last < 0)
};
// Who has the tiles of the unit that the walk is in, and whether the first one's partial is in its slot 1.
__device__ __forceinline__ void tree_owners(const TreeShare& s, const TreeWalk& w, int& first, int& last, int& slot1) {
  first = s.g_first, last = s.g_last, slot1 = 0;
  if (s.g_last >= 0) return;
  const long long start = w.t - w.local;
  first = share_owner(start, s.total, s.ng);
  last = share_owner(start + w.u.n - 1, s.total, s.ng);
  slot1 = start != share_begin(first, s.total, s.ng);
}
// A unit's two ends -- its first maximum, masks, sums, way out -- cost a CTA what some three tiles do.  Where equal
// numbers of CTAs a unit give no CTA more than that above an even share, no CTA has two units' ends: three requests of
// 12 heads of 64 at 1,000 some 17 us for the slowest CTA, whose 2 tiles were two units', and 9 for the others.
constexpr int kUnitEnds = 3;
__device__ __forceinline__ TreeShare tree_share(long long total) {
  TreeShare s;
  s.total = total;
  s.g_first = s.g_last = -1;
  s.ng = static_cast<int>(min(static_cast<long long>(gridDim.x), total));
  const bool active = static_cast<int>(blockIdx.x) < s.ng;
  s.t_begin = active ? share_begin(blockIdx.x, total, s.ng) : 0;
  s.t_end = active ? share_begin(blockIdx.x + 1, total, s.ng) : 0;
  return s;
}
__device__ __forceinline__ TreeShare tree_place(const PagedTreeParams& p, TreeWalk& w, long long* tot, int* ctl) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  TreeShare s;
  if (p.a.R <= 32) {
    PagedRow x = {0, 0, 0};
    long long mine = 0;
    int units = 0, longest = 0;  // (counts stop at 2^20: no more are shared out unit by unit)
    if (lane < p.a.R) {
      x = paged_row(p.a, lane);
      if (blockIdx.x == 0 && warp == 0 && !paged_row_fits(p.a, lane, x)) record_error(kErrPositionBeyondCache);
      const int nqb = tree_blocks(p, x);
      for (int qb = 0; qb < nqb; ++qb) {
        const int n = tree_unit(p, x, lane, qb, nqb).n;
        mine += n;
        longest = max(longest, n);
      }
      mine *= p.a.Hkv;
      units = static_cast<int>(min(static_cast<long long>(nqb) * p.a.Hkv, 1ll << 20));
    }
    long long incl = mine;
    int units_incl = units;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const long long o = __shfl_up_sync(0xffffffffu, incl, m);
      const int u = __shfl_up_sync(0xffffffffu, units_incl, m);
      longest = max(longest, __shfl_xor_sync(0xffffffffu, longest, m));
      if (lane >= m) {
        incl += o;
        units_incl += u;
      }
    }
    const int all_units = __shfl_sync(0xffffffffu, units_incl, 31);
    const int each = all_units > 0 ? static_cast<int>(gridDim.x) / all_units : 0;  // CTAs a unit
    const long long total = __shfl_sync(0xffffffffu, incl, 31);
    if (each > 0 && (longest + each - 1) / each <= total / static_cast<int>(gridDim.x) + kUnitEnds) {
      s.total = total;
      s.ng = all_units * each;
      s.t_begin = s.t_end = 0;
      s.g_first = blockIdx.x / each * each;
      s.g_last = 0;
      const int unit = blockIdx.x / each;
      if (unit < all_units) {
        const int r = __ffs(__ballot_sync(0xffffffffu, unit < units_incl)) - 1;
        const int at = unit - __shfl_sync(0xffffffffu, units_incl - units, r);
        x.tok0 = __shfl_sync(0xffffffffu, x.tok0, r);
        x.T = __shfl_sync(0xffffffffu, x.T, r);
        x.L = __shfl_sync(0xffffffffu, x.L, r);
        w.u = tree_unit(p, x, r, at / p.a.Hkv, tree_blocks(p, x));
        w.h = at % p.a.Hkv;
        const int parts = min(each, w.u.n), part = static_cast<int>(blockIdx.x) - s.g_first;
        s.g_last = s.g_first + parts - 1;
        if (part < parts) {  // tiles counted from the unit's first
          s.t_begin = static_cast<long long>(w.u.n) * part / parts;
          s.t_end = static_cast<long long>(w.u.n) * (part + 1) / parts;
        }
      }
      w.t = s.t_begin;
      w.local = static_cast<int>(s.t_begin);
      __syncthreads();
      return s;
    }
    s = tree_share(total);
    w.t = s.t_begin;
    if (s.t_begin < s.t_end) {
      const int r = __ffs(__ballot_sync(0xffffffffu, s.t_begin < incl)) - 1;  // (t_begin < total: some lane's)
      long long left = s.t_begin - __shfl_sync(0xffffffffu, incl - mine, r);
      x.tok0 = __shfl_sync(0xffffffffu, x.tok0, r);
      x.T = __shfl_sync(0xffffffffu, x.T, r);
      x.L = __shfl_sync(0xffffffffu, x.L, r);
      const int nqb = tree_blocks(p, x);
      w.u = tree_unit(p, x, r, 0, nqb);
      while (left >= static_cast<long long>(w.u.n) * p.a.Hkv) {
        left -= static_cast<long long>(w.u.n) * p.a.Hkv;
        w.u = tree_unit(p, x, r, w.u.qb + 1, nqb);
      }
      const uint32_t at = static_cast<uint32_t>(left);  // < n Hkv
      w.h = static_cast<int>(at / static_cast<uint32_t>(w.u.n));
      w.local = static_cast<int>(at % static_cast<uint32_t>(w.u.n));
    }
    __syncthreads();
    return s;
  }
  const int per = (p.a.R + kPtWarps - 1) / kPtWarps;
  const int row_a = min(warp * per, p.a.R), row_b = min(row_a + per, p.a.R);
  long long mine = 0;
  tree_rows(p, row_a, row_b, [&](int, int, int n) {
    mine += n;
    return false;
  });
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, m);
  mine *= p.a.Hkv;
  if (lane == 0) tot[warp] = mine;
  __syncthreads();
  long long total = 0, before = 0;
#pragma unroll
  for (int i = 0; i < kPtWarps; ++i) {
    if (i < warp) before += tot[i];
    total += tot[i];
  }
  s = tree_share(total);
  const long long t_begin = s.t_begin;
  if (t_begin < s.t_end && before <= t_begin && t_begin < before + mine) {
    long long left = t_begin - before;
    tree_rows(p, row_a, row_b, [&](int r, int qb, int n) {
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
  __syncthreads();
  w.t = t_begin;
  if (t_begin < s.t_end) {
    const PagedRow x = paged_row(p.a, ctl[0]);
    w.u = tree_unit(p, x, ctl[0], ctl[1], tree_blocks(p, x));
    w.h = ctl[2];
    w.local = ctl[3];
  }
  return s;
}

// paged_fill by threads 0 .. threads - 1 of every CTA, this one `index`.
__device__ __forceinline__ void tree_fill(const PagedAttnParams& p, int D, int index, int threads) {
  const long long per = static_cast<long long>(p.Hq) * D / 8;  // 16-byte words a token
  const int first = min(max(p.cu_new[0], 0), p.N), last = max(min(p.cu_new[p.R], p.N), first);
  const long long lead = first * per, gap = (last - first) * per, end = p.N * per;
  uint4* out = reinterpret_cast<uint4*>(p.out);
  for (long long i = static_cast<long long>(blockIdx.x) * threads + index; i < end - gap;
       i += static_cast<long long>(gridDim.x) * threads)
    out[i < lead ? i : i + gap] = make_uint4(0, 0, 0, 0);
}

// Bits a .. b of a word (none when b < a; 0 <= a, b <= 31).
__device__ __forceinline__ uint32_t bit_range(int a, int b) {
  return b < a ? 0u : (b - a == 31 ? 0xffffffffu : ((1u << (b - a + 1)) - 1)) << a;
}

// Which of the 32 keys from k0 on a row sees.  Out of line: a tile in a request's interior asks for none.
// (Arguments by value: what has an address lives in local memory, and shared memory leaves the L1 cache next to
// nothing to keep it.)  [see_lo, see_hi]: its interval of cached keys (a chunk's token: of all); L, T, tok0 the
// request's; tok its own place in the packed batch (-1: by the interval alone), pos its position.
__device__ __noinline__ uint32_t tree_bits(const PagedTreeParams& p, int see_lo, int see_hi, int L, int T, int tok0,
                                           int tok, int pos, int k0) {
  uint32_t bits = bit_range(max(see_lo - k0, 0), min(see_hi - k0, 31));
  const int j0 = k0 - L;  // the first key's place among the new tokens
  if (tok < 0 || j0 <= -32 || j0 >= T) return bits;
  const int w = j0 >> 5, sh = j0 & 31;
  const uint32_t* row = p.mask + static_cast<long long>(tok) * p.words;
  const uint32_t a = w >= 0 && w < p.words ? row[w] : 0u, b = w + 1 < p.words ? row[w + 1] : 0u;
  uint32_t fresh = __funnelshift_r(a, b, sh) & bit_range(max(-j0, 0), min(T - 1 - j0, 31));
  if (p.a.window >= 0 && pos - L > p.a.window)  // (a new token's position is L or more)
    for (uint32_t left = fresh; left != 0; left &= left - 1) {
      const int e = __ffs(left) - 1;
      if (pos - max(p.positions[tok0 + j0 + e], L) > p.a.window) fresh &= ~(1u << e);
    }
  return bits | fresh;
}

// COLS columns of this warp's rows, O_0 w0 + O_1 w1 (a weight of 0: not read): as chunk_store.
template <int COLS>
__device__ __noinline__ void tree_store(uint32_t o0, uint32_t o1, float w0, float w1, int orow, uint16_t* out,
                                        long long pitch, float* part) {
  const int lane = threadIdx.x & 31;
  const bool any0 = __any_sync(0xffffffffu, w0 != 0.f), any1 = __any_sync(0xffffffffu, w1 != 0.f);
#pragma unroll 1
  for (int c = 0; c < COLS; c += 32) {
    uint32_t o[32];
    if (any0) {
      tmem_ld32(o0 + c, o);
#pragma unroll
      for (int e = 0; e < 32; ++e) o[e] = w0 != 0.f ? __float_as_uint(__uint_as_float(o[e]) * w0) : 0u;
    } else {
#pragma unroll
      for (int e = 0; e < 32; ++e) o[e] = 0u;
    }
    if (any1) {
      uint32_t b[32];
      tmem_ld32(o1 + c, b);
#pragma unroll
      for (int e = 0; e < 32; ++e)
        if (w1 != 0.f) o[e] = __float_as_uint(fmaf(__uint_as_float(b[e]), w1, __uint_as_float(o[e])));
    }
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
__global__ void __launch_bounds__(kPtThreads, 1)
    paged_tree_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                      const __grid_constant__ CUtensorMap vmap, const __grid_constant__ PagedTreeParams p) {
  using Cfg = PagedTreeConfig<D>;
  constexpr int ST = Cfg::kStages, SK = Cfg::kK, SV = Cfg::kV;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::kBarOff);
  // [3][ST] the rings: K of key tile g at g mod kK, V at kK + g mod kV.  A set a reader -- group 0, group 1, both -- whose
  // phases only its reader's uses advance: a wait is for the phase after the last one waited for, never
  // for one that another reader's copy, still on its way, would have to complete first
  uint64_t* full = bars;
  // [ST] two arrivals: both groups' products; one tile's keys: its group's and the producer's own
  uint64_t* empty = full + 3 * ST;
  uint64_t* q_full = empty + ST;     // [2]
  uint64_t* q_empty = q_full + 2;    // [2] two arrivals, as empty
  uint64_t* s_full = q_empty + 2;    // [4] group * 2 + half of the key tile
  uint64_t* p_full = s_full + 4;     // [4] 128 arrivals
  uint64_t* pv_done = p_full + 4;    // [2] a half's P V is complete
  uint64_t* v_ready = pv_done + 2;   // [2] a tile's values have landed, told for tiles with keys outside [lo, hi]
  uint64_t* o_done = v_ready + 2;    // [2] a part's products are complete
  uint64_t* epi_done = o_done + 2;   // [2] 128 arrivals: ... and its O has been read
  // [4] a description is there.  Description x is written once the queries' place of part x - 2 or later is
  // free, so after every thread is past x - 4
  uint64_t* seg_full = epi_done + 2;
  uint64_t* pair_bar = seg_full + 4; // [4] two arrivals: the two warps of a row quarter
  uint64_t* drained = pair_bar + 4;  // two arrivals
  static_assert(4 * ST + 29 == Cfg::kNumBars, "the barriers above");
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + Cfg::kNumBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* ctl = reinterpret_cast<int*>(tmem_slot + 2);  // start: r, qb, h, local
  TreeSeg* segs = reinterpret_cast<TreeSeg*>(smem + Cfg::kSegOff);
  float* xch = reinterpret_cast<float*>(smem + Cfg::kXchOff);  // [2][128]
  long long* warp_tot = reinterpret_cast<long long*>(xch);     // [12], before the roles begin
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < Cfg::kNumBars; ++i) {
      uint64_t* b = bars + i;
      const bool two = (b >= empty && b < q_full) || (b >= q_empty && b < s_full) || b >= pair_bar;
      const bool threads = (b >= p_full && b < pv_done) || (b >= epi_done && b < seg_full);
      mbar_init(b, threads ? 128 : two ? 2 : 1);
    }
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
  pdl_wait();
  pdl_launch_dependents();

  // ---- the sequence's length and this CTA's first tile ----
  if (threadIdx.x == 0) p.cuts[blockIdx.x].h = -1;
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

  if (warp < 4) {
    if (warp == 0 || warp == 3) {
      // ---------------- producers: of K, the queries and the descriptions; of V ----------------
      // (one warp for both tiles, a chain of some 100 dependent instructions a tile and 1,000 cycles, was what
      // bounded head size 64)
      const int kv = warp == 3;
      const CUtensorMap* map = kv ? &vmap : &kmap;
      const uint64_t policy = l2_policy_evict_first();
      const int box_shift = min(p.a.page_shift, 7);  // positions a box: min(page, 128)
      const int box = 1 << box_shift, nch = kPtTile >> box_shift;
      const uint32_t box_bytes = static_cast<uint32_t>(box) * 128u;
      const uint32_t q_bytes = static_cast<uint32_t>(p.a.tpb * p.a.G) * 128u;
      const int lch = lane / Cfg::kPanels, lpn = lane % Cfg::kPanels;
      const uint32_t lane_dst = Cfg::kRingOff + lpn * kPtTile * 128 + lch * box_bytes;
      uint32_t gt = 0;        // key tiles so far
      uint32_t sets = 0, armed[3] = {0, 0, 0};  // two bits a stage: the set of its last copy; a bit: that set's phase
      uint32_t mine = 0;                        // stages with a copy of this warp's last
      int k = 0, place = 1;   // parts so far; the queries' place of the last one with one tile
      int uses[2] = {0, 0};   // of the two places
      bool ok = true;
      while (ok && w.t < t_end) {
        const int seg = static_cast<int>(min(static_cast<long long>(w.u.n - w.local), t_end - w.t));
        const bool both = w.u.c1 > 0;
        const int32_t* table = p.a.block_table + w.u.r * p.a.table_stride;
        // lane l holds the page of chunk pbase + l; the next 32 are on their way
        int pbase = 0, pg = 0, pg_next = 0;
        bool in_next = false;
        auto page_at = [&](int c) {
          const long long key = static_cast<long long>(c + lane) << box_shift;
          in_next = key <= w.u.hi && key + box > w.u.lo;
          return in_next ? table[key >> p.a.page_shift] : 0;
        };
        const int c_first = (w.u.kb + w.local * kPtTile) >> box_shift;
        pg_next = page_at(c_first);
        pbase = c_first - 32;
        if (!kv) {
          if (!both) place ^= 1;
          for (int s = 0; s < 2 && ok; ++s)
            if ((both || s == place) && uses[s] > 0) ok = wait(&q_empty[s], (uses[s] - 1) & 1);
          if (!ok) break;
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
            d.first = w.u.qb * p.unit_tok;
            d.c0 = w.u.c0;
            d.c1 = w.u.c1;
            d.h = w.h;
            d.part = whole ? -1 : k > 0 ? 1 : 0;
            d.q = place | (uses[0] & 1) << 1 | (uses[1] & 1) << 2;
            d.last = w.t + seg >= t_end;
            d.pad[0] = d.pad[1] = 0;
            segs[k & 3] = d;
            mbar_arrive(&seg_full[k & 3]);
            if (!whole && w.local == 0) {  // it starts here and ends in another CTA's share
              PagedCut c;
              int first, slot1;
              tree_owners(share, w, first, c.g_last, slot1);
              c.tok0 = d.tok0 + d.first;
              c.tok1 = c.tok0 + d.c0 + d.c1;
              c.h = w.h;
              c.slot1 = d.part;
              c.pad[0] = c.pad[1] = c.pad[2] = 0;
              p.cuts[blockIdx.x] = c;
            }
            for (int s = 0; s < 2; ++s) {
              if (!both && s != place) continue;
              if (both) mbar_arrive(&q_empty[s]);  // one group reads it; the other's arrival
              mbar_arrive_expect_tx(&q_full[s], Cfg::kPanels * q_bytes);
#pragma unroll
              for (int pn = 0; pn < Cfg::kPanels; ++pn)
                tma_load_3d(smem + s * Cfg::kTileBytes + pn * kPtTile * 128, &qmap, &q_full[s], pn * 64, w.h * p.a.G,
                            d.tok0 + d.first + (both ? s * p.a.tpb : 0), policy);
            }
          }
          __syncwarp();
          for (int s = 0; s < 2; ++s) uses[s] += both || s == place;
          ++k;
        }
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
          const int set = both ? 2 : i & 1;
          uint64_t* bar = full + set * ST + st;
          if (lane == 0) {
            if (!both) mbar_arrive(&empty[st]);  // one group reads it; the other's arrival
            mbar_arrive_expect_tx(bar, bytes);
          }
          mine |= 1u << st;
          sets = (sets & ~(3u << 2 * st)) | static_cast<uint32_t>(set) << 2 * st;
#pragma unroll
          for (int x = 0; x < 3; ++x) armed[x] ^= x == set ? 1u << st : 0u;
          __syncwarp();
          if (load) tma_load_4d(smem + lane_dst + st * Cfg::kTileBytes, map, bar, 0, pos, lpn, row, policy);
          __syncwarp();
        }
        if (!ok) break;
        w.t += seg;
        w.local += seg;
        if (w.local == w.u.n && w.t < t_end) tree_next(p, w);
      }
      if (*abort_flag && lane == 0) {  // the copies in flight land before the CTA can exit
        for (int st = 0; st < ST; ++st) {
          if (!(mine >> st & 1)) continue;
          const int set = sets >> 2 * st & 3;
          const uint32_t a = set == 0 ? armed[0] : set == 1 ? armed[1] : armed[2];
          mbar_wait(full + set * ST + st, ((a >> st) & 1) ^ 1);
        }
        for (int s = 0; s < 2; ++s)
          if (uses[s] > 0) mbar_wait(&q_full[s], (uses[s] - 1) & 1);
      }
      __syncwarp();
    } else if (warp < 3) {
      // ---------------- product issuers, one a group ----------------
      constexpr uint32_t idesc_s = umma_idesc_bf16(128, 64, 0);
      constexpr uint32_t idesc_o = umma_idesc_bf16(128, D, 1);
      tree_fill(p.a, D, threadIdx.x - 32, 64);
      const int t = __shfl_sync(0xffffffffu, warp - 1, 0);
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      const uint32_t s_col = tm + t * kPtTile, o_col = tm + Cfg::kOCol + t * D;
      const uint64_t q0_desc = smem_desc_sw128(base, 16, 1024);
      const uint64_t k0_desc = smem_desc_sw128(base + Cfg::kRingOff, 16, 1024);
      const uint64_t v0_desc = smem_desc_sw128(base + Cfg::kRingOff, kPtTile * 128, 1024);
      uint32_t g = 0, cnt = 0;  // key tiles of the parts before; this group's own products'
      uint32_t own_phase = 0, both_phase = 0;  // a bit a stage: the phases of this group's set and of both's
      auto landed = [&](bool both, uint32_t st, bool poll) {
        uint64_t* bar = full + (both ? 2 : t) * ST + st;
        const uint32_t parity = (both ? both_phase : own_phase) >> st & 1;
        if (poll) {
          if (!__all_sync(0xffffffffu, mbar_test_wait(bar, parity))) return false;
        } else if (!wait(bar, parity)) {
          return false;
        }
        if (both) both_phase ^= 1u << st;
        else own_phase ^= 1u << st;
        return true;
      };
      bool ok = true;
      TreeSeg d;
      d.last = t_begin >= t_end;
      for (int k = 0; ok && !d.last; ++k) {
        if (!(ok = next_seg(k, d))) break;
        const bool both = d.c1 > 0;
        const int place = both ? t : d.q & 1, step = both ? 1 : 2, j0 = both ? 0 : t;
        const uint64_t q_desc = q0_desc + place * (Cfg::kTileBytes >> 4);
        if (j0 >= d.seg) {
          if (lane == 0) mbar_arrive(&q_empty[place]);
        } else {
          ok = wait(&q_full[place], (d.q >> (1 + place)) & 1);
        }
        // Half by half: P V of key tile j and, over its S, the S of this group's next one (first both
        // halves' S of the part's first tile).
#pragma unroll 1
        for (int j = j0 - step; ok && j0 < d.seg && j < d.seg; j += step) {
          const bool pv = j >= j0, sn = j + step < d.seg;
          const uint32_t sv = SK + (g + j) % SV, sk = (g + j + step) % SK;
          if (pv) {
            if (!(ok = landed(both, sv, false))) break;
            const int kt = d.kt0 + j * kPtTile;
            if ((kt < d.lo || kt + kPtTile - 1 > d.hi) && lane == 0) mbar_arrive(&v_ready[t]);
          }
          auto issue_pv = [&](int h) {
            if (!(ok = wait(&p_full[t * 2 + h], cnt & 1))) return;
            // (a part's first product overwrites O_t: the last part's has been read)
            if (j == j0 && h == 0 && k > 0 && !(ok = wait(&epi_done[t], (k - 1) & 1))) return;
            tc_fence_after();
            if (elect_one()) {
              const uint64_t va = v0_desc + sv * (Cfg::kTileBytes >> 4) + h * ((64 * 128) >> 4);
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                umma_ts(o_col, s_col + h * 64 + kk * 8, va + kk * ((16 * 128) >> 4), idesc_o,
                        kk > 0 || h > 0 || j > j0 ? 1u : 0u);
              umma_commit(&pv_done[t]);
              if (h) umma_commit(&empty[sv]);
              if (h && !sn) umma_commit(&o_done[t]);
            }
            __syncwarp();
          };
          auto issue_s = [&](int h) {
            tc_fence_after();
            if (elect_one()) {
              const uint64_t ka = k0_desc + sk * (Cfg::kTileBytes >> 4) + h * ((64 * 128) >> 4);
#pragma unroll
              for (int kk = 0; kk < D / 16; ++kk) {
                const int off = (kk >> 2) * ((kPtTile * 128) >> 4) + (kk & 3) * (32 >> 4);
                umma_ss(s_col + h * 64, q_desc + off, ka + off, idesc_s, kk > 0 ? 1u : 0u);
              }
              umma_commit(&s_full[t * 2 + h]);
              if (h) umma_commit(&empty[sk]);
              if (h && j + 2 * step >= d.seg) umma_commit(&q_empty[place]);
            }
            __syncwarp();
          };
          // S of the next tile's first half goes between the two P V where its keys are there already
          bool first_s = false;
          if (pv) {
            issue_pv(0);
            if (!ok) break;
            if (sn && landed(both, sk, true)) {
              issue_s(0);
              first_s = true;
            }
            issue_pv(1);
            if (!ok) break;
          }
          if (sn) {
            if (!first_s) {
              if (!(ok = landed(both, sk, false))) break;
              issue_s(0);
            }
            issue_s(1);
          }
          cnt += pv;
        }
        g += d.seg;
      }
      if (elect_one()) umma_commit(drained);  // every product has completed before TMEM is freed
      __syncwarp();
      mbar_wait(drained, 0);
      __syncwarp();
    }
  } else {
    // ---------------- softmax: four warps a group, a thread a query row ----------------
    const int t = (warp - 4) >> 2, quarter = warp & 3;  // group; TMEM lanes 32 * quarter .. +31
    const int row = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_addr = tmem + lane_off + t * kPtTile;  // S, and P over it
    const uint32_t o_addr = tmem + lane_off + Cfg::kOCol;   // O_0; O_1 D columns on
    const int rt = row / p.a.G;                             // the row's token in its tile
    const float sc = p.a.scale_log2;
    const uint64_t sc2 = pair_f32(sc, sc);
    uint32_t g = 0, cnt = 0, all_halves = 0, edges = 0, ends = 0, ex = 0;
    bool ok = true;
    // the other group's v of this row (both warps of the quarter take part)
    auto exchange = [&](float v) -> float {
      xch[t * kPtTile + row] = v;
      __syncwarp();
      if (lane == 0) mbar_arrive(&pair_bar[quarter]);
      if (!wait(&pair_bar[quarter], ex++ & 1)) ok = false;
      const float o = xch[(t ^ 1) * kPtTile + row];
      __syncwarp();
      if (lane == 0) mbar_arrive(&pair_bar[quarter]);  // read: the slots are free again
      if (!wait(&pair_bar[quarter], ex++ & 1)) ok = false;
      return o;
    };
    TreeSeg d;
    d.last = t_begin >= t_end;
    for (int k = 0; ok && !d.last; ++k) {
      if (!(ok = next_seg(k, d))) break;
      const bool both = d.c1 > 0, causal = d.T > 32 * p.words;
      const int tile = both ? t : 0, step = both ? 1 : 2;
      const int local = d.first + tile * p.a.tpb + rt;  // the row's token, counted from the request's first
      const bool valid = rt < (tile ? d.c1 : d.c0);     // (rows past tpb * G have rt >= tpb)
      int pos = d.L, tok = -1, see_lo = 0, see_hi = -1;
      if (valid) {
        pos = causal ? d.L + local : max(p.positions[d.tok0 + local], d.L);
        tok = causal ? -1 : d.tok0 + local;
        see_lo = p.a.window >= 0 ? max(pos - p.a.window, 0) : 0;
        see_hi = min(causal ? pos : d.L - 1, d.hi);
      }
      const bool warp_rows = __any_sync(0xffffffffu, valid);
      float m_used = -INFINITY, l = 0.f;
      int halves = 0;  // of this group's, of the part
      for (int j = both ? 0 : t; j < d.seg; j += step, ++cnt) {
        const int kt = d.kt0 + j * kPtTile;
        if (kt < d.lo || kt + kPtTile - 1 > d.hi) {
          // rows of V outside [lo, hi] to zero, a thread a row
          if (!(ok = wait(&v_ready[t], edges++ & 1))) break;
          if (kt + row < d.lo || kt + row > d.hi) {
            const uint32_t at = base + Cfg::kRingOff + (SK + (g + j) % SV) * Cfg::kTileBytes + row * 128;
#pragma unroll
            for (int c = 0; c < 8 * Cfg::kPanels; ++c)
              sts128(at + (c >> 3) * (kPtTile * 128) + (c & 7) * 16, make_uint4(0, 0, 0, 0));
          }
          fence_proxy_async_shared();
        }
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          const int k0 = kt + h * 64;
          const bool plain = __all_sync(0xffffffffu, !valid || (k0 >= see_lo && k0 + 63 <= see_hi));
          uint32_t bits[2];
          if (!plain && warp_rows)
#pragma unroll
            for (int c = 0; c < 2; ++c) bits[c] = tree_bits(p, see_lo, see_hi, d.L, d.T, d.tok0, tok, pos, k0 + 32 * c);
          if (!(ok = wait(&s_full[t * 2 + h], cnt & 1))) break;
          tc_fence_after();
          if (warp_rows) {  // (else P may be anything)
            uint32_t s[64];
            tmem_ld64(s_addr + h * 64, s);
            if (!plain)
#pragma unroll
              for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int e = 0; e < 32; ++e)
                  if (!(bits[c] >> e & 1)) s[32 * c + e] = __float_as_uint(-INFINITY);
            float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
#pragma unroll
            for (int e = 0; e < 64; e += 8) {
              mx0 = fmax3(mx0, __uint_as_float(s[e]), __uint_as_float(s[e + 1]));
              mx1 = fmax3(mx1, __uint_as_float(s[e + 2]), __uint_as_float(s[e + 3]));
              mx2 = fmax3(mx2, __uint_as_float(s[e + 4]), __uint_as_float(s[e + 5]));
              mx3 = fmax3(mx3, __uint_as_float(s[e + 6]), __uint_as_float(s[e + 7]));
            }
            const float mx = fmaxf(fmax3(mx0, mx1, mx2), mx3) * sc;
            float alpha = 1.f;
            if (mx > m_used + 8.f) {
              alpha = fast_exp2(m_used - mx);  // 0 when m was -inf
              m_used = mx;
              l *= alpha;
            }
            if (halves > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
              // the half's before: the one product that S does not say is complete
              if (!(ok = wait(&pv_done[t], (all_halves - 1) & 1))) break;
              tc_fence_after();
              tmem_scale(o_addr + t * D, D, alpha);
            }
            const float neg_m = m_used == -INFINITY ? 0.f : -m_used;
            const uint64_t nm2 = pair_f32(neg_m, neg_m);
            uint64_t acc0 = 0, acc1 = 0;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              uint32_t w[16];
              exp32(*reinterpret_cast<const uint32_t(*)[32]>(&s[32 * c]), sc2, nm2, w, acc0, acc1);
              tmem_st16_nowait(s_addr + h * 64 + 16 * c, w);
            }
            acc0 = add2(acc0, acc1);
            l += lo_f(acc0) + hi_f(acc0);
            tmem_st_wait();
          }
          ++halves;
          ++all_halves;
          tc_fence_before();
          mbar_arrive(&p_full[t * 2 + h]);
        }
        if (!ok) break;
      }
      if (!ok) break;
      if (halves > 0 && !(ok = wait(&o_done[t], ends++ & 1))) break;
      tc_fence_after();
      if (__any_sync(0xffffffffu, valid) || !both) {
        float w_own = 0.f, w_other = 0.f, lse;
        if (both) {
          w_own = l == 0.f ? 0.f : 1.f / l;  // (a NaN stays one)
          lse = l == 0.f ? -INFINITY : m_used + __log2f(l);
        } else {
          tc_fence_before();
          const float m_other = exchange(m_used);  // (and the other group's O is complete)
          const float m = fmaxf(m_used, m_other);
          const float f_own = m_used == -INFINITY ? 0.f : fast_exp2(m_used - m);
          const float f_other = m_other == -INFINITY ? 0.f : fast_exp2(m_other - m);
          // (a sum of NaN under a maximum of -inf: every score was a NaN)
          const float l_own = m_used == -INFINITY ? l : l * f_own, l_other = exchange(l_own);
          tc_fence_after();
          const float all = t ? l_other + l_own : l_own + l_other;
          const float inv = all == 0.f ? 0.f : 1.f / all;
          w_own = all != all ? all : f_own * inv;
          w_other = all != all ? all : f_other * inv;
          lse = all == 0.f ? -INFINITY : (m == -INFINITY ? all : m + __log2f(all));
        }
        if (!ok) break;
        const long long slot = static_cast<long long>(blockIdx.x) * 2 + d.part;
        const int prow = tile * kPtTile + row;
        if (d.part >= 0 && valid && (both || t == 0)) p.a.part_lse[slot * 256 + prow] = lse;
        const int orow = valid ? (d.tok0 + local) * p.a.Hq + d.h * p.a.G + (row - rt * p.a.G) : -1;
        if (both) {
          float* part = d.part < 0 ? nullptr : p.a.part_o + (slot * (D / 4) * 256 + prow) * 4;
          tree_store<D>(o_addr + t * D, 0, w_own, 0.f, orow, p.a.out, D, part);
        } else {  // half of the columns each
          float* part = d.part < 0 ? nullptr : p.a.part_o + ((slot * (D / 4) + t * (D / 8)) * 256 + prow) * 4;
          tree_store<D / 2>(o_addr + t * (D / 2), o_addr + D + t * (D / 2), t ? w_other : w_own, t ? w_own : w_other, orow,
                            p.a.out + t * (D / 2), D, part);
          tc_fence_before();
          exchange(0.f);  // both have read both
        }
      }
      tc_fence_before();
      mbar_arrive(&epi_done[t]);  // O is read: the issuer may overwrite it
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
}

// Merges the units cut between CTAs: blockIdx.x is the CTA whose share the unit starts in, blockIdx.y
// 32 of its rows.  A lane is a row, a warp takes every eighth group of four columns (the partials' layout: a
// load is 512 contiguous bytes), two groups and four contributors' loads on their way at once; the rows
// leave through shared memory, whole.
constexpr int kTreeMostCuts = 160;  // contributors (no GPU of these has as many SMs)
template <int D>
__global__ void __launch_bounds__(256) tree_combine_kernel(const PagedTreeParams p) {
  __shared__ float weight[kTreeMostCuts][32];
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
  const int cnt = min(c.g_last - static_cast<int>(blockIdx.x) + 1, kTreeMostCuts);
  auto slot = [&](int k) { return (static_cast<long long>(blockIdx.x) + k) * 2 + (k == 0 && c.slot1 ? 1 : 0); };
  for (int k = warp; k < cnt; k += 8) weight[k][lane] = valid ? __ldcg(p.a.part_lse + slot(k) * 256 + n) : -CUDART_INF_F;
  __syncthreads();
  float mx = -CUDART_INF_F, wsum = 0.f;
  for (int k = 0; k < cnt; ++k) mx = fmaxf(mx, weight[k][lane]);
  for (int k = 0; k < cnt; ++k) {
    const float ls = weight[k][lane];
    wsum += ls == -CUDART_INF_F ? 0.f : fast_exp2(ls - mx);
  }
  const float inv = wsum == 0.f ? 0.f : 1.f / wsum;
  __syncthreads();
  for (int k = warp; k < cnt; k += 8) {
    const float ls = weight[k][lane];
    weight[k][lane] = ls == -CUDART_INF_F ? 0.f : fast_exp2(ls - mx) * inv;  // (0: its partial was not written)
  }
  if (warp == 0) out_row[lane] = valid ? tok * p.a.Hq + c.h * p.a.G + (rr - rt * p.a.G) : -1;
  __syncthreads();
#pragma unroll 1
  for (int q = warp; q < D / 4; q += 16) {
    float a[2][4] = {};
    const bool two = q + 8 < D / 4;
    for (int k0 = 0; k0 < cnt; k0 += 4) {
      float4 v[2][4];
      float w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = min(k0 + i, cnt - 1);
        w[i] = k0 + i < cnt ? weight[k][lane] : 0.f;
#pragma unroll
        for (int j = 0; j < 2; ++j)
          if (valid && (j == 0 || two))
            v[j][i] = __ldcg(reinterpret_cast<const float4*>(p.a.part_o) + (slot(k) * (D / 4) + q + 8 * j) * 256 + n);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (!valid || w[i] == 0.f) continue;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (j == 1 && !two) continue;
          a[j][0] = fmaf(w[i], v[j][i].x, a[j][0]);
          a[j][1] = fmaf(w[i], v[j][i].y, a[j][1]);
          a[j][2] = fmaf(w[i], v[j][i].z, a[j][2]);
          a[j][3] = fmaf(w[i], v[j][i].w, a[j][3]);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (j == 0 || two) rows[lane][q + 8 * j] = make_uint2(pack_bf16x2(a[j][0], a[j][1]), pack_bf16x2(a[j][2], a[j][3]));
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * (D / 4); i += 256) {
    const int r = i / (D / 4), q = i % (D / 4);
    if (out_row[r] >= 0)
      *reinterpret_cast<uint2*>(p.a.out + static_cast<long long>(out_row[r]) * D + 4 * q) = rows[r][q];
  }
}

}  // namespace mcb
