// The append of packed new tokens to a paged cache: rope + QK-norm + scale of q and k, k and v
// written to their slots.
//
// Per head vector x = (x1, x2) of token t at position pos_t, c and s the rotary rows there:
//   y1 = x1 c + x2 s,  y2 = x2 c - x1 s,  z = y / sqrt(mean(y^2) + eps),  out = scale z
// round_each: every product, sum, norm and scale rounded to bf16, as modelcore's torch ops round
// (kv_append_rope's bits, so a paged cache holds what KVCache holds); otherwise fp32 throughout
// and one rounding at the end.
// K page layout (n_pages, Hkv, page, D): slot s is position s % page of page s / page.
//
// A warp takes a token (or, for few tokens, one of `parts` shares of its heads): the position, the
// slot and the rotary row are read once for all its heads -- a lane keeps the same 16 table values --
// and the heads go by in steps of 32 / (D/16) vectors, D/16 lanes each, the next step's loads in flight.
// With a vector's position and table row read per vector the two dependent loads ahead of every
// vector bounded it.  16,381 tokens of 16/4 heads of 128 (206 MB): 43 us so, 40 us now, 5.2 TB/s; two
// or more steps in flight cost registers and with them warps (44 to 65 us).  Every step rounded to bf16
// 41 us (both 33.5 at 12/12 heads of 64, 153 MB).  64 registers, with 28 bytes spilled in the form rounded once.
// Bound by HBM (each byte read and written once) for long batches, by launch and dependent-load
// latency for a decode step.
#pragma once

#include "common.cuh"
#include "kv_append.cuh"

namespace mcb {

struct PagedAppendParams {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  long long qs[2], ks[2], vs[2];  // element strides: token, head
  uint16_t* q_out;                // (N, Hq, D) contiguous
  uint16_t* k_pages;              // (n_pages, Hkv, page, D)
  uint16_t* v_pages;
  const int32_t* positions;       // (N,), -1: padding (q_out zeroed)
  const long long* slot_map;      // (N,), -1: not written
  const uint16_t* cos;
  const uint16_t* sin;
  int N, Hq, Hkv, page_shift, rot_len;
  long long n_slots;              // n_pages * page
  float eps, scale;
  int nk;                         // key (and value) vectors a token: Hkv, or 0 without k and v
  int rotate_k;
  int parts;                      // warps a token
};

// rope_norm_vec_tab with every step in fp32 and one rounding: products and sums fused.
template <int D>
__device__ __forceinline__ void rope_norm_vec_once(const uint4& x1v, const uint4& x2v, const uint4& cv,
                                                   const uint4& sv, bool rotate, float eps, float scale, uint4& w1,
                                                   uint4& w2) {
  constexpr int L = D / 16;
  float x1[8], x2[8], c[8], s[8];
  unpack8(x1v, x1);
  unpack8(x2v, x2);
  unpack8(cv, c);
  unpack8(sv, s);
  float acc = 0.f;
  if (rotate) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = fmaf(x1[i], c[i], x2[i] * s[i]), b = fmaf(x2[i], c[i], -(x1[i] * s[i]));
      x1[i] = a;
      x2[i] = b;
      acc = fmaf(a, a, fmaf(b, b, acc));
    }
  }
#pragma unroll
  for (int m = L / 2; m >= 1; m >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, m);
  if (rotate) {
    const float r = rsqrtf(acc * (1.f / D) + eps) * scale;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x1[i] *= r;
      x2[i] *= r;
    }
    w1 = pack8(x1);
    w2 = pack8(x2);
  } else {
    w1 = x1v;
    w2 = x2v;
  }
}

template <int D, bool EACH>
__global__ void __launch_bounds__(kAppendVecThreads, 4) paged_append_kernel(const PagedAppendParams p) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int L = D / 16, VPW = 32 / L, HALF = D / 2;
  const int lane = threadIdx.x & 31, sub = lane % L;
  const int heads = p.Hq + 2 * p.nk;
  const long long items = static_cast<long long>(p.N) * p.parts;
  const long long warps = static_cast<long long>(gridDim.x) * (kAppendVecThreads / 32);
  for (long long item = static_cast<long long>(blockIdx.x) * (kAppendVecThreads / 32) + (threadIdx.x >> 5);
       item < items; item += warps) {
    const int t = static_cast<int>(item / p.parts), part = static_cast<int>(item - static_cast<long long>(t) * p.parts);
    const int pos = p.positions[t];
    const long long slot = p.nk > 0 ? p.slot_map[t] : -1;
    auto load = [&](int j, uint4& x1, uint4& x2) {
      x1 = x2 = make_uint4(0, 0, 0, 0);
      if (j >= heads) return;
      const uint16_t* src = j < p.Hq          ? p.q + t * p.qs[0] + j * p.qs[1]
                            : j < p.Hq + p.nk ? p.k + t * p.ks[0] + (j - p.Hq) * p.ks[1]
                                              : p.v + t * p.vs[0] + (j - p.Hq - p.nk) * p.vs[1];
      x1 = *reinterpret_cast<const uint4*>(src + 8 * sub);
      x2 = *reinterpret_cast<const uint4*>(src + HALF + 8 * sub);
    };
    const int step = p.parts * VPW;
    int j = part * VPW + lane / L;
    uint4 x1, x2;
    load(j, x1, x2);
    const bool rot_ok = pos >= 0 && pos < p.rot_len;
    if (pos >= p.rot_len && part == 0 && lane == 0) record_error(kErrPositionBeyondRotary);
    const bool slot_ok = slot >= 0 && slot < p.n_slots;
    if (slot >= p.n_slots && part == 0 && lane == 0) record_error(kErrPageOutOfRange);
    uint4 cv = make_uint4(0, 0, 0, 0), sv = cv;
    if (rot_ok) {
      const long long row = static_cast<long long>(pos) * HALF + 8 * sub;
      cv = *reinterpret_cast<const uint4*>(p.cos + row);
      sv = *reinterpret_cast<const uint4*>(p.sin + row);
    }
    // the slot's row for head 0; a head further is one page of one head further
    const long long slot_row = ((slot >> p.page_shift) * p.Hkv << p.page_shift) + (slot & ((1ll << p.page_shift) - 1));
#pragma unroll 1
    for (int j0 = part * VPW; j0 < heads; j0 += step, j += step) {  // warp-uniform
      const uint4 a = x1, b = x2;
      if (j0 + step < heads) load(j + step, x1, x2);
      const bool is_q = j < p.Hq, is_k = !is_q && j < p.Hq + p.nk;
      const bool turn = is_q || (is_k && p.rotate_k);
      uint4 w1, w2;  // every lane takes part in the butterfly
      if constexpr (EACH) rope_norm_vec_tab<D>(a, b, cv, sv, turn && rot_ok, p.eps, p.scale, w1, w2);
      else rope_norm_vec_once<D>(a, b, cv, sv, turn && rot_ok, p.eps, p.scale, w1, w2);
      if (j >= heads) continue;
      uint16_t* dst;
      if (is_q) {
        if (!rot_ok) w1 = w2 = make_uint4(0, 0, 0, 0);  // a padding token
        dst = p.q_out + (static_cast<long long>(t) * p.Hq + j) * D;
      } else {
        if (!slot_ok || (turn && !rot_ok)) continue;
        const int h = is_k ? j - p.Hq : j - p.Hq - p.nk;
        dst = (is_k ? p.k_pages : p.v_pages) + (slot_row + (static_cast<long long>(h) << p.page_shift)) * D;
      }
      *reinterpret_cast<uint4*>(dst + 8 * sub) = w1;
      *reinterpret_cast<uint4*>(dst + HALF + 8 * sub) = w2;
    }
  }
}

}  // namespace mcb
