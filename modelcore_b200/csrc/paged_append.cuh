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
// D/16 lanes a vector, 16-byte loads and stores, grid-stride over groups of vectors, two groups'
// loads in flight before either's arithmetic: kv_append_rope_vec_kernel's shape.  Bound by HBM
// (each byte read and written once) for long batches, by launch and dependent-load latency for
// a decode step.
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
  long long total_vectors;
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

struct PagedVec {
  int j, pos;
  long long slot;
  int t;
  bool active;
  uint4 x1v, x2v, cv, sv;
};

template <int D>
__device__ __forceinline__ void paged_vec_load(const PagedAppendParams& p, long long w, int sub, PagedVec& r) {
  constexpr int HALF = D / 2;
  r.active = w < p.total_vectors;
  const unsigned wv = r.active ? static_cast<unsigned>(w) : 0u;  // total_vectors < 2^31 (host)
  const unsigned per = static_cast<unsigned>(p.Hq + 2 * p.nk);
  r.t = static_cast<int>(wv / per);
  r.j = static_cast<int>(wv - static_cast<unsigned>(r.t) * per);
  const bool is_q = r.j < p.Hq, is_k = !is_q && r.j < p.Hq + p.nk;
  const uint16_t* src = is_q ? p.q + r.t * p.qs[0] + r.j * p.qs[1]
                       : is_k ? p.k + r.t * p.ks[0] + (r.j - p.Hq) * p.ks[1]
                              : p.v + r.t * p.vs[0] + (r.j - p.Hq - p.nk) * p.vs[1];
  r.pos = p.positions[r.t];
  r.slot = is_q ? 0 : p.slot_map[r.t];
  r.x1v = *reinterpret_cast<const uint4*>(src + 8 * sub);
  r.x2v = *reinterpret_cast<const uint4*>(src + HALF + 8 * sub);
}

template <int D>
__device__ __forceinline__ void paged_vec_tables(const PagedAppendParams& p, int sub, PagedVec& r) {
  r.cv = r.sv = make_uint4(0, 0, 0, 0);
  const bool is_v = r.j >= p.Hq + p.nk;
  if (r.active && !is_v && r.pos >= 0 && r.pos < p.rot_len) {
    const long long row = static_cast<long long>(r.pos) * (D / 2) + 8 * sub;
    r.cv = *reinterpret_cast<const uint4*>(p.cos + row);
    r.sv = *reinterpret_cast<const uint4*>(p.sin + row);
  }
}

template <int D, bool EACH>
__device__ __forceinline__ void paged_vec_store(const PagedAppendParams& p, const PagedVec& r, int sub) {
  constexpr int HALF = D / 2;
  const bool is_q = r.j < p.Hq, is_k = !is_q && r.j < p.Hq + p.nk;
  const bool turn = is_q || (is_k && p.rotate_k);
  bool rot_ok = r.pos >= 0;
  if (r.active && turn && r.pos >= p.rot_len) {
    if (sub == 0) record_error(kErrPositionBeyondRotary);
    rot_ok = false;
  }
  const bool rotate = r.active && turn && rot_ok;
  uint4 w1, w2;  // every lane takes part in the butterfly
  if constexpr (EACH) rope_norm_vec_tab<D>(r.x1v, r.x2v, r.cv, r.sv, rotate, p.eps, p.scale, w1, w2);
  else rope_norm_vec_once<D>(r.x1v, r.x2v, r.cv, r.sv, rotate, p.eps, p.scale, w1, w2);
  if (!r.active) return;
  uint16_t* dst;
  if (is_q) {
    if (!rotate) w1 = w2 = make_uint4(0, 0, 0, 0);  // a padding token
    dst = p.q_out + (static_cast<long long>(r.t) * p.Hq + r.j) * D;
  } else {
    if (r.slot < 0 || (turn && !rot_ok)) return;
    if (r.slot >= p.n_slots) {
      if (sub == 0) record_error(kErrPageOutOfRange);
      return;
    }
    const int h = is_k ? r.j - p.Hq : r.j - p.Hq - p.nk;
    const long long page = r.slot >> p.page_shift;
    const long long row = ((page * p.Hkv + h) << p.page_shift) + (r.slot & ((1ll << p.page_shift) - 1));
    dst = (is_k ? p.k_pages : p.v_pages) + row * D;
  }
  *reinterpret_cast<uint4*>(dst + 8 * sub) = w1;
  *reinterpret_cast<uint4*>(dst + HALF + 8 * sub) = w2;
}

template <int D, bool EACH>
__global__ void __launch_bounds__(kAppendVecThreads, 4) paged_append_kernel(const PagedAppendParams p) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int L = D / 16, VPW = 32 / L;
  const int lane = threadIdx.x & 31, sub = lane % L;
  const long long stride = static_cast<long long>(gridDim.x) * (kAppendVecThreads / 32) * VPW;
  const long long first =
      (static_cast<long long>(blockIdx.x) * (kAppendVecThreads / 32) + (threadIdx.x >> 5)) * VPW;
  constexpr int U = 2;
  for (long long base = first; base < p.total_vectors; base += U * stride) {  // warp-uniform
    PagedVec v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) paged_vec_load<D>(p, base + u * stride + lane / L, sub, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) paged_vec_tables<D>(p, sub, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) paged_vec_store<D, EACH>(p, v[u], sub);
  }
}

}  // namespace mcb
