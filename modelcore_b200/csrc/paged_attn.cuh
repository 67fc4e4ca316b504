// Attention of packed new tokens over a paged cache: the plain kernel, one warp a (token, q head).
//
//   out[t, h] = sum_c softmax_c(q[t, h] . K[c, h / G] * softmax_scale) V[c, h / G]
// over the keys c of the token's request with c <= pos and (window < 0 or pos - c <= window).
#pragma once

#include <math_constants.h>

#include "common.cuh"

namespace mcb {

struct PagedAttnParams {
  const uint16_t* q;
  long long qs[2];             // element strides: token, head
  const uint16_t* k_pages;     // (n_pages, Hkv, page, D)
  const uint16_t* v_pages;
  const int32_t* block_table;  // (R, max_pages)
  long long table_stride;
  const int32_t* seqlens;      // (R,)
  const int32_t* cu_new;       // (R + 1,)
  uint16_t* out;               // (N, Hq, D) contiguous
  int R, N, Hq, Hkv, G, n_pages, max_pages, page_shift, window;
  float scale_log2;
};

template <int D>
__global__ void __launch_bounds__(128) paged_attn_plain_kernel(const PagedAttnParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const long long w = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (w >= static_cast<long long>(p.N) * p.Hq) return;
  const int t = static_cast<int>(w / p.Hq), h = static_cast<int>(w % p.Hq);
  constexpr int E = D / 32;
  float o[E], qv[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  float m = -CUDART_INF_F, l = 0.f;
  if (t < p.cu_new[p.R]) {
    int lo = 0, hi = p.R;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (p.cu_new[mid] <= t) lo = mid;
      else hi = mid;
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
      qv[e] = bf16_bits_to_float(p.q[t * p.qs[0] + h * p.qs[1] + lane * E + e]) * p.scale_log2;
    const int pos = max(p.seqlens[lo], 0) + t - p.cu_new[lo];
    const long long cap = static_cast<long long>(p.max_pages) << p.page_shift;
    if (pos >= cap || p.seqlens[lo] < 0) record_error(kErrPositionBeyondCache);
    const int last = static_cast<int>(min(static_cast<long long>(pos), cap - 1));
    for (int c = p.window >= 0 ? max(0, pos - p.window) : 0; c <= last; ++c) {
      const int page = p.block_table[lo * p.table_stride + (c >> p.page_shift)];
      if (page < 0 || page >= p.n_pages) {
        record_error(kErrPageOutOfRange);
        continue;
      }
      const long long row = ((static_cast<long long>(page) * p.Hkv + h / p.G) << p.page_shift) +
                            (c & ((1 << p.page_shift) - 1));
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) s = fmaf(qv[e], bf16_bits_to_float(p.k_pages[row * D + lane * E + e]), s);
#pragma unroll
      for (int x = 16; x >= 1; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
      const float mn = fmaxf(m, s), a = exp2f(m - mn), pr = exp2f(s - mn);
      m = mn;
      l = fmaf(l, a, pr);
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = fmaf(o[e], a, pr * bf16_bits_to_float(p.v_pages[row * D + lane * E + e]));
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) p.out[w * D + lane * E + e] = float_to_bf16_bits(o[e] * inv);
}

}  // namespace mcb
