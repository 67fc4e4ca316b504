// Attention of trees of drafted tokens over a paged cache.
//
//   out[t, h] = sum_c softmax_c(q[t, h] . K[c, h / G] * softmax_scale) V[c, h / G]
// over the cached keys c < L with position_t - c <= window, and the request's new tokens j with mask
// bit j of t and position_t - position_j <= window (window < 0: all).  A request of more new tokens
// than the mask has bits is a chunk of a prompt: token t sees the new tokens up to itself.
#pragma once

#include "paged_decode.cuh"

namespace mcb {

struct PagedTreeParams {
  PagedAttnParams a;
  const uint16_t* k_pages;
  const uint16_t* v_pages;
  const int32_t* positions;  // (N,)
  const uint32_t* mask;      // (N, words)
  int words;
};

// One warp a token and query head, one key after another.
template <int D>
__global__ void __launch_bounds__(128) paged_tree_simple_kernel(const PagedTreeParams p) {
  constexpr int E = D / 32;
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const long long id = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (id >= static_cast<long long>(p.a.N) * p.a.Hq) return;
  const int t = static_cast<int>(id / p.a.Hq), h = static_cast<int>(id % p.a.Hq), kvh = h / p.a.G;
  int r = 0;
  while (r < p.a.R && !(t >= p.a.cu_new[r] && t < p.a.cu_new[r + 1])) ++r;
  float acc[E] = {}, m = -CUDART_INF_F, l = 0.f;
  if (r < p.a.R) {
    const PagedRow x = paged_row(p.a, r);
    if (t == x.tok0 && h == 0 && lane == 0 && !paged_row_fits(p.a, r, x)) record_error(kErrPositionBeyondCache);
    const int i = t - x.tok0, page = 1 << p.a.page_shift;
    const bool chunk = x.T > 32 * p.words;
    const int pos = chunk ? x.L + i : max(p.positions[t], x.L);
    float q[E];
    for (int e = 0; e < E; ++e) q[e] = bf16_bits_to_float(p.a.q[t * p.a.qs[0] + h * p.a.qs[1] + lane * E + e]);
    for (int c = p.a.window >= 0 ? max(0, min(x.L, pos - p.a.window)) : 0; c < x.L + x.T; ++c) {
      const int j = c - x.L;
      if (j >= 0) {
        const bool seen = chunk ? j <= i : (p.mask[static_cast<long long>(t) * p.words + (j >> 5)] >> (j & 31)) & 1;
        const int kp = chunk ? c : max(p.positions[x.tok0 + j], x.L);
        if (!seen || (p.a.window >= 0 && pos - kp > p.a.window)) continue;
      }
      const int pg = p.a.block_table[r * p.a.table_stride + (c >> p.a.page_shift)];
      if (pg < 0 || pg >= p.a.n_pages) {
        record_error(kErrPageOutOfRange);
        continue;
      }
      const long long at = ((static_cast<long long>(pg) * p.a.Hkv + kvh) * page + (c & (page - 1))) * D + lane * E;
      float s = 0.f;
      for (int e = 0; e < E; ++e) s = fmaf(q[e], bf16_bits_to_float(p.k_pages[at + e]), s);
      for (int o = 16; o >= 1; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      s *= p.a.scale_log2;
      const float mn = fmaxf(m, s);
      if (mn == -CUDART_INF_F) continue;
      const float alpha = fast_exp2(m - mn), w = fast_exp2(s - mn);
      m = mn;
      l = fmaf(l, alpha, w);
      for (int e = 0; e < E; ++e) acc[e] = fmaf(acc[e], alpha, w * bf16_bits_to_float(p.v_pages[at + e]));
    }
  }
  for (int e = 0; e < E; ++e)
    p.a.out[id * D + lane * E + e] = float_to_bf16_bits(l == 0.f ? 0.f : acc[e] / l);
}

}  // namespace mcb
