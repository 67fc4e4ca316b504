// Trees of drafted tokens: each token's position and ancestors, from the tokens' parents.
//
// Request r's new tokens [cu_r, cu_{r+1}) hang together by parents: p_t is an earlier token of the
// request's, or -1 where t follows the cached tokens.  With A_t the set of t and its ancestors,
//   A_t = {t} u A_{p_t},   position_t = L_r + |A_t| - 1,   mask bit j of t: j in A_t.
// The sets grow by doubling: after k rounds a token holds its 2^k nearest ancestors and a pointer to
// the next one, so a tree of T tokens takes log2 of its depth rounds whatever its shape.
//
// A request of more than 32 W tokens has no masks: it is a chunk of a prompt, its tokens follow each
// other (position L + t).  A CTA of 32 W threads a request; a few KB to a few MB of integers: bound by the
// launch and a chain of dependent loads (lengths, parents, a shared-memory round a doubling): 64 trees of 16 7.3 us as
// called, 1,000 of 200 beside chunks 11 us (7 MB, 1.1 us at HBM's rate).
#pragma once

#include "paged_plan.cuh"

namespace mcb {

constexpr int kTreeMaxWords = 8;

struct DraftTreeParams {
  const int32_t* parents;  // (N,)
  const int32_t* cu;       // (R + 1,)
  const int32_t* seqlens;  // (R,)
  int32_t* positions;      // (N,)
  uint32_t* mask;          // (N, W)
  int R, N;
};

__device__ __forceinline__ int position_add(int len, int n) {
  const long long p = static_cast<long long>(max(len, 0)) + n;
  return static_cast<int>(min(p, 2147483647ll));
}

template <int W>
__global__ void __launch_bounds__(32 * W) draft_tree_kernel(const DraftTreeParams p) {
  constexpr int THREADS = 32 * W;
  __shared__ int s_up[THREADS];
  __shared__ uint32_t s_bits[THREADS][W];
  pdl_wait();
  pdl_launch_dependents();
  const int t = threadIdx.x;
  for (int r = blockIdx.x; r < p.R; r += gridDim.x) {
    const int tok0 = min(max(p.cu[r], 0), p.N), T = min(max(p.cu[r + 1], tok0), p.N) - tok0;
    const int len = p.seqlens[r];
    if (T > THREADS) {
      for (int i = t; i < T; i += THREADS) p.positions[tok0 + i] = position_add(len, i);
      for (long long i = t; i < static_cast<long long>(T) * W; i += THREADS)
        p.mask[static_cast<long long>(tok0) * W + i] = 0;
      continue;
    }
    int up = -1;
    if (t < T) {
      up = p.parents[tok0 + t];
      if (up < -1 || up >= t) {
        record_error(kErrDraftOutOfRange);
        up = -1;
      }
    }
    uint32_t bits[W];
#pragma unroll
    for (int w = 0; w < W; ++w) bits[w] = (t >> 5) == w ? 1u << (t & 31) : 0u;
    while (__syncthreads_or(up >= 0)) {  // (all reads of the round before are done)
      s_up[t] = up;
#pragma unroll
      for (int w = 0; w < W; ++w) s_bits[t][w] = bits[w];
      __syncthreads();
      if (up >= 0) {
#pragma unroll
        for (int w = 0; w < W; ++w) bits[w] |= s_bits[up][w];
        up = s_up[up];
      }
    }
    if (t < T) {
      int n = -1;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        n += __popc(bits[w]);
        p.mask[static_cast<long long>(tok0 + t) * W + w] = bits[w];
      }
      p.positions[tok0 + t] = position_add(len, n);
    }
  }
  // tokens that no request has
  const int first = min(max(p.cu[0], 0), p.N), last = max(min(p.cu[p.R], p.N), first);
  for (int i = blockIdx.x * THREADS + t; i < p.N; i += gridDim.x * THREADS) {
    if (i >= first && i < last) continue;
    p.positions[i] = -1;
#pragma unroll
    for (int w = 0; w < W; ++w) p.mask[static_cast<long long>(i) * W + w] = 0;
  }
}

}  // namespace mcb
