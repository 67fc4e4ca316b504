// Verification of drafted tokens against the target's probabilities.
//
// Request r's tokens [cu_r, cu_{r+1}) are a tree: token 0 is part of the answer already, each other one
// was drafted to follow its parent.  A walk from token 0 at token u, with p = softmax(logits_u / T),
// takes u's children c_1, c_2, ... in order, x_i the token of c_i, a_i its uniform:
//   rest_0 = p;   c_i is kept when a_i q(x_i) |rest| < rest(x_i), |rest| the sum of rest,
//   otherwise     rest <- max(rest / |rest| - q, 0)   with q = draft_probs_u, of which the x_i were drawn
//                 rest <- rest, but rest(x_i) = 0     without draft_probs: q is 1 at x_i
//   (rest = p again should nothing be left of it).
// The walk goes on at a kept child; where none is kept the next token is the first x with
//   rest(0) + ... + rest(x) > draw |rest|.
// So the tokens are distributed as if each had been drawn from its p, whatever the draft was.  T = 0: a
// child is kept when its token is the first one of the largest logit, which is the next token otherwise.
//
// Only the rows on the walk are read: a cluster of C CTAs a request, the vocabulary divided among them.
// Weights, their sums and the draw are in 64 bits: a vocabulary of 10^5 has borders everywhere, and
// 32-bit sums put a draw on their wrong side now and then.  Every CTA takes the walk's decisions itself,
// from the same numbers, exchanged through distributed shared memory.
#pragma once

#include "paged_plan.cuh"

namespace mcb {

constexpr int kVerifyThreads = 512;
constexpr int kVerifyWarps = kVerifyThreads / 32;
constexpr int kVerifyMaxTried = 256;  // children of a token that are tried

struct VerifyParams {
  const void* logits;          // (N, V)
  long long logits_stride;
  const long long* tokens;     // (N,)
  const int32_t* parents;      // (N,)
  const int32_t* cu;           // (R + 1,)
  const float* accept;         // (N,)
  const float* draws;          // (R,)
  const float* draft;          // (N, V) or null
  long long draft_stride;
  int32_t* accepted;           // (R,)
  int32_t* path;               // (R, max_path)
  long long* next;             // (R,)
  int R, N, V, max_path;
  float temperature;
};

__device__ __forceinline__ float logit_of(const float* p) { return *p; }
__device__ __forceinline__ float logit_of(const uint16_t* p) { return bf16_bits_to_float(*p); }

__device__ __forceinline__ void st_dsmem_f64(uint32_t addr, double v) {
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(addr), "d"(v) : "memory");
}

struct VerifyShared {
  double xch[2][8];              // what the cluster's CTAs exchange
  double warp_sum[kVerifyWarps]; // this CTA's warps' sums of the last pass
  double part[kVerifyWarps];
  double inv_mass[kVerifyMaxTried];  // with draft: 1 / |rest| after each refused child
  long long gone[kVerifyMaxTried];   // without: the refused tokens
  int child;
  int tried;
};

template <typename T>
__global__ void __launch_bounds__(kVerifyThreads) verify_kernel(const VerifyParams p) {
  __shared__ VerifyShared s;
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t rank, C;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(C));
  const int r = blockIdx.x / C;
  const int tok0 = min(max(p.cu[r], 0), p.N), count = min(max(p.cu[r + 1], tok0), p.N) - tok0;
  // this warp's tokens [v0, v1) of the vocabulary
  const int nw = C * kVerifyWarps, wi = rank * kVerifyWarps + warp;
  const int per = (p.V + nw - 1) / nw;
  const int v0 = static_cast<int>(min(static_cast<long long>(wi) * per, static_cast<long long>(p.V)));
  const int v1 = min(v0 + per, p.V);
  int phase = 0;
  // A value of every CTA to all of them (thread 0's), reduced in the CTAs' order.
  auto exchange = [&](double v, auto reduce) -> double {
    if (tid == 0)
      for (uint32_t c = 0; c < C; ++c) st_dsmem_f64(map_to_rank(&s.xch[phase][rank], c), v);
    cluster_sync();
    double a = s.xch[phase][0];
    for (uint32_t c = 1; c < C; ++c) a = reduce(a, s.xch[phase][c]);
    phase ^= 1;
    return a;
  };
  auto add = [](double a, double b) { return a + b; };
  auto greater = [](double a, double b) { return a != a || a > b ? a : b; };  // (a NaN stays)
  // A value of every thread, reduced over the CTA in order; the warps' values stay in warp_sum.
  auto block_reduce = [&](double v, auto reduce) -> double {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) v = reduce(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if (lane == 0) s.warp_sum[warp] = v;
    __syncthreads();
    double a = s.warp_sum[0];
    for (int w = 1; w < kVerifyWarps; ++w) a = reduce(a, s.warp_sum[w]);
    return a;
  };
  const double inv_t = p.temperature > 0.f ? 1.0 / static_cast<double>(p.temperature) : 1.0;
  const bool greedy = p.temperature == 0.f;
  int node = 0, kept = 0;
  long long answer = -1;
  while (count > 0) {
    if (rank == 0 && tid == 0 && kept < p.max_path) p.path[static_cast<long long>(r) * p.max_path + kept] = node;
    ++kept;
    const T* row = static_cast<const T*>(p.logits) + (tok0 + node) * p.logits_stride;
    const float* q = p.draft != nullptr && !greedy ? p.draft + (tok0 + node) * p.draft_stride : nullptr;
    // ---- the largest logit ----
    double mx = -CUDART_INF;
    bool nan = false;
    for (int i = v0 + lane; i < v1; i += 32) {
      const double x = logit_of(row + i);
      nan |= x != x;
      mx = fmax(mx, x);
    }
    if (nan) mx = CUDART_NAN;
    const double top = exchange(block_reduce(mx, greater), greater);
    if (!(top > -CUDART_INF && top < CUDART_INF)) {  // NaN, an infinity, or no token at all
      if (rank == 0 && tid == 0) record_error(kErrNoProbabilities);
      break;
    }
    double total = 0.0;
    long long best = -1;
    if (greedy) {
      int first = p.V;
      for (int i = v0 + lane; i < v1 && first == p.V; i += 32)
        if (logit_of(row + i) == top) first = i;
      auto less = [](double a, double b) { return a < b ? a : b; };
      best = static_cast<long long>(exchange(block_reduce(static_cast<double>(first), less), less));
    } else {
      double sum = 0.0;
      for (int i = v0 + lane; i < v1; i += 32) sum += exp((logit_of(row + i) - top) * inv_t);
      total = exchange(block_reduce(sum, add), add);
    }
    // ---- its children in turn ----
    const double inv_total = 1.0 / total;
    double mass = 1.0;
    int tried = 0;  // refused so far (0 again where nothing was left)
    auto rest = [&](int x) {  // of p, after the refused children
      double v = exp((logit_of(row + x) - top) * inv_t) * inv_total;
      if (q != nullptr) {
        for (int k = 0; k < tried; ++k) v = fmax(v * s.inv_mass[k] - static_cast<double>(q[x]), 0.0);
      } else {
        for (int k = 0; k < tried; ++k)
          if (s.gone[k] == x) v = 0.0;
      }
      return v;
    };
    auto rest_sum = [&] {
      double sum = 0.0;
      for (int i = v0 + lane; i < v1; i += 32) sum += rest(i);
      return exchange(block_reduce(sum, add), add);
    };
    int next = -1, last = node;
    for (int tries = 0; kept < p.max_path && tries < kVerifyMaxTried; ++tries) {
      if (warp == 0) {  // the next child
        int found = -1;
        for (int j0 = last + 1; j0 < count && found < 0; j0 += 32) {
          const int j = j0 + lane;
          const unsigned b = __ballot_sync(0xffffffffu, j < count && p.parents[tok0 + j] == node);
          if (b) found = j0 + __ffs(b) - 1;
        }
        if (lane == 0) s.child = found;
      }
      __syncthreads();
      const int c = s.child;
      if (c < 0) break;
      last = c;
      const long long x = p.tokens[tok0 + c];
      if (x < 0 || x >= p.V) {
        if (rank == 0 && tid == 0) record_error(kErrTokenOutOfRange);
        __syncthreads();
        continue;
      }
      if (greedy) {
        if (x == best) next = c;
      } else {
        const double of_draft = q != nullptr ? static_cast<double>(q[x]) : 1.0;
        if (static_cast<double>(p.accept[tok0 + c]) * of_draft * mass < rest(static_cast<int>(x))) next = c;
      }
      __syncthreads();
      if (next >= 0) break;
      if (greedy) continue;
      if (tid == 0) {
        if (q != nullptr) s.inv_mass[tried] = 1.0 / mass;
        else s.gone[tried] = x;
      }
      ++tried;
      __syncthreads();
      mass = rest_sum();
      if (!(mass > 0.0)) {
        tried = 0;
        mass = 1.0;
      }
    }
    if (next >= 0) {
      node = next;
      continue;
    }
    // ---- the walk ends here: draw ----
    if (greedy) {
      answer = rank == 0 ? best : -1;
      break;
    }
    double sum = 0.0;
    int positive = -1;
    for (int i = v0 + lane; i < v1; i += 32) {
      const double v = rest(i);
      sum += v;
      if (v > 0.0) positive = i;
    }
    const double mine = block_reduce(sum, add);
    if (tid == 0)
      for (uint32_t c = 0; c < C; ++c) st_dsmem_f64(map_to_rank(&s.xch[phase][rank], c), mine);
    cluster_sync();
    double before = 0.0, all = 0.0;
    for (uint32_t c = 0; c < C; ++c) {
      if (c == rank) before = all;
      all += s.xch[phase][c];
    }
    phase ^= 1;
    const double target = static_cast<double>(p.draws[r]) * all;
    // the warp that the target falls into: the last one whose tokens begin at or below it (all compute
    // the same borders, in the same order)
    for (int w = 0; w < warp; ++w) before += s.warp_sum[w];
    auto last_of = [](double a, double b) { return a > b ? a : b; };
    const bool may = s.warp_sum[warp] > 0.0 && before <= target;
    const double owner = exchange(block_reduce(may ? static_cast<double>(wi) : -1.0, last_of), last_of);
    if (owner == wi) {
      double cum = before;
      long long pick = -1;
      for (int i0 = v0; i0 < v1 && pick < 0; i0 += 32) {
        const int i = i0 + lane;
        const double v = i < v1 ? rest(i) : 0.0;
        double incl = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double y = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += y;
        }
        const unsigned b = __ballot_sync(0xffffffffu, v > 0.0 && cum + incl > target);
        if (b) pick = i0 + __ffs(b) - 1;
        cum += __shfl_sync(0xffffffffu, incl, 31);
      }
      if (pick < 0) {  // the target is past the last one: rounding, or a draw of 1
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) positive = max(positive, __shfl_xor_sync(0xffffffffu, positive, o));
        pick = positive;
      }
      if (lane == 0) p.next[r] = pick;
    }
    answer = -2;  // written by its owner
    break;
  }
  if (rank == 0 && tid == 0) {
    p.accepted[r] = min(kept, p.max_path);
    if (answer != -2) p.next[r] = answer;
  }
  if (rank == 0)
    for (int i = kept + tid; i < p.max_path; i += kVerifyThreads) p.path[static_cast<long long>(r) * p.max_path + i] = -1;
  cluster_sync();  // no CTA leaves while another may still write to it
}

}  // namespace mcb
