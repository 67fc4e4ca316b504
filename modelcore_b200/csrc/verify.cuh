// Verification of drafted tokens against the target's probabilities.
//
// Request r's tokens [cu_r, cu_{r+1}) are a tree: token 0 is part of the answer already, each other one
// was drafted to follow its parent.  A walk from token 0 at token u, with p = softmax(logits_u / T),
// takes u's children c_1, c_2, ... in order, x_i the token of c_i, a_i its uniform:
//   rest_0 = p;   c_i is kept when a_i q(x_i) |rest| < rest(x_i), |rest| the sum of rest,
//   otherwise     rest <- max(rest / |rest| - q, 0)   with q = draft_probs_u, of which the x_i were drawn
//                 rest <- rest, but rest(x_i) = 0     without draft_probs: q is 1 at x_i
//   (rest = p again should nothing be left of it).
// With q >= 0 the steps' maxima can wait: a term that is below 0 once stays there, so after refusals with
// |rest| = m_0 = 1, m_1, ... the rest is max(A p - B q, 0), A = A / m_i and B = B / m_i + 1 a step.
// The walk goes on at a kept child; where none is kept the next token is the first x with
//   rest(0) + ... + rest(x) > draw |rest|.
// So the tokens are distributed as if each had been drawn from its p, whatever the draft was.  T = 0: a
// child is kept when its token is the first one of the largest logit, which is the next token otherwise.
//
// Only the rows on the walk are read: a cluster of C CTAs a request, the vocabulary divided among them,
// and every CTA takes the walk's decisions itself from the same numbers, exchanged through distributed shared
// memory.  What is decided is what 64-bit sums decide, to their rounding: a vocabulary of 10^5 has borders
// everywhere, and 32-bit sums put a draw on their wrong side now and then.
//   A token's row is first summed in 32 bits (one pass, bound by its bytes), with a bound on how far off the
//   sums can be (it grows with the tokens a lane adds up); children are kept or refused by these while the sides of the comparison are further apart than
//   that, in nearly all cases.  Where they are not, and where the walk ends and a token is drawn, the row is
//   summed again in 64 bits (bound by the 64-bit units: about 11 operations a token and pass).
// Measured: 64 requests of 16 tokens, wide 3, 131,071 logits of fp32 and draft_probs 146 to 156 us by the draws (207 MB; the slowest
// request's chain of passes, 4 CTAs: 8 us a row in 32 bits, 15 to 30 a pass in 64), 3 requests of 8 tokens and 32,768
// logits 25 us, latency; greedy 78 and 16 us, bf16 logits 141 and 25.
// 2^t in 64 bits: 32 t = n + f with |f| <= 1/2, a table of 2^(j/32) and five terms of 2^(f/32)'s series in f ln 2 / 32
// (the remainder, (ln 2 / 64)^6 / 720, is 2e-15): Tang's table-driven method, ACM TOMS 15, 1989.
#pragma once

#include <type_traits>

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
// Four values from an address that four of them divide.
__device__ __forceinline__ float4 logits4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 logits4(const uint16_t* p) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16),
                     __uint_as_float(v.y & 0xffff0000u));
}

__device__ __forceinline__ void st_dsmem_u64(uint32_t addr, unsigned long long v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}

struct VerifyShared {
  unsigned long long xch[2][8];      // what the cluster's CTAs exchange
  double table[32];                  // 2^(j / 32)
  double warp_sum[kVerifyWarps];     // this CTA's warps' 64-bit sums of the last pass
  unsigned long long warp_word[kVerifyWarps];
  double inv[kVerifyMaxTried];       // with draft: 1 / the rest's sum before each refused child, the first's 1 / all
  int gone[kVerifyMaxTried];         // without draft: the refused children's tokens
  int parent[kVerifyMaxTried], token[kVerifyMaxTried];  // the request's first tokens' (those behind are read)
  float accept[kVerifyMaxTried];
};

// A float as a double by integer operations (the conversion unit takes 16 a clock): exact for normal numbers; a 0
// becomes 2^-127, an infinity 2^128.
__device__ __forceinline__ double double_of(float x) {
  const uint32_t u = __float_as_uint(x);
  return __hiloint2double(static_cast<int>((u & 0x80000000u) | ((u & 0x7fffffffu) >> 3) + 0x38000000u),
                          static_cast<int>(u << 29));
}

// This warp's share of a row: the vocabulary in groups of four at the row's own alignment, `mis` elements
// before the row's first, shared out to the cluster's warps in order.
struct VerifySpan {
  int y0, y1, mis;
  __device__ __forceinline__ VerifySpan(const void* row, int size, int V, int wi, int nw) {
    mis = static_cast<int>(reinterpret_cast<uintptr_t>(row) / size & 3);
    const long long total = static_cast<long long>(V) + mis;
    const long long per = (total + nw * 128ll - 1) / (nw * 128ll) * 128;
    y0 = static_cast<int>(min(wi * per, total));
    y1 = static_cast<int>(min(y0 + per, total));
  }
};

template <typename T>
__device__ __forceinline__ void load4(const T* row, int v, int V, float outside, float (&x)[4]) {
  if (v >= 0 && v + 4 <= V) {
    const float4 q = logits4(row + v);
    x[0] = q.x, x[1] = q.y, x[2] = q.z, x[3] = q.w;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = v + e >= 0 && v + e < V ? logit_of(row + v + e) : outside;
  }
}

// Four of the draft's probabilities; its rows may lie otherwise than the logits'.
__device__ __forceinline__ void draft4(const float* q, bool vec, int v, int V, float (&x)[4]) {
  if (vec && v >= 0 && v + 4 <= V) {
    const float4 f = *reinterpret_cast<const float4*>(q + v);
    x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = v + e >= 0 && v + e < V ? q[v + e] : 0.f;
  }
}

// f(v, x[4], q[4]) for every group of a lane's, the loads of several on their way at once: those of whole turns
// inside the row without a branch between them (a branch each cost a trip to memory each: 20,000 cycles for
// 33,000 logits).  Without WITH_Q the q are not read.
template <bool WITH_Q, typename T, typename F>
__device__ __forceinline__ void each4(const T* row, const float* q, bool q_vec, const VerifySpan& s, int V, F f) {
  constexpr int U = WITH_Q ? 2 : 4;
  const int lane = threadIdx.x & 31;
  int b = s.y0;  // (the same in all lanes)
  auto turn = [&](auto u_const) {
    constexpr int N = decltype(u_const)::value;
    float x[N][4], d[N][4];
    const int v0 = b + lane * 4 - s.mis;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const float4 t = logits4(row + v0 + u * 128);
      x[u][0] = t.x, x[u][1] = t.y, x[u][2] = t.z, x[u][3] = t.w;
    }
    if constexpr (WITH_Q) {
      if (q_vec) {
#pragma unroll
        for (int u = 0; u < N; ++u) {
          const float4 t = *reinterpret_cast<const float4*>(q + v0 + u * 128);
          d[u][0] = t.x, d[u][1] = t.y, d[u][2] = t.z, d[u][3] = t.w;
        }
      } else {
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) d[u][e] = q[v0 + u * 128 + e];
      }
    }
#pragma unroll
    for (int u = 0; u < N; ++u) f(v0 + u * 128, x[u], d[u]);
    b += N * 128;
  };
  while (b < s.y1) {
    const int room = min(s.y1, V + s.mis) - b;
    if (b >= s.mis && room >= U * 128) {
      turn(std::integral_constant<int, U>());
    } else if (b >= s.mis && room >= 128) {
      turn(std::integral_constant<int, 1>());
    } else {  // a row's ends
      const int y = b + lane * 4;
      float x[4], d[4] = {0.f, 0.f, 0.f, 0.f};
      if (y < s.y1) {
        load4(row, y - s.mis, V, -CUDART_INF_F, x);
        if constexpr (WITH_Q) draft4(q, q_vec, y - s.mis, V, d);
        f(y - s.mis, x, d);
      }
      b += 128;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kVerifyThreads, 2) verify_kernel(const VerifyParams p) {
  __shared__ VerifyShared s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t rank, C;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(C));
  cluster_arrive_relaxed();  // started: its shared memory may be written
  if (tid < 32) s.table[tid] = exp2(tid / 32.0);
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  const int r = blockIdx.x / C;
  const int tok0 = min(max(p.cu[r], 0), p.N), count = min(max(p.cu[r + 1], tok0), p.N) - tok0;
  const int nw = C * kVerifyWarps, wi = rank * kVerifyWarps + warp;
  int phase = 0;
  // A word of every CTA, its first thread's, to all of them: lane c gets CTA c's.  (A butterfly of fused products and
  // sums leaves the lanes results that differ in their last bit; a cluster whose CTAs got a lane each would decide
  // on different sums, and meet at different barriers.)
  auto exchange = [&](unsigned long long a) {
    a = __shfl_sync(0xffffffffu, a, 0);
    if (warp == 0 && lane < C) st_dsmem_u64(map_to_rank(&s.xch[phase][rank], lane), a);
    cluster_sync();
    const unsigned long long got = s.xch[phase][lane & 7];
    phase ^= 1;  // (a slot is written again two exchanges on: every thread has read it by the one between)
    return got;
  };
  // A warp's word to all warps: lane w gets warp w's.
  auto spread = [&](unsigned long long a) {
    __syncthreads();
    if (lane == 0) s.warp_word[warp] = a;
    __syncthreads();
    return s.warp_word[lane & (kVerifyWarps - 1)];
  };
  auto sum_lanes = [&](double v, int n) {  // over lanes 0 .. n - 1, n a power of two; the same in all lanes
    for (int o = n >> 1; o >= 1; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return __shfl_sync(0xffffffffu, v, 0);
  };
  for (int i = tid; i < min(count, kVerifyMaxTried); i += kVerifyThreads) {
    s.parent[i] = p.parents[tok0 + i];
    const long long x = p.tokens[tok0 + i];
    s.token[i] = x < 0 || x >= p.V ? -1 : static_cast<int>(x);
    s.accept[i] = p.accept[tok0 + i];
  }
  __syncthreads();
  cluster_wait();  // every block has started
  const float inv_t32 = p.temperature > 0.f ? 1.f / p.temperature : 1.f;
  const double scale = (p.temperature > 0.f ? 1.0 / static_cast<double>(p.temperature) : 1.0) * 32.0 * 1.4426950408889634074;
  const float scale32 = inv_t32 * 1.4426950408889634f;
  const bool greedy = p.temperature == 0.f;
  // How far a 32-bit sum of weights may be off, relative to it, in e = 2^-24, with n groups of four a lane.  A weight
  // 2^t: 5 e |t| ln 2 for the difference, the scale and their product, 4 e for the exponential; |t| in the mean over p
  // is at most log2 V.  A lane's sum: 3 e for a group's additions, 5 e where the maximum moves, at most with every
  // group.  Lanes, warps and blocks joined: 5 e each for their maximum, 12 e of additions.  (33 + 3.5 log2 V + 8 n) e;
  // 15 e and (8 n e)^2 for the products of these factors.  A rest's sum, of a p - b q, stays within that times b (>= a).
  auto eps32 = [&] {
    const float n = static_cast<float>((p.V + nw * 128 + 2) / (nw * 128));
    return (48.f + 3.5f * (32 - __clz(p.V)) + (8.f + 0x1p-18f * n) * n) * 0x1p-24f;
  };
  int node = 0, kept = 0;
  long long answer = -1;
  while (count > 0) {
    if (rank == 0 && tid == 0) p.path[static_cast<long long>(r) * p.max_path + kept] = node;
    ++kept;
    const T* row = static_cast<const T*>(p.logits) + (tok0 + node) * p.logits_stride;
    const float* q = p.draft != nullptr && !greedy ? p.draft + (tok0 + node) * p.draft_stride : nullptr;
    const VerifySpan span(row, sizeof(T), p.V, wi, nw);
    const bool q_vec = q != nullptr && (reinterpret_cast<uintptr_t>(q) / 4 & 3) == span.mis;

    // ---- the largest logit, and the first that is; or the sum of the weights, in 32 bits ----
    float top;
    long long best = -1;
    float total32 = 0.f;
    if (greedy) {
      unsigned long long word = 0;  // order-preserving image of the logit, then of the first index
      each4<false>(row, nullptr, false, span, p.V, [&](int v, const float (&x)[4], const float (&)[4]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t u = __float_as_uint(x[e] + 0.f);  // (no -0)
          const uint32_t key = x[e] != x[e] ? 0xffffffffu : u & 0x80000000u ? ~u : u | 0x80000000u;
          const unsigned long long w = static_cast<unsigned long long>(key) << 32 | static_cast<uint32_t>(~(v + e));
          if (w > word && v + e >= 0 && v + e < p.V) word = w;
        }
      });
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, word, o);
        word = max(word, other);
      }
      auto largest = [&](unsigned long long v) {
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) {
          const unsigned long long other = __shfl_xor_sync(0xffffffffu, v, o);
          v = max(v, other);
        }
        return v;
      };
      word = largest(spread(word));
      word = exchange(word);
      word = largest(lane < C ? word : 0);
      const uint32_t key = static_cast<uint32_t>(word >> 32);
      top = key == 0xffffffffu ? CUDART_NAN_F : __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
      best = static_cast<uint32_t>(~static_cast<uint32_t>(word));
    } else {
      float m = -CUDART_INF_F, sum = 0.f;
      bool odd = false;  // NaN or +infinity
      each4<false>(row, nullptr, false, span, p.V, [&](int, const float (&x)[4], const float (&)[4]) {
        const float big = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
        odd |= !(x[0] < CUDART_INF_F) | !(x[1] < CUDART_INF_F) | !(x[2] < CUDART_INF_F) | !(x[3] < CUDART_INF_F);
        if (big > m) {
          sum *= fast_exp2((m - big) * scale32);
          m = big;
        }
        if (m > -CUDART_INF_F)
          sum += (fast_exp2((x[0] - m) * scale32) + fast_exp2((x[1] - m) * scale32)) +
                 (fast_exp2((x[2] - m) * scale32) + fast_exp2((x[3] - m) * scale32));
      });
      if (odd) m = CUDART_INF_F;
      auto join = [&](int n) {  // over groups of n lanes
        float big = m;
        for (int o = n >> 1; o >= 1; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
        if (big > -CUDART_INF_F && big < CUDART_INF_F) sum *= fast_exp2((m - big) * scale32);  // (once: each costs precision)
        m = big;
        for (int o = n >> 1; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      };
      auto word = [&] { return static_cast<unsigned long long>(__float_as_uint(m)) << 32 | __float_as_uint(sum); };
      auto unpack = [&](unsigned long long a) {
        m = __uint_as_float(static_cast<uint32_t>(a >> 32));
        sum = __uint_as_float(static_cast<uint32_t>(a));
      };
      join(32);
      unpack(spread(word()));
      join(kVerifyWarps);
      unpack(exchange(word()));
      join(static_cast<int>(C));
      m = __shfl_sync(0xffffffffu, m, 0);  // (C lanes have it)
      sum = __shfl_sync(0xffffffffu, sum, 0);
      top = m;
      total32 = sum;
    }
    if (!(top > -CUDART_INF_F && top < CUDART_INF_F)) {  // NaN, an infinity, or no token at all
      if (rank == 0 && tid == 0) record_error(kErrNoProbabilities);
      break;
    }

    // ---- the same in 64 bits ----
    const double top64 = top;
    auto weight = [&](float x) -> double {
      const double d = double_of(x) - top64;        // (first: with a small temperature's scale neither is exact)
      constexpr double magic = 6755399441055744.0;  // 1.5 * 2^52
      const double kd = fma(d, scale, magic);       // 32 t = n + f
      const int n = __double2loint(kd);
      const double f = fma(d, scale, magic - kd);
      double e = 0x1p-25 * 1.3333558146428443e-3;   // (ln 2 / 32)^k / k!, k = 5 .. 1
      e = fma(e, f, 0x1p-20 * 9.6181291076284772e-3);
      e = fma(e, f, 0x1p-15 * 5.5504108664821580e-2);
      e = fma(e, f, 0x1p-10 * 2.4022650695910071e-1);
      e = fma(e, f, 0x1p-5 * 6.9314718055994531e-1);
      const double tab = s.table[n & 31];
      const double w = fma(tab * f, e, tab);
      // times 2^(n / 32); below 2^-1000 nothing (a logit of -infinity among them)
      return kd > magic - 32000.0 ? __hiloint2double(__double2hiint(w) + ((n >> 5) << 20), __double2loint(w)) : 0.0;
    };
    int tried = 0;                  // without draft: refused so far, of those that the rest is without
    bool exact = false;             // mass and the factors come of 64-bit sums
    double mass = 1.0;              // of the rest
    // the rest is max(of_p w - of_q q, 0), w the weight before its division by all.  The two products grow with every
    // division by a small sum, and cancel; past 2^16 (2^-36 of a rest) it is taken step by step, each rest
    // divided by its own sum
    double of_p = 1.0 / static_cast<double>(total32), of_q = 0.0;
    int refused = 0;
    auto rest_of = [&](double w, float qx, int x) {  // of token x
      if (q != nullptr) {
        double v = w;
        if (exact && of_q > 65536.0)
          for (int k = 0; k < refused; ++k) v = fma(v, s.inv[k], -static_cast<double>(qx));
        else v = fma(w, of_p, -(static_cast<double>(qx) * of_q));
        return v > 0.0 ? v : 0.0;
      }
      double v = w * of_p;
      for (int k = 0; k < tried; ++k)
        if (s.gone[k] == x) v = 0.0;
      return v;
    };
    auto refuse = [&] {  // a draft's child, the rest's sum being mass
      if (exact) {
        __syncthreads();
        if (tid == 0) s.inv[refused] = refused == 0 ? of_p : 1.0 / mass;
        __syncthreads();
      }
      of_p /= mass;
      of_q = of_q / mass + 1.0;
      ++refused;
    };
    auto restart = [&](double all) {
      of_p = 1.0 / all;
      of_q = 0.0;
      mass = 1.0;
      refused = tried = 0;
    };
    // The rest's sum over the vocabulary, in 64 bits: warp_sum and the last exchange's slots keep its parts.
    int positive = -1;              // this lane's last token with any
    auto sum64 = [&](bool raw) {    // raw: of the weights themselves
      double sum = 0.0;
      positive = -1;
      auto add = [&](double y, int v) {
        sum += y;
        if (y > 0.0) positive = v;
      };
      if (raw || (q != nullptr && refused == 0) || (q == nullptr && tried == 0)) {
        const double unit = raw ? 1.0 : of_p;
        each4<false>(row, nullptr, false, span, p.V, [&](int v, const float (&x)[4], const float (&)[4]) {
#pragma unroll
          for (int e = 0; e < 4; ++e) add(weight(x[e]) * unit, v + e);
        });
      } else if (q != nullptr && of_q > 65536.0) {  // (rare: a token at a time)
        for (int y = span.y0 + lane; y < span.y1; y += 32) {
          const int v = y - span.mis;
          if (v >= 0 && v < p.V) add(rest_of(weight(logit_of(row + v)), q[v], v), v);
        }
      } else if (q != nullptr) {
        const double a = of_p, b = -of_q;
        each4<true>(row, q, q_vec, span, p.V, [&](int v, const float (&x)[4], const float (&d)[4]) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const double y = fma(weight(x[e]), a, double_of(d[e]) * b);
            if (y > 0.0) add(y, v + e);
          }
        });
      } else {
        each4<false>(row, nullptr, false, span, p.V, [&](int v, const float (&x)[4], const float (&)[4]) {
#pragma unroll
          for (int e = 0; e < 4; ++e) add(rest_of(weight(x[e]), 0.f, v + e), v + e);
        });
      }
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      __syncthreads();
      if (lane == 0) s.warp_sum[warp] = sum;
      __syncthreads();
      const double mine = sum_lanes(s.warp_sum[lane & (kVerifyWarps - 1)], kVerifyWarps);
      return sum_lanes(__longlong_as_double(exchange(__double_as_longlong(mine))), static_cast<int>(C));
    };
    // Everything so far at this token again in 64 bits.
    auto make_exact = [&] {
      const int n = refused, gone = tried;
      restart(sum64(true));
      exact = true;
      if (q == nullptr) {
        tried = gone;
        if (tried > 0) mass = sum64(false);
        return;
      }
      while (refused < n) {
        refuse();
        mass = sum64(false);
        if (!(mass > 0.0)) {  // (only where 32 bits saw something left that is not)
          restart(sum64(true));
          break;
        }
      }
    };

    // ---- its children in turn ----
    // how far the 32-bit sums of p, or of the rest, may be off, and any of their terms; and at most how far, relative to
    // themselves, of_p and of_q, the factors of a child's 64-bit weight and q
    double off = eps32();
    int next = -1, last = node;
    for (int tries = 0; kept < p.max_path && tries < kVerifyMaxTried; ++tries) {
      // the next child (every warp looks for itself)
      int c = -1;
      for (int j0 = last + 1; j0 < count && c < 0; j0 += 32) {
        const int j = j0 + lane;
        int parent = -1;
        if (j < count) parent = j < kVerifyMaxTried ? s.parent[j] : p.parents[tok0 + j];
        const unsigned b = __ballot_sync(0xffffffffu, parent == node);
        if (b) c = j0 + __ffs(b) - 1;
      }
      if (c < 0) break;
      last = c;
      long long x = c < kVerifyMaxTried ? s.token[c] : p.tokens[tok0 + c];
      if (x < 0 || x >= p.V) {
        if (rank == 0 && tid == 0) record_error(kErrTokenOutOfRange);
        continue;
      }
      if (greedy) {
        if (x == best) {
          next = c;
          break;
        }
        continue;
      }
      const float u = c < kVerifyMaxTried ? s.accept[c] : p.accept[tok0 + c];
      if (!(u >= 0.f)) {
        if (rank == 0 && tid == 0) record_error(kErrUniformOutOfRange);
        continue;
      }
      const float qx = q != nullptr ? q[x] : 1.f;
      const double w = weight(logit_of(row + x)), bar = static_cast<double>(u) * qx;
      double have = rest_of(w, qx, static_cast<int>(x));
      if (!exact && !(fabs(bar * mass - have) > 2.0 * off * fmin(bar + w * of_p + qx * of_q, 1.0))) {  // too close (or a NaN)
        make_exact();
        have = rest_of(w, qx, static_cast<int>(x));
      }
      if (bar * mass < have) {
        next = c;
        break;
      }
      // refused: the rest is without it
      if (q == nullptr) {
        __syncthreads();
        if (tid == 0) s.gone[tried] = static_cast<int>(x);
        __syncthreads();
        mass -= have;
        ++tried;
        // a difference says little of a small rest, and nothing of an empty one
        if (mass < 1e-3) {
          make_exact();
          if (!(mass > 0.0)) {
            tried = 0;
            mass = 1.0;
          }
        }
        continue;
      }
      const double before = mass;
      refuse();
      if (!exact) {
        const float a = static_cast<float>(of_p), b = -static_cast<float>(of_q);
        float sum = 0.f;
        each4<true>(row, q, q_vec, span, p.V, [&](int, const float (&x)[4], const float (&d)[4]) {
          float y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = fmaxf(fmaf(fast_exp2((x[e] - top) * scale32), a, d[e] * b), 0.f);
          sum += (y[0] + y[1]) + (y[2] + y[3]);
        });
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const double mine = sum_lanes(__longlong_as_double(spread(__double_as_longlong(static_cast<double>(sum)))), kVerifyWarps);
        mass = sum_lanes(__longlong_as_double(exchange(__double_as_longlong(mine))), static_cast<int>(C));
        off = 2.0 * off / before + eps32() * of_q;
        if (!(mass > 4.0 * off)) make_exact();  // nothing left, as far as 32 bits can tell
      } else {
        mass = sum64(false);
        if (!(mass > 0.0)) restart(sum64(true));
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
    if (!(p.draws[r] >= 0.f)) {  // (no token's share begins below it)
      if (rank == 0 && tid == 0) record_error(kErrUniformOutOfRange);
      break;
    }
    // The rest's parts in 64 bits, in any unit; without draft_probs, or with no child refused, from the weights alone.
    if (q != nullptr && refused > 0 && !exact) {
      make_exact();  // (ends with the rest's sum, or the weights')
      if (refused == 0) of_p = 1.0;
    } else {
      if (q == nullptr || refused == 0) of_p = 1.0;
      mass = sum64(false);
      if (!(mass > 0.0)) {
        restart(1.0);
        mass = sum64(true);
      }
    }
    double before = 0.0, all = 0.0;
    for (uint32_t c = 0; c < C; ++c) {
      if (c == rank) before = all;
      all += __longlong_as_double(s.xch[phase ^ 1][c]);
    }
    const double target = static_cast<double>(p.draws[r]) * all;
    // the warp that the target falls into: the last one whose tokens begin at or below it (all compute
    // the same borders, in the same order)
    for (int w = 0; w < warp; ++w) before += s.warp_sum[w];
    const bool may = s.warp_sum[warp] > 0.0 && before <= target;
    auto largest = [&](unsigned long long v) {
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, v, o);
        v = max(v, other);
      }
      return v;
    };
    unsigned long long owner = largest(spread(may ? wi + 1 : 0));
    owner = exchange(owner);
    owner = largest(lane < C ? owner : 0);
    if (owner == static_cast<unsigned long long>(wi) + 1) {
      // within it: the lanes' 32 spans first, then the one's tokens
      auto rest_at = [&](int v) {
        if (v < 0 || v >= p.V) return 0.0;
        return rest_of(weight(logit_of(row + v)), q != nullptr ? q[v] : 0.f, v);
      };
      auto scan = [&](double v) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double y = __shfl_up_sync(0xffffffffu, v, o);
          if (lane >= o) v += y;
        }
        return v;
      };
      const int per = (span.y1 - span.y0 + 31) / 32, a = span.y0 + lane * per - span.mis;
      const int end = span.y1 - span.mis;
      double sum = 0.0;
      for (int i = 0; i < per; ++i) sum += a + i < end ? rest_at(a + i) : 0.0;
      double incl = scan(sum);
      unsigned b = __ballot_sync(0xffffffffu, sum > 0.0 && before + incl > target);
      long long pick = -1;
      if (b) {
        const int l = __ffs(b) - 1;
        double cum = before + __shfl_sync(0xffffffffu, incl - sum, l);
        const int from = __shfl_sync(0xffffffffu, a, l), to = min(from + per, end);
        int some = -1;
        for (int i0 = from; i0 < to && pick < 0; i0 += 32) {
          const double v = i0 + lane < to ? rest_at(i0 + lane) : 0.0;
          incl = scan(v);
          const unsigned has = __ballot_sync(0xffffffffu, v > 0.0);
          b = __ballot_sync(0xffffffffu, v > 0.0 && cum + incl > target);
          if (b) pick = i0 + __ffs(b) - 1;
          if (has) some = i0 + 31 - __clz(has);
          cum += __shfl_sync(0xffffffffu, incl, 31);
        }
        if (pick < 0) pick = some;  // (the span's last: its sum in another order went past the target)
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
    p.accepted[r] = kept;
    if (answer != -2) p.next[r] = answer;
  }
  if (rank == 0)
    for (int i = kept + tid; i < p.max_path; i += kVerifyThreads) p.path[static_cast<long long>(r) * p.max_path + i] = -1;
  cluster_sync();  // no CTA leaves while another may still write to it
}

}  // namespace mcb
