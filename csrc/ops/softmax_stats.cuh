// Running statistics of a softmax row in base 2, shared by the kernels that read logits and by the vocabulary GEMM.
#pragma once

#include "../common/ptx.cuh"

namespace b200 {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// 2^x is 0 in fp32 below this, so clamping the factor of p log p here keeps 0 * -inf out of the sums
constexpr float kFloor2 = -1000.f;

__device__ __forceinline__ long long load_label(const void* labels, bool labels64, long long row) {
  return labels64 ? reinterpret_cast<const long long*>(labels)[row] : reinterpret_cast<const int*>(labels)[row];
}

// Running softmax statistics relative to the largest logit m, with d = (x - m) c and c = logit_scale log2 e:
// s = sum 2^d, u = sum 2^d d. m stays a logit, unscaled: scaled, a mask of fp32's lowest value would overflow to -inf, and
// the difference of two logits loses less than the difference of their products. A row's log-sum-exp is kept as the pair
// (m, log2 s) for the same reasons.
struct Stats {
  float m, s, u;
};

__device__ __forceinline__ Stats empty_stats() { return {-INFINITY, 0.f, 0.f}; }

template <bool ENTROPY>
__device__ __forceinline__ void rescale(Stats& a, float m, float c) {
  // m >= a.m; while a is empty (a.m = -inf) s and u are 0 and stay so
  if (a.m == -INFINITY) {
    a.m = m;
    return;
  }
  const float shift = (a.m - m) * c, f = fast_exp2(shift);
  if (ENTROPY) a.u = f > 0.f ? (a.u + a.s * shift) * f : 0.f;
  a.s *= f;
  a.m = m;
}

template <bool ENTROPY>
__device__ __forceinline__ Stats merge(Stats a, Stats b, float c) {
  const float m = fmaxf(a.m, b.m);
  rescale<ENTROPY>(a, m, c);
  rescale<ENTROPY>(b, m, c);
  return {m, a.s + b.s, a.u + b.u};
}

template <bool ENTROPY, int N>
__device__ __forceinline__ void accumulate(Stats& a, const float* f, float c) {
  float top = f[0];
#pragma unroll
  for (int e = 1; e < N; ++e) top = fmaxf(top, f[e]);
  if (top > a.m) rescale<ENTROPY>(a, top, c);
  const float m = a.m == -INFINITY ? 0.f : a.m;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float d = (f[e] - m) * c, x = fast_exp2(d);
    a.s += x;
    if (ENTROPY) a.u = fmaf(x, fmaxf(d, kFloor2), a.u);
  }
}

// Log-probability in base 2 of logit x under a row's (m, log2 s).
__device__ __forceinline__ float log2_prob(float x, float2 lse, float c) { return fmaf(x - lse.x, c, -lse.y); }

// d(score) / d(z_j) times logit_scale, from the log-probability d in base 2: gs, hs = upstream gradients times logit_scale, H = entropy. The
// label's own +gs is added by the caller.
template <bool ENTROPY>
__device__ __forceinline__ float score_gradient(float d, float gs, float hs, float H) {
  const float w = ENTROPY ? fmaf(hs, fmaf(fmaxf(d, kFloor2), kLn2, H), gs) : gs;
  return -fast_exp2(d) * w;
}

}  // namespace b200
