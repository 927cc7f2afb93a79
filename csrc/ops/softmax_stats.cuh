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

// Two fp32 values in one register pair: one instruction for two FMAs, adds or products.
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 pack2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack2(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

// N logits (an even number, in pairs) whose maximum is `top` enter the statistics. The difference x - m is formed before it is scaled:
// d = x c - m c in one FMA would carry the rounding of m c into the sums, which grows with the row's distance from zero (5e-3 in a
// log-probability at logits around 1e5) and differs between the parts of a row, whose maxima differ, so that nothing takes it back.
template <bool ENTROPY, int N>
__device__ __forceinline__ void accumulate(Stats& a, const F2 (&f)[N / 2], float top, float c) {
  if (top > a.m) rescale<ENTROPY>(a, top, c);
  const float m = a.m == -INFINITY ? 0.f : a.m;
  F2 s0 = pack2(0.f, 0.f), s1 = s0, u0 = s0, u1 = s0;
  const F2 c2 = pack2(c, c);
  auto add = [&](F2 d2, int i) {
    const float2 d = unpack2(d2);
    const F2 x = pack2(fast_exp2(d.x), fast_exp2(d.y));
    if (i & 1) s1 = add2(s1, x);
    else s0 = add2(s0, x);
    if (ENTROPY) {
      const F2 e = pack2(fmaxf(d.x, kFloor2), fmaxf(d.y, kFloor2));
      if (i & 1) u1 = fma2(x, e, u1);
      else u0 = fma2(x, e, u0);
    }
  };
  const F2 off = pack2(-m, -m);
#pragma unroll
  for (int i = 0; i < N / 2; ++i) add(mul2(add2(f[i], off), c2), i);
  const float2 s = unpack2(add2(s0, s1));
  a.s += s.x + s.y;
  if (ENTROPY) {
    const float2 u = unpack2(add2(u0, u1));
    a.u += u.x + u.y;
  }
}

// Log-probability (natural) of logit x under a row's (m, log2 s). Not formed in base 2: next to a mask of the type's lowest value the factor
// log2 e would overflow before ln 2 takes it back.
__device__ __forceinline__ float log_prob(float x, float2 lse, float logit_scale) { return fmaf(x - lse.x, logit_scale, -lse.y * kLn2); }

// The same in base 2, as the exponent of a probability (where -inf is as good as any number below -150).
__device__ __forceinline__ float log2_prob(float x, float2 lse, float c) { return fmaf(x - lse.x, c, -lse.y); }

// d(score) / d(z_j) times logit_scale, from the log-probability d in base 2: gs, hs = upstream gradients times logit_scale, H = entropy. The
// label's own +gs is added by the caller.
template <bool ENTROPY>
__device__ __forceinline__ float score_gradient(float d, float gs, float hs, float H) {
  const float w = ENTROPY ? fmaf(hs, fmaf(fmaxf(d, kFloor2), kLn2, H), gs) : gs;
  return -fast_exp2(d) * w;
}

}  // namespace b200
