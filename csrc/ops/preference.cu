// Losses over per-token log-probabilities of packed answers, reduced per sequence.
//
// Preference loss: with d_t = lp_t - ref_t, s_i = sum (or mean) of d_t over sequence i and D = s_chosen - s_rejected,
//   sigmoid: (1 - e) softplus(-b D) + e softplus(b D)      dD: -b ((1 - e) sigmoid(-b D) - e sigmoid(b D))
//   hinge:   max(0, 1 - b D)                               dD: -b where b D < 1
//   ipo:     (D - 1 / (2 b))^2                             dD: 2 (D - 1 / (2 b))
// Policy loss: with r = exp(lp - old), k = ref - lp,
//   l = max(-A r, -A clip(r, lo, hi)) + c (expm1(k) - k)    dlp: -A r where the clip does not bind, - c expm1(k)
// optionally with a bound -dual A for A < 0 (no gradient where it binds).
//
// Both read 8 to 20 bytes a token once. The unit of work is a warp with a chunk of 64 or 256 consecutive tokens, whose loads are
// issued before the sequences that overlap it are looked up; its partial sums of sequence i go to slot (chunk + i), which no
// other (chunk, sequence) pair shares, so that nothing is added atomically and results do not depend on the order in which
// blocks run. A second phase adds a sequence's slots, one warp per sequence, in 64 bits. Up to kOneLaunch tokens both phases run in
// one launch of a cluster of eight blocks (one launch latency, the phases separated by the cluster's barrier) and chunks are
// short, since a chunk's chain of loads and functions is all the time there is; above it the first phase takes a grid of its own.
#include <cmath>

#include "../common/cta_pair.cuh"
#include "../common/launch.h"
#include "../common/ptx.cuh"
#include "vocabulary.h"

namespace b200 {

namespace {

constexpr int WIDE = 8, NARROW = 2;       // tokens of a lane; a chunk is 32 times as many
constexpr int CLUSTER = 8;
constexpr int CLUSTER_THREADS = 512;
constexpr int WARPS_A = 8;                // warps per block of the wide first phase
constexpr int WORDS = 4;                  // fp32 words per slot
constexpr long long kOneLaunch = 65536;

struct Span {
  long long begin, end;
};

__device__ __forceinline__ Span sequence_span(const PackedTokens& p, int i) {
  if (p.cu == nullptr) return {min(p.T, i * p.length), min(p.T, (i + 1) * p.length)};
  const long long b = max(0LL, min(p.T, (long long)p.cu[i])), e = max(b, min(p.T, (long long)p.cu[i + 1]));
  return {b, e};
}

// First sequence that ends behind token t (all lanes call it with the same t).
__device__ __forceinline__ int first_sequence(const PackedTokens& p, long long t) {
  if (p.cu == nullptr) return p.length > 0 ? (int)min((long long)p.sequences, t / p.length) : p.sequences;
  int lo = 0, hi = p.sequences;  // answer in [lo, hi]
  while (lo < hi) {
    // 32 probes at a time
    const int span = hi - lo;
    const int probe = lo + (int)(((long long)span * (threadIdx.x & 31)) >> 5);
    const bool ends_before = (long long)p.cu[probe + 1] <= t;
    const unsigned votes = __ballot_sync(0xffffffffu, ends_before);
    const int n = __popc(votes);  // ends are ordered: the first n probes lie before the answer
    if (n == 0) {
      hi = lo;
    } else {
      const int last = lo + (int)(((long long)span * (n - 1)) >> 5);
      const int next = n < 32 ? lo + (int)(((long long)span * n) >> 5) : hi;
      lo = last + 1;
      hi = max(lo, next);
    }
  }
  return lo;
}

// Value of `local` (a shared-memory word) in block `rank` of this cluster.
__device__ __forceinline__ double cluster_read(const double* local, unsigned rank) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(map_to_cta(smem_u32(local), rank)) : "memory");
  return v;
}

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sums of N values over all threads of the cluster, in a fixed order, valid in thread 0 of block 0.
template <int N>
struct SumSpace {
  double warp[CLUSTER_THREADS / 32][N];
  double block[N];
};
template <int N>
__device__ __forceinline__ void cluster_sums(double (&v)[N], SumSpace<N>& space) {
#pragma unroll
  for (int n = 0; n < N; ++n) v[n] = warp_sum_f64(v[n]);
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int n = 0; n < N; ++n) space.warp[threadIdx.x >> 5][n] = v[n];
  }
  __syncthreads();
  if (threadIdx.x < N) {
    double s = 0;
    for (int w = 0; w < CLUSTER_THREADS / 32; ++w) s += space.warp[w][threadIdx.x];
    space.block[threadIdx.x] = s;
  }
  cluster_sync_all();
  if (cluster_ctarank() == 0 && threadIdx.x == 0) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      v[n] = 0;
      for (int b = 0; b < CLUSTER; ++b) v[n] += cluster_read(&space.block[n], b);
    }
  }
  cluster_sync_all();  // nobody leaves while block 0 reads
}

// The tokens of a warp's chunk, K per lane: token base + lane + 32 k.
template <int K>
struct Chunk {
  long long base;
  int count;  // tokens below T

  __device__ __forceinline__ Chunk(const PackedTokens& p, long long chunk)
      : base(chunk * (32 * K)), count((int)min((long long)(32 * K), p.T - base)) {}
  __device__ __forceinline__ int at(int k) const { return (threadIdx.x & 31) + 32 * k; }
  template <typename V>
  __device__ __forceinline__ void load(const V* p, V (&v)[K]) const {
    if (count == 32 * K) {  // no condition between the loads: all are in flight together
#pragma unroll
      for (int k = 0; k < K; ++k) v[k] = p[base + at(k)];
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k) v[k] = at(k) < count ? p[base + at(k)] : V(0);
    }
  }
  // seq[k]: the token's sequence, -1 where it has none (or lies behind T) or is masked. Returns the first sequence that ends behind base;
  // `last` is the last one that overlaps the chunk (first - 1 if none does).
  __device__ __forceinline__ int sequences(const PackedTokens& p, const unsigned char (&mask)[K], int (&seq)[K], int& last) const {
#pragma unroll
    for (int k = 0; k < K; ++k) seq[k] = -1;
    const int first = first_sequence(p, base);
    last = first - 1;
    for (int i = first; i < p.sequences; ++i) {
      const Span s = sequence_span(p, i);
      if (s.begin >= base + count) break;
      last = i;
      const int b = (int)max(s.begin - base, 0LL), e = (int)min(s.end - base, (long long)count);
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (at(k) >= b && at(k) < e) seq[k] = mask[k] != 0 ? i : -1;
      if (s.end >= base + count) break;
    }
    return first;
  }
  // The same where only membership counts: seq[k] = 0 for tokens of any sequence.
  __device__ __forceinline__ void members(const PackedTokens& p, const unsigned char (&mask)[K], int (&seq)[K]) const {
    long long lo = 0, hi = p.length * p.sequences;
    if (p.cu != nullptr) {
      lo = p.cu[0];
      hi = p.cu[p.sequences];
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const long long t = base + at(k);
      seq[k] = at(k) < count && t >= lo && t < hi && mask[k] != 0 ? 0 : -1;
    }
  }
  __device__ __forceinline__ void load_mask(const PackedTokens& p, unsigned char (&mask)[K]) const {
    if (p.mask != nullptr) {
      load(p.mask, mask);
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k) mask[k] = 1;
    }
  }
  __device__ __forceinline__ void store(float* p, const float (&v)[K]) const {
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (at(k) < count) p[base + at(k)] = v[k];
  }
};

template <int K>
__device__ __forceinline__ long long chunk_count(const PackedTokens& p) {
  return (p.T + 32 * K - 1) / (32 * K);
}

// ------------------------------------------------------------------------- preference
struct PreferenceIn {
  const float* log_probs;
  const float* reference;
};

// Partial (sum of lp - ref, number of tokens) of the sequences that overlap the warp's chunk.
template <int K>
__device__ __forceinline__ void preference_chunk(const PreferenceIn& in, const PackedTokens& p, long long chunk, float* partials) {
  const Chunk<K> c(p, chunk);
  float lp[K], ref[K];
  unsigned char mask[K];
  int seq[K], last;
  c.load(in.log_probs, lp);
  if (in.reference != nullptr) c.load(in.reference, ref);
  c.load_mask(p, mask);
  const int first = c.sequences(p, mask, seq, last);
  for (int i = first; i <= last; ++i) {
    double sum = 0;  // differences of nearly equal numbers of both signs: kept exact, summed in 64 bits
    int count = 0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (seq[k] == i) {
        sum += (double)lp[k] - (in.reference != nullptr ? (double)ref[k] : 0.0);
        ++count;
      }
    }
    sum = warp_sum_f64(sum);
    count = __reduce_add_sync(0xffffffffu, count);
    if ((threadIdx.x & 31) == 0) *reinterpret_cast<double2*>(partials + (chunk + i) * WORDS) = make_double2(sum, (double)count);
  }
}

// A sequence's log-ratio and token count from its slots (whole warp).
template <int K>
__device__ __forceinline__ double2 preference_sequence(const PackedTokens& p, int i, const float* partials) {
  const Span s = sequence_span(p, i);
  double sum = 0, count = 0;
  if (s.end > s.begin) {
    const long long first = s.begin / (32 * K), last = (s.end - 1) / (32 * K);
    for (long long c = first + (threadIdx.x & 31); c <= last; c += 32) {
      const double2 v = __ldcg(reinterpret_cast<const double2*>(partials + (c + i) * WORDS));
      sum += v.x;
      count += v.y;
    }
  }
  return make_double2(warp_sum_f64(sum), warp_sum_f64(count));
}

__device__ __forceinline__ double softplus(double x) { return fmax(x, 0.0) + log1p(exp(-fabs(x))); }
__device__ __forceinline__ double sigmoid(double x) {
  const double e = exp(-fabs(x));
  return x >= 0 ? 1 / (1 + e) : e / (1 + e);
}

// Second phase: a warp of the cluster takes a pair at a time.
template <int K>
__device__ __forceinline__ void preference_pairs(const PackedTokens& p, const PreferenceArgs& a, const float* partials, float* loss,
                                                 float* chosen, float* rejected, float* slope, SumSpace<1>& space) {
  const int pairs = p.sequences / 2, lane = threadIdx.x & 31;
  const double beta = a.beta, eps = a.label_smoothing;
  const double scale = a.reduction == 2 ? 1.0 / pairs : 1.0;
  double total[1] = {0};
  for (int i = cluster_ctarank() * (CLUSTER_THREADS / 32) + (threadIdx.x >> 5); i < pairs; i += CLUSTER * (CLUSTER_THREADS / 32)) {
    const double2 w = preference_sequence<K>(p, i, partials), l = preference_sequence<K>(p, pairs + i, partials);
    const double inv_w = a.average ? 1 / fmax(w.y, 1.0) : 1.0, inv_l = a.average ? 1 / fmax(l.y, 1.0) : 1.0;
    if (lane == 0) {
      const double sw = w.x * inv_w, sl = l.x * inv_l, diff = sw - sl, margin = beta * diff;
      double value, d;
      if (a.kind == PreferenceKind::kSigmoid) {
        value = (1 - eps) * softplus(-margin);
        if (eps != 0) value += eps * softplus(margin);
        d = -beta * ((1 - eps) * sigmoid(-margin) - eps * sigmoid(margin));
      } else if (a.kind == PreferenceKind::kHinge) {
        value = margin != margin ? margin : fmax(0.0, 1 - margin);
        d = margin < 1 ? -beta : margin != margin ? margin : 0.0;
      } else {
        const double off = diff - 0.5 / beta;
        value = off * off;
        d = 2 * off;
      }
      chosen[i] = (float)(beta * sw);
      rejected[i] = (float)(beta * sl);
      slope[i] = (float)(d * scale * inv_w);
      slope[pairs + i] = (float)(-d * scale * inv_l);
      if (a.reduction == 0) loss[i] = (float)value;
      total[0] += value;
    }
  }
  if (a.reduction == 0) return;
  cluster_sums(total, space);
  if (cluster_ctarank() == 0 && threadIdx.x == 0) loss[0] = (float)(total[0] * scale);
}

template <int K, bool ONE_LAUNCH>
__global__ void __launch_bounds__(CLUSTER_THREADS)
    preference_cluster_kernel(PreferenceIn in, PackedTokens p, PreferenceArgs args, float* partials, float* loss, float* chosen,
        float* rejected, float* slope) {
  __shared__ SumSpace<1> space;
  if (ONE_LAUNCH) {
    for (long long c = cluster_ctarank() * (CLUSTER_THREADS / 32) + (threadIdx.x >> 5); c < chunk_count<K>(p); c += CLUSTER * (CLUSTER_THREADS / 32))
      preference_chunk<K>(in, p, c, partials);
    __threadfence();
    cluster_sync_all();
  }
  preference_pairs<K>(p, args, partials, loss, chosen, rejected, slope, space);
}

template <int K>
__global__ void __launch_bounds__(WARPS_A * 32) preference_chunks_kernel(PreferenceIn in, PackedTokens p, float* partials) {
  const long long c = (long long)blockIdx.x * WARPS_A + (threadIdx.x >> 5);
  if (c < chunk_count<K>(p)) preference_chunk<K>(in, p, c, partials);
}

template <int K>
__global__ void __launch_bounds__(WARPS_A * 32)
    preference_bwd_kernel(const float* __restrict__ slope, const float* __restrict__ d_loss, long long d_loss_stride, PackedTokens p,
        float* __restrict__ grad) {
  const long long chunk = (long long)blockIdx.x * WARPS_A + (threadIdx.x >> 5);
  if (chunk >= chunk_count<K>(p)) return;
  const Chunk<K> c(p, chunk);
  const int pairs = p.sequences / 2;
  unsigned char mask[K];
  int seq[K], last;
  float g[K];
  c.load_mask(p, mask);
  c.sequences(p, mask, seq, last);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    g[k] = 0.f;
    if (seq[k] >= 0) g[k] = slope[seq[k]] * d_loss[(seq[k] < pairs ? seq[k] : seq[k] - pairs) * d_loss_stride];
  }
  c.store(grad, g);
}

// ------------------------------------------------------------------------- policy
struct PolicyIn {
  const float* log_probs;
  const float* old_log_probs;
  const float* reference;
  const float* advantages;
};

// expm1(k) - k for |k| <= 1/4 without the cancellation of its first terms: the series k^2 (1/2 + k/6 + k^2/24 + ...), whose first term
// left out is below 2^-28 of the sum. (Beyond 1/4 the difference loses at most three bits.)
__device__ __forceinline__ float expm1_minus_small(float k) {
  float q = 1.f / 362880.f;
  q = fmaf(q, k, 1.f / 40320.f);
  q = fmaf(q, k, 1.f / 5040.f);
  q = fmaf(q, k, 1.f / 720.f);
  q = fmaf(q, k, 1.f / 120.f);
  q = fmaf(q, k, 1.f / 24.f);
  q = fmaf(q, k, 1.f / 6.f);
  q = fmaf(q, k, 0.5f);
  return q * k * k;
}

struct TokenLoss {
  float value, slope, kl;
  int clipped;
};

__device__ __forceinline__ TokenLoss policy_token(float lp, float old, float ref, bool has_ref, float adv, const PolicyArgs& a) {
  // the difference decides by which side of a border the token's gradient vanishes: formed and compared in 64 bits, where it
  // is exact up to the borders' own rounding
  const double delta = (double)lp - (double)old;
  const float d_hi = (float)delta;
  const float ratio = expf(d_hi);
  TokenLoss out;
  out.clipped = (adv > 0.f && delta > a.log_high) || (adv < 0.f && delta < a.log_low);
  if (out.clipped) {
    out.value = -adv * (adv > 0.f ? a.ratio_high : a.ratio_low);
    out.slope = 0.f;
  } else {
    out.value = adv == 0.f ? 0.f : -adv * ratio;  // an infinite ratio of a token without advantage counts nothing
    out.slope = out.value;
  }
  if (a.dual_clip != 0.f && adv < 0.f && out.value > -a.dual_clip * adv) {
    out.value = -a.dual_clip * adv;
    out.slope = 0.f;
    out.clipped = 1;
  }
  out.kl = 0.f;
  if (has_ref) {
    const float k = ref - lp, e = expm1f(k);
    out.kl = fabsf(k) > 0.25f ? e - k : expm1_minus_small(k);
    if (a.kl_coef == 0.f) return out;  // reported only; an infinite estimate must not reach the loss as 0 * inf
    out.value = fmaf(a.kl_coef, out.kl, out.value);
    out.slope = fmaf(-a.kl_coef, e, out.slope);
  }
  return out;
}

// Partial (loss, kl, clipped, tokens) of the warp's chunk: per sequence into slot (chunk + sequence) for the mean over
// sequences, else all together into slot `chunk`. Writes the tokens' slopes.
template <int K>
__device__ __forceinline__ void policy_chunk(const PolicyIn& in, const PackedTokens& p, const PolicyArgs& a, long long chunk,
    float* partials, float* slope) {
  const Chunk<K> c(p, chunk);
  const int lane = threadIdx.x & 31;
  float lp[K], old[K], ref[K], adv[K];
  unsigned char mask[K];
  int seq[K], first = 0, last = 0;
  c.load(in.log_probs, lp);
  c.load(in.old_log_probs, old);
  if (in.reference != nullptr) c.load(in.reference, ref);
  if (a.per_token_advantage) c.load(in.advantages, adv);
  c.load_mask(p, mask);
  if (a.per_token_advantage && a.reduction != 2) c.members(p, mask, seq);
  else first = c.sequences(p, mask, seq, last);
  TokenLoss v[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    v[k] = {0.f, 0.f, 0.f, 0};
    if (seq[k] < 0) continue;
    v[k] = policy_token(lp[k], old[k], in.reference != nullptr ? ref[k] : 0.f, in.reference != nullptr,
        a.per_token_advantage ? adv[k] : in.advantages[seq[k]], a);
  }
  if (slope != nullptr) {
    float s[K];
#pragma unroll
    for (int k = 0; k < K; ++k) s[k] = v[k].slope;
    c.store(slope, s);
  }
  const bool by_sequence = a.reduction == 2;
  for (int i = first; i <= (by_sequence ? last : first); ++i) {
    float loss = 0.f, kl = 0.f;
    int clipped = 0, count = 0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (by_sequence ? seq[k] == i : seq[k] >= 0) {
        loss += v[k].value;
        kl += v[k].kl;
        clipped += v[k].clipped;
        ++count;
      }
    }
    loss = warp_sum(loss);
    kl = warp_sum(kl);
    clipped = __reduce_add_sync(0xffffffffu, clipped);
    count = __reduce_add_sync(0xffffffffu, count);
    if (lane == 0)
      *reinterpret_cast<float4*>(partials + (chunk + (by_sequence ? i : 0)) * WORDS) =
          make_float4(loss, kl, (float)clipped, (float)count);
  }
}

template <int K>
__device__ __forceinline__ void policy_totals(const PackedTokens& p, const PolicyArgs& a, const float* partials, const PolicyOut& out,
    float* weight, SumSpace<5>& space) {
  const int lane = threadIdx.x & 31;
  const int warp = cluster_ctarank() * (CLUSTER_THREADS / 32) + (threadIdx.x >> 5);
  constexpr int kWarps = CLUSTER * (CLUSTER_THREADS / 32);
  double loss = 0, kl = 0, clipped = 0, count = 0, used = 0;
  if (a.reduction == 2) {
    for (int i = warp; i < p.sequences; i += kWarps) {
      const Span s = sequence_span(p, i);
      double l = 0, n = 0;
      if (s.end > s.begin) {
        const long long first = s.begin / (32 * K), last = (s.end - 1) / (32 * K);
        for (long long c = first + lane; c <= last; c += 32) {
          const float4 v = __ldcg(reinterpret_cast<const float4*>(partials + (c + i) * WORDS));
          l += v.x;
          kl += v.y;
          clipped += v.z;
          n += v.w;
        }
      }
      l = warp_sum_f64(l);
      n = warp_sum_f64(n);
      if (lane == 0) {
        if (n > 0) {
          loss += l / n;
          count += n;
          used += 1;
        }
        weight[i] = (float)(1.0 / fmax(n, 1.0));
      }
    }
  } else {
    for (long long c = warp * 32 + lane; c < chunk_count<K>(p); c += kWarps * 32) {
      const float4 v = __ldcg(reinterpret_cast<const float4*>(partials + c * WORDS));
      loss += v.x;
      kl += v.y;
      clipped += v.z;
      count += v.w;
    }
  }
  double sums[5] = {loss, kl, clipped, count, used};
  cluster_sums(sums, space);
  if (cluster_ctarank() == 0 && threadIdx.x == 0) {
    const double tokens = fmax(sums[3], 1.0);
    const double divisor = a.reduction == 0 ? 1.0 : a.reduction == 1 ? tokens : fmax(sums[4], 1.0);
    *out.loss = (float)(sums[0] / divisor);
    *out.kl = (float)(sums[1] / tokens);
    *out.clipped = (float)(sums[2] / tokens);
    *out.factor = (float)(1.0 / divisor);
  }
}

template <int K, bool ONE_LAUNCH>
__global__ void __launch_bounds__(CLUSTER_THREADS)
    policy_cluster_kernel(PolicyIn in, PackedTokens p, PolicyArgs args, float* partials, PolicyOut out, float* slope, float* weight) {
  __shared__ SumSpace<5> space;
  if (ONE_LAUNCH) {
    for (long long c = cluster_ctarank() * (CLUSTER_THREADS / 32) + (threadIdx.x >> 5); c < chunk_count<K>(p); c += CLUSTER * (CLUSTER_THREADS / 32))
      policy_chunk<K>(in, p, args, c, partials, slope);
    __threadfence();
    cluster_sync_all();
  }
  policy_totals<K>(p, args, partials, out, weight, space);
}

template <int K>
__global__ void __launch_bounds__(WARPS_A * 32) policy_chunks_kernel(PolicyIn in, PackedTokens p, PolicyArgs args, float* partials,
    float* slope) {
  const long long c = (long long)blockIdx.x * WARPS_A + (threadIdx.x >> 5);
  if (c < chunk_count<K>(p)) policy_chunk<K>(in, p, args, c, partials, slope);
}

template <int K>
__global__ void __launch_bounds__(WARPS_A * 32)
    policy_bwd_kernel(const float* __restrict__ slope, const float* __restrict__ factor, const float* __restrict__ weight,
        const float* __restrict__ d_loss, PackedTokens p, int reduction, float* __restrict__ grad) {
  const long long chunk = (long long)blockIdx.x * WARPS_A + (threadIdx.x >> 5);
  if (chunk >= chunk_count<K>(p)) return;
  const Chunk<K> c(p, chunk);
  unsigned char mask[K];
  int seq[K], last;
  float g[K];
  c.load(slope, g);
  c.load_mask(p, mask);
  const float w = factor[0] * d_loss[0];
  if (reduction == 2) c.sequences(p, mask, seq, last);
  else c.members(p, mask, seq);
#pragma unroll
  for (int k = 0; k < K; ++k) g[k] = seq[k] < 0 ? 0.f : g[k] * (reduction == 2 ? w * weight[seq[k]] : w);
  c.store(grad, g);
}

template <int K>
unsigned chunk_blocks(long long T) {
  return (unsigned)(((T + 32 * K - 1) / (32 * K) + WARPS_A - 1) / WARPS_A);
}

template <typename Kernel, typename... Args>
void launch_cluster(Kernel kernel, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(CLUSTER, 1, 1);
  cfg.blockDim = dim3(CLUSTER_THREADS, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CLUSTER;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  check_cuda(cudaLaunchKernelEx(&cfg, kernel, args...), "loss cluster launch");
  count_launch();
}

}  // namespace

long long packed_partials(long long T, int sequences) {
  const long long tokens = 32 * (T <= kOneLaunch ? NARROW : WIDE);
  return ((T + tokens - 1) / tokens + sequences) * WORDS;
}

void preference_loss_fwd(const float* log_probs, const float* reference, PackedTokens tokens, PreferenceArgs args, float* partials,
                         float* loss, float* chosen, float* rejected, float* slope, cudaStream_t stream) {
  const PreferenceIn in = {log_probs, reference};
  if (tokens.T <= kOneLaunch) {
    launch_cluster(preference_cluster_kernel<NARROW, true>, stream, in, tokens, args, partials, loss, chosen, rejected, slope);
    return;
  }
  preference_chunks_kernel<WIDE><<<chunk_blocks<WIDE>(tokens.T), WARPS_A * 32, 0, stream>>>(in, tokens, partials);
  count_launch();
  check_cuda(cudaGetLastError(), "preference_loss launch");
  launch_cluster(preference_cluster_kernel<WIDE, false>, stream, in, tokens, args, partials, loss, chosen, rejected, slope);
}

void preference_loss_bwd(const float* slope, const float* d_loss, long long d_loss_stride, PackedTokens tokens, float* grad,
    cudaStream_t stream) {
  if (tokens.T == 0) return;
  if (tokens.T <= kOneLaunch)
    preference_bwd_kernel<NARROW><<<chunk_blocks<NARROW>(tokens.T), WARPS_A * 32, 0, stream>>>(slope, d_loss, d_loss_stride, tokens, grad);
  else preference_bwd_kernel<WIDE><<<chunk_blocks<WIDE>(tokens.T), WARPS_A * 32, 0, stream>>>(slope, d_loss, d_loss_stride, tokens, grad);
  count_launch();
  check_cuda(cudaGetLastError(), "preference_loss backward launch");
}

void policy_loss_fwd(const float* log_probs, const float* old_log_probs, const float* reference, const float* advantages,
    PackedTokens tokens, PolicyArgs args, float* partials, PolicyOut out, float* slope, float* weight, cudaStream_t stream) {
  const PolicyIn in = {log_probs, old_log_probs, reference, advantages};
  if (tokens.T <= kOneLaunch) {
    launch_cluster(policy_cluster_kernel<NARROW, true>, stream, in, tokens, args, partials, out, slope, weight);
    return;
  }
  policy_chunks_kernel<WIDE><<<chunk_blocks<WIDE>(tokens.T), WARPS_A * 32, 0, stream>>>(in, tokens, args, partials, slope);
  count_launch();
  check_cuda(cudaGetLastError(), "policy_loss launch");
  launch_cluster(policy_cluster_kernel<WIDE, false>, stream, in, tokens, args, partials, out, slope, weight);
}

void policy_loss_bwd(const float* slope, const float* factor, const float* weight, const float* d_loss, PackedTokens tokens, int reduction,
                     float* grad, cudaStream_t stream) {
  if (tokens.T == 0) return;
  if (tokens.T <= kOneLaunch)
    policy_bwd_kernel<NARROW><<<chunk_blocks<NARROW>(tokens.T), WARPS_A * 32, 0, stream>>>(slope, factor, weight, d_loss, tokens,
        reduction, grad);
  else
    policy_bwd_kernel<WIDE><<<chunk_blocks<WIDE>(tokens.T), WARPS_A * 32, 0, stream>>>(slope, factor, weight, d_loss, tokens, reduction,
        grad);
  count_launch();
  check_cuda(cudaGetLastError(), "policy_loss backward launch");
}

}  // namespace b200
