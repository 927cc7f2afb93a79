// Log-probability of one given token per row of logits, and the row's entropy:
//   z = logit_scale * logits,  L = logsumexp(z),  p = exp(z - L)
//   log_prob = z[label] - L,   entropy = L - sum_j p_j z_j
//   d logits_j = logit_scale * ( g (1[j = label] - p_j) - h p_j (z_j - L + entropy) )
// with g, h the upstream gradients of the two outputs. Exponents are held in base 2, where the exponential is one
// instruction; sums are fp32 and each value is rounded once, when it is stored.
//
// Forward: one pass with the running statistics of softmax_stats.cuh per thread, joined
// over the CTA. Backward: one pass that reads the logits again and writes the gradient, since no gradient of a row is
// known before its last logit has been read and a row (100 to 500 KB) does not stay on the SM until the upstream
// gradient arrives. Both are bound by HBM.
//
// Rows may start at any element: a row that is not 16-byte aligned is read as aligned 16-byte words that are shifted
// together (a row's shift is uniform), its first and last vectors element by element, so nothing outside of the row is
// ever read. Ignored rows (label == ignore_index or outside of [0, V)) are not read at all: their outputs and gradients are 0,
// whatever they hold.
#include <cuda_fp16.h>

#include "../common/cta_pair.cuh"
#include "../common/launch.h"
#include "../common/ptx.cuh"
#include "softmax_stats.cuh"
#include "vocabulary.h"

namespace b200 {

namespace {

__device__ __forceinline__ long long row_offset(const RowMap& m, long long row) {
  const long long o = row / m.inner;
  return o * m.outer_stride + (row - o * m.inner) * m.row_stride;
}

// 16 bytes of logits: as fp32 pairs, their maximum, and back.
template <typename T>
struct Vec;
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(uint4 v, F2* f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = pack2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ float top(uint32_t w) { return fmaxf(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
  static __device__ __forceinline__ uint32_t pack(float2 f) { return pack_bf16x2(f.x, f.y); }
  static __device__ __forceinline__ float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, float f) { *p = __float2bfloat16(f); }
  static __device__ __forceinline__ uint32_t bits(const __nv_bfloat16* p) { return *reinterpret_cast<const uint16_t*>(p); }
  static constexpr uint32_t kNegInf = 0xff80u;
};
template <>
struct Vec<__half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(uint4 v, F2* f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[i] = pack2(a.x, a.y);
    }
  }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    const __half2 r = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ float top(uint32_t w) {
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w));
    return fmaxf(a.x, a.y);
  }
  static __device__ __forceinline__ uint32_t pack(float2 f) {
    const __half2 h = __floats2half2_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float load(const __half* p) { return __half2float(*p); }
  static __device__ __forceinline__ void store(__half* p, float f) { *p = __float2half_rn(f); }
  static __device__ __forceinline__ uint32_t bits(const __half* p) { return *reinterpret_cast<const uint16_t*>(p); }
  static constexpr uint32_t kNegInf = 0xfc00u;
};
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(uint4 v, F2* f) {
    f[0] = pack2(__uint_as_float(v.x), __uint_as_float(v.y));
    f[1] = pack2(__uint_as_float(v.z), __uint_as_float(v.w));
  }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }
  static __device__ __forceinline__ float top(uint32_t w) { return __uint_as_float(w); }
  static __device__ __forceinline__ float load(const float* p) { return *p; }
  static __device__ __forceinline__ void store(float* p, float f) { *p = f; }
  static __device__ __forceinline__ uint32_t bits(const float* p) { return __float_as_uint(*p); }
  static constexpr uint32_t kNegInf = 0xff800000u;
};

template <typename T>
__device__ __forceinline__ uint4 pack_vector(const F2* f) {
  if constexpr (sizeof(T) == 4) {
    const float2 a = unpack2(f[0]), b = unpack2(f[1]);
    return make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
  } else {
    return make_uint4(Vec<T>::pack(unpack2(f[0])), Vec<T>::pack(unpack2(f[1])), Vec<T>::pack(unpack2(f[2])), Vec<T>::pack(unpack2(f[3])));
  }
}

// The 16 bytes at `p + shift` of two aligned words, shift in bytes (1..15).
__device__ __forceinline__ uint4 join_words(uint4 a, uint4 b, int shift) {
  uint32_t w0, w1, w2, w3, w4;
  switch (shift >> 2) {
    case 0: w0 = a.x; w1 = a.y; w2 = a.z; w3 = a.w; w4 = b.x; break;
    case 1: w0 = a.y; w1 = a.z; w2 = a.w; w3 = b.x; w4 = b.y; break;
    case 2: w0 = a.z; w1 = a.w; w2 = b.x; w3 = b.y; w4 = b.z; break;
    default: w0 = a.w; w1 = b.x; w2 = b.y; w3 = b.z; w4 = b.w; break;
  }
  const int bits = (shift & 3) * 8;
  return make_uint4(__funnelshift_r(w0, w1, bits), __funnelshift_r(w1, w2, bits), __funnelshift_r(w2, w3, bits),
                    __funnelshift_r(w3, w4, bits));
}

// A row cut into vectors of Vec<T>::N elements: vector i covers elements [i N, i N + N), the last one may be short.
template <typename T>
struct Row {
  const T* p;
  int V, vectors, shift;  // shift: bytes by which the row start lies above a 16-byte boundary

  __device__ __forceinline__ Row(const T* start, int v)
      : p(start), V(v), vectors((v + Vec<T>::N - 1) / Vec<T>::N), shift((int)(reinterpret_cast<uintptr_t>(start) & 15)) {}

  // [first_wide, end_wide): whole vectors whose 16-byte words all lie inside of the row
  __device__ __forceinline__ int first_wide() const { return shift == 0 ? 0 : 1; }
  __device__ __forceinline__ int end_wide() const { return shift == 0 ? V / Vec<T>::N : max(1, V / Vec<T>::N - 1); }
  template <bool ALIGNED>
  __device__ __forceinline__ uint4 load_wide(int i) const {
    if constexpr (ALIGNED) return __ldg(reinterpret_cast<const uint4*>(p) + i);
    const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(p + (long long)i * Vec<T>::N) & ~uintptr_t(15));
    return join_words(__ldg(q), __ldg(q + 1), shift);
  }
  __device__ __forceinline__ uint4 load(int i) const {
    if (i < first_wide() || i >= end_wide()) return load_narrow(i);
    return shift == 0 ? load_wide<true>(i) : load_wide<false>(i);
  }
  // element by element; elements past the row's end read as -inf (probability 0)
  __device__ __forceinline__ uint4 load_narrow(int i) const {
    uint32_t w[4];
    constexpr int kPerWord = 4 / (int)sizeof(T);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      w[k] = 0;
#pragma unroll
      for (int e = 0; e < kPerWord; ++e) {
        const int j = i * Vec<T>::N + k * kPerWord + e;
        w[k] |= (j < V ? Vec<T>::bits(p + j) : Vec<T>::kNegInf) << (16 * e);
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// Measured at 4096 x 128256 bf16, one row in eight ignored (0.92 GB): two blocks of 512 threads on an SM with four vectors a thread in flight
// 174 us, four of 256 158, five of 256 with three vectors 156 (5.9 TB/s); fetching the next vectors before the present ones are
// worked on gains 2 us more at the cost of the registers of one block, and is left out.
constexpr int FWD_THREADS = 256;
constexpr int FWD_UNROLL = 3;
constexpr int FWD_BLOCKS = 5;

// COUNT vectors of a thread at once; one comparison of their common maximum with the running one decides about rescaling.
template <typename T, bool ENTROPY, int COUNT>
__device__ __forceinline__ void accumulate_vectors(Stats& st, const uint4 (&v)[COUNT], float scale2) {
  constexpr int N = Vec<T>::N;
  uint32_t top = v[0].x;
  F2 f[COUNT * N / 2];
#pragma unroll
  for (int k = 0; k < COUNT; ++k) {
    top = Vec<T>::max2(top, Vec<T>::max2(Vec<T>::max2(v[k].x, v[k].y), Vec<T>::max2(v[k].z, v[k].w)));
    Vec<T>::unpack(v[k], f + k * (N / 2));
  }
  accumulate<ENTROPY, COUNT * N>(st, f, Vec<T>::top(top), scale2);
}

// The wide vectors of a row in groups of three per thread whose loads have no condition between them (the compiler keeps loads
// behind a branch in order, one in flight: 222 instead of 150 us at 4096 x 128256 bf16).
template <typename T, bool ENTROPY, bool ALIGNED>
__device__ __forceinline__ void accumulate_wide(Stats& st, const Row<T>& r, int first, int end, float scale2) {
  int i = first + threadIdx.x;
  for (; i + (FWD_UNROLL - 1) * FWD_THREADS < end; i += FWD_UNROLL * FWD_THREADS) {
    uint4 v[FWD_UNROLL];
#pragma unroll
    for (int k = 0; k < FWD_UNROLL; ++k) v[k] = r.template load_wide<ALIGNED>(i + k * FWD_THREADS);
    accumulate_vectors<T, ENTROPY, FWD_UNROLL>(st, v, scale2);
  }
  for (; i < end; i += FWD_THREADS) {
    const uint4 v[1] = {r.template load_wide<ALIGNED>(i)};
    accumulate_vectors<T, ENTROPY, 1>(st, v, scale2);
  }
}

// CLUSTER blocks share a row.
template <typename T, bool ENTROPY, int CLUSTER>
__global__ void __launch_bounds__(FWD_THREADS, FWD_BLOCKS)
    token_log_probs_fwd_kernel(const T* __restrict__ logits, const void* __restrict__ labels, bool labels64,
                               float* __restrict__ log_probs, float* __restrict__ entropy, float2* __restrict__ lse, int V,
                               RowMap map, float logit_scale, float scale2, long long ignore_index) {
  __shared__ Stats red[FWD_THREADS / 32];
  __shared__ Stats block_stats;
  const long long row = blockIdx.x / CLUSTER;
  const int rank = blockIdx.x % CLUSTER;
  const long long label = load_label(labels, labels64, row);
  if (label == ignore_index || label < 0 || label >= V) {  // all blocks of the row leave
    if (threadIdx.x == 0 && rank == 0) {
      log_probs[row] = 0.f;
      lse[row] = make_float2(0.f, 0.f);
      if (ENTROPY) entropy[row] = 0.f;
    }
    return;
  }
  const Row<T> r(logits + row_offset(map, row), V);
  Stats st = empty_stats();
  const int before = r.first_wide(), behind = max(r.end_wide(), before);
  const int share = (behind - before + CLUSTER - 1) / CLUSTER;
  const int first = before + rank * share, end = min(behind, first + share);
  if (r.shift == 0) accumulate_wide<T, ENTROPY, true>(st, r, first, end, scale2);
  else accumulate_wide<T, ENTROPY, false>(st, r, first, end, scale2);
  // the (at most three) vectors at the ends of the row that are not wide, one thread each
  const int narrow = before + r.vectors - behind;
  if (rank == 0 && threadIdx.x < narrow) {
    const uint4 v[1] = {r.load_narrow(threadIdx.x < before ? threadIdx.x : behind + threadIdx.x - before)};
    accumulate_vectors<T, ENTROPY, 1>(st, v, scale2);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stats other;
    other.m = __shfl_xor_sync(0xffffffffu, st.m, o);
    other.s = __shfl_xor_sync(0xffffffffu, st.s, o);
    other.u = ENTROPY ? __shfl_xor_sync(0xffffffffu, st.u, o) : 0.f;
    st = merge<ENTROPY>(st, other, scale2);
  }
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = st;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < FWD_THREADS / 32; ++w) st = merge<ENTROPY>(st, red[w], scale2);
    block_stats = st;
  }
  if (CLUSTER > 1) {
    cluster_sync_all();
    if (rank == 0 && threadIdx.x == 0) {
#pragma unroll
      for (int b = 1; b < CLUSTER; ++b) {
        Stats other;
        const uint32_t at = map_to_cta(smem_u32(&block_stats), b);
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(other.m) : "r"(at) : "memory");
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(other.s) : "r"(at + 4) : "memory");
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(other.u) : "r"(at + 8) : "memory");
        st = merge<ENTROPY>(st, other, scale2);
      }
    }
    cluster_sync_all();  // nobody leaves while its statistics are read
  }
  if (threadIdx.x == 0 && rank == 0) {
    const float log2_s = log2f(st.s);
    lse[row] = make_float2(st.m, log2_s);
    log_probs[row] = log_prob(Vec<T>::load(r.p + label), make_float2(st.m, log2_s), logit_scale);
    if (ENTROPY) entropy[row] = (log2_s - st.u / st.s) * kLn2;
  }
}

constexpr int BWD_THREADS = 256;
constexpr int BWD_UNROLL = 8;  // 32 KB of a row per block; with 16 KB 335 us, with 64 KB 350

template <typename T, bool ENTROPY>
__global__ void __launch_bounds__(BWD_THREADS)
    token_log_probs_bwd_kernel(const T* __restrict__ logits, const void* __restrict__ labels, bool labels64,
                               const float2* __restrict__ lse, const float* __restrict__ entropy,
                               const float* __restrict__ d_log_probs, long long d_log_probs_stride,
                               const float* __restrict__ d_entropy, long long d_entropy_stride, T* __restrict__ grad, int V,
                               RowMap map, long long grad_stride, float logit_scale, float scale2,
                               long long ignore_index, unsigned chunks) {
  constexpr int N = Vec<T>::N;
  // last row first: the logits that the forward pass (or the model) touched last are still in L2
  // and the blocks of a row are consecutive: 4096 x 128256 354 -> 333 us with 16 KB a block, 301 us (6.5 TB/s of 2.0 GB) with 32 KB
  const unsigned chunk = blockIdx.x % chunks;
  const long long row = gridDim.x / chunks - 1 - blockIdx.x / chunks;
  const long long label = load_label(labels, labels64, row);
  const bool ignored = label == ignore_index || label < 0 || label >= V;
  const Row<T> r(logits + row_offset(map, row), V);
  T* out = grad + row * grad_stride;
  const float g = ignored ? 0.f : d_log_probs[row * d_log_probs_stride];
  const float h = ignored || !ENTROPY ? 0.f : d_entropy[row * d_entropy_stride];
  const int i0 = chunk * (BWD_THREADS * BWD_UNROLL) + threadIdx.x;
  // rows without an upstream gradient get zeros and are not read
  const bool zero = g == 0.f && h == 0.f;
  const float2 L = lse[row];
  const float H = ENTROPY ? entropy[row] : 0.f;
  const float gs = g * logit_scale, hs = h * logit_scale;
  uint4 v[BWD_UNROLL];
  const int last = chunk * (BWD_THREADS * BWD_UNROLL) + BWD_THREADS * BWD_UNROLL;
  if (zero) {
#pragma unroll
    for (int k = 0; k < BWD_UNROLL; ++k) v[k] = make_uint4(0, 0, 0, 0);
  } else if (r.shift == 0 && last <= r.end_wide()) {
#pragma unroll
    for (int k = 0; k < BWD_UNROLL; ++k) v[k] = r.template load_wide<true>(i0 + k * BWD_THREADS);
  } else if (chunk > 0 && last <= r.end_wide()) {
#pragma unroll
    for (int k = 0; k < BWD_UNROLL; ++k) v[k] = r.template load_wide<false>(i0 + k * BWD_THREADS);
  } else {
#pragma unroll
    for (int k = 0; k < BWD_UNROLL; ++k) {
      const int i = i0 + k * BWD_THREADS;
      v[k] = make_uint4(0, 0, 0, 0);
      if (i < r.vectors) v[k] = r.load(i);
    }
  }
  const F2 c2 = pack2(scale2, scale2), off2 = pack2(-L.x, -L.x), log2_s = pack2(-L.y, -L.y), gs2 = pack2(-gs, -gs);
  const int label_vector = zero ? -1 : (int)(label / N);
#pragma unroll
  for (int k = 0; k < BWD_UNROLL; ++k) {
    const int i = i0 + k * BWD_THREADS;
    if (i >= r.vectors) return;
    F2 f[N / 2];
    Vec<T>::unpack(v[k], f);
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
      if (zero) {
        f[j] = pack2(0.f, 0.f);
        continue;
      }
      const float2 d = unpack2(fma2(add2(f[j], off2), c2, log2_s));
      const F2 p = pack2(fast_exp2(d.x), fast_exp2(d.y));
      if (ENTROPY) {
        const F2 w = pack2(-fmaf(hs, fmaf(fmaxf(d.x, kFloor2), kLn2, H), gs), -fmaf(hs, fmaf(fmaxf(d.y, kFloor2), kLn2, H), gs));
        f[j] = mul2(p, w);
      } else {
        f[j] = mul2(p, gs2);
      }
    }
    if ((i + 1) * N <= V) {
      *reinterpret_cast<uint4*>(out + (long long)i * N) = pack_vector<T>(f);
    } else {
#pragma unroll
      for (int j = 0; j < N / 2; ++j) {
        const float2 a = unpack2(f[j]);
        if (i * N + 2 * j < V) Vec<T>::store(out + i * N + 2 * j, a.x);
        if (i * N + 2 * j + 1 < V) Vec<T>::store(out + i * N + 2 * j + 1, a.y);
      }
    }
    // the label's own gradient, over the vector just written by this thread
    if (i == label_vector) {
      const float d = log2_prob(Vec<T>::load(r.p + label), L, scale2);
      Vec<T>::store(out + label, gs + score_gradient<ENTROPY>(d, gs, hs, H));
    }
  }
}

// One block: 32 rows (one per lane) x 32 warps that share the slices, eight loads in flight each; then every warp takes one row
// and its lanes join the 32 warps' statistics pairwise.
template <bool ENTROPY>
__global__ void __launch_bounds__(1024)
    token_log_probs_join_kernel(const float4* __restrict__ stats, int slices, int slice_width, const void* __restrict__ labels,
        bool labels64, float* __restrict__ log_probs, float* __restrict__ entropy, float2* __restrict__ lse, LiveRows live, int V,
        float logit_scale, float scale2, long long ignore_index) {
  __shared__ Stats red[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rows = live.count == nullptr ? live.rows : min(live.rows, *live.count - live.base);
  const int r0 = blockIdx.x * 32;
  if (r0 >= rows) return;
  Stats st = empty_stats();
  const float4* column = stats + min(r0 + lane, rows - 1);  // lanes behind the last row repeat it
  constexpr int BATCH = 8;
  for (int i0 = warp; i0 < slices; i0 += 32 * BATCH) {
    float4 v[BATCH];
#pragma unroll
    for (int k = 0; k < BATCH; ++k) v[k] = column[(long long)min(i0 + 32 * k, slices - 1) * live.rows];
#pragma unroll
    for (int k = 0; k < BATCH; ++k)
      if (i0 + 32 * k < slices) st = merge<ENTROPY>(st, Stats{v[k].x, v[k].y, v[k].z}, scale2);
  }
  red[warp][lane] = st;
  __syncthreads();
  const int r = r0 + warp;
  if (r >= rows) return;
  st = red[lane][warp];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stats other;
    other.m = __shfl_xor_sync(0xffffffffu, st.m, o);
    other.s = __shfl_xor_sync(0xffffffffu, st.s, o);
    other.u = ENTROPY ? __shfl_xor_sync(0xffffffffu, st.u, o) : 0.f;
    st = merge<ENTROPY>(st, other, scale2);
  }
  if (lane != 0) return;
  const long long row = live.index != nullptr ? live.index[live.base + r] : live.base + r;
  const long long label = load_label(labels, labels64, row);
  if (label == ignore_index || label < 0 || label >= V) {
    log_probs[row] = 0.f;
    lse[row] = make_float2(0.f, 0.f);
    if (ENTROPY) entropy[row] = 0.f;
    return;
  }
  const float log2_s = log2f(st.s), x = stats[(long long)(label / slice_width) * live.rows + r].w;
  lse[row] = make_float2(st.m, log2_s);
  log_probs[row] = log_prob(x, make_float2(st.m, log2_s), logit_scale);
  if (ENTROPY) entropy[row] = (log2_s - st.u / st.s) * kLn2;
}

template <typename T>
void fwd(const void* logits, const void* labels, bool labels64, float* log_probs, float* entropy, float2* lse, long long rows,
         int V, RowMap map, float logit_scale, long long ignore_index, cudaStream_t stream) {
  const T* x = reinterpret_cast<const T*>(logits);
  auto launch = [&](auto kernel, int cluster) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * cluster), 1, 1);
    cfg.blockDim = dim3(FWD_THREADS, 1, 1);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 1 : 0;
    check_cuda(cudaLaunchKernelEx(&cfg, kernel, x, labels, labels64, log_probs, entropy, lse, V, map, logit_scale,
        logit_scale * kLog2e, ignore_index), "token_log_probs forward launch");
  };
  // Blocks per row: more than one only while all of them run at once, four per SM, and each has a vector per thread. Few long rows
  // gain (32 x 49152 bf16: 7.8 us with one block of 1024 threads, 6.6 with eight of 256); with more blocks than run at a time the
  // two cluster barriers of a row cost more than the shorter last wave saves (1531 x 50001 fp32: 54 us with one, 61 with two).
  const int vectors = V / Vec<T>::N;
  int cluster = 1;
  while (cluster < 8 && 2 * rows * cluster <= 4LL * sm_count() && vectors / (2 * cluster) >= FWD_THREADS) cluster *= 2;
  const bool e = entropy != nullptr;
  switch (cluster) {
    case 1: e ? launch(token_log_probs_fwd_kernel<T, true, 1>, 1) : launch(token_log_probs_fwd_kernel<T, false, 1>, 1); break;
    case 2: e ? launch(token_log_probs_fwd_kernel<T, true, 2>, 2) : launch(token_log_probs_fwd_kernel<T, false, 2>, 2); break;
    case 4: e ? launch(token_log_probs_fwd_kernel<T, true, 4>, 4) : launch(token_log_probs_fwd_kernel<T, false, 4>, 4); break;
    default: e ? launch(token_log_probs_fwd_kernel<T, true, 8>, 8) : launch(token_log_probs_fwd_kernel<T, false, 8>, 8); break;
  }
}

template <typename T>
void bwd(const void* logits, const void* labels, bool labels64, const float2* lse, const float* entropy, const float* d_log_probs,
         long long d_log_probs_stride, const float* d_entropy, long long d_entropy_stride, void* grad, long long rows, int V,
         RowMap map, long long grad_stride, float logit_scale, long long ignore_index, cudaStream_t stream) {
  const T* x = reinterpret_cast<const T*>(logits);
  const int vectors = (V + Vec<T>::N - 1) / Vec<T>::N;
  const unsigned chunks = (unsigned)((vectors + BWD_THREADS * BWD_UNROLL - 1) / (BWD_THREADS * BWD_UNROLL));
  const unsigned grid = (unsigned)rows * chunks;
  const float scale2 = logit_scale * kLog2e;
  if (d_entropy != nullptr)
    token_log_probs_bwd_kernel<T, true><<<grid, BWD_THREADS, 0, stream>>>(x, labels, labels64, lse, entropy, d_log_probs,
        d_log_probs_stride, d_entropy, d_entropy_stride, reinterpret_cast<T*>(grad), V, map, grad_stride, logit_scale, scale2,
        ignore_index, chunks);
  else
    token_log_probs_bwd_kernel<T, false><<<grid, BWD_THREADS, 0, stream>>>(x, labels, labels64, lse, entropy, d_log_probs,
        d_log_probs_stride, d_entropy, d_entropy_stride, reinterpret_cast<T*>(grad), V, map, grad_stride, logit_scale, scale2,
        ignore_index, chunks);
}

}  // namespace

void token_log_probs_fwd(const void* logits, Scalar type, const void* labels, bool labels64, float* log_probs, float* entropy,
                         float2* lse, long long T, int V, RowMap map, float logit_scale, long long ignore_index, cudaStream_t stream) {
  if (T == 0) return;
  auto launch = type == Scalar::kBf16 ? fwd<__nv_bfloat16> : type == Scalar::kF16 ? fwd<__half> : fwd<float>;
  launch(logits, labels, labels64, log_probs, entropy, lse, T, V, map, logit_scale, ignore_index, stream);
  count_launch();
  check_cuda(cudaGetLastError(), "token_log_probs forward launch");
}

void token_log_probs_bwd(const void* logits, Scalar type, const void* labels, bool labels64, const float2* lse,
                         const float* entropy, const float* d_log_probs, long long d_log_probs_stride, const float* d_entropy,
                         long long d_entropy_stride, void* grad, long long T, int V, RowMap map, long long grad_stride,
                         float logit_scale, long long ignore_index, cudaStream_t stream) {
  if (T == 0) return;
  auto launch = type == Scalar::kBf16 ? bwd<__nv_bfloat16> : type == Scalar::kF16 ? bwd<__half> : bwd<float>;
  launch(logits, labels, labels64, lse, entropy, d_log_probs, d_log_probs_stride, d_entropy, d_entropy_stride, grad, T, V, map,
         grad_stride, logit_scale, ignore_index, stream);
  count_launch();
  check_cuda(cudaGetLastError(), "token_log_probs backward launch");
}

void token_log_probs_join(const float* stats, int slices, int slice_width, const void* labels, bool labels64, float* log_probs,
    float* entropy, float2* lse, LiveRows live, int V, float logit_scale, long long ignore_index, cudaStream_t stream) {
  if (live.rows <= 0) return;
  const unsigned blocks = (unsigned)((live.rows + 31) / 32);
  const float4* st = reinterpret_cast<const float4*>(stats);
  if (entropy != nullptr)
    token_log_probs_join_kernel<true><<<blocks, 1024, 0, stream>>>(st, slices, slice_width, labels, labels64, log_probs, entropy, lse,
        live, V, logit_scale, logit_scale * kLog2e, ignore_index);
  else
    token_log_probs_join_kernel<false><<<blocks, 1024, 0, stream>>>(st, slices, slice_width, labels, labels64, log_probs, entropy, lse,
        live, V, logit_scale, logit_scale * kLog2e, ignore_index);
  count_launch();
  check_cuda(cudaGetLastError(), "token_log_probs join launch");
}

// ------------------------------------------------------------------------- gradient of kept logits
namespace {

constexpr int GRAD_THREADS = 256;
constexpr int GRAD_UNROLL = 4;  // vectors of eight columns per thread: 32 KB of a row per block

// fp32 rows in, bf16 rows out; the blocks of a row are consecutive. Rows from the live ones to the next multiple of 256 are cleared, those
// behind are left alone.
template <bool ENTROPY>
__global__ void __launch_bounds__(GRAD_THREADS)
    grad_rows_kernel(const float* __restrict__ logits, long long ldl, const void* __restrict__ labels, bool labels64,
        const float2* __restrict__ lse, const float* __restrict__ entropy, const float* __restrict__ d_log_probs,
        long long d_log_probs_stride, const float* __restrict__ d_entropy, long long d_entropy_stride, __nv_bfloat16* __restrict__ grad,
        long long ldg, LiveRows live, int V, float logit_scale, float scale2, long long ignore_index, unsigned chunks) {
  const unsigned chunk = blockIdx.x % chunks;
  const int r = blockIdx.x / chunks;
  const int rows = live.count == nullptr ? live.rows : max(0, min(live.rows, *live.count - live.base));
  if (r >= rows && (live.count == nullptr || r >= max(256, (rows + 255) / 256 * 256))) return;
  float gs = 0.f, hs = 0.f, H = 0.f;
  float2 L = make_float2(0.f, 0.f);
  long long label = -1;
  if (r < rows) {
    const long long t = live.index != nullptr ? live.index[live.base + r] : live.base + r;
    label = load_label(labels, labels64, t);
    if (label != ignore_index && label >= 0 && label < V) {
      L = lse[t];
      gs = d_log_probs[t * d_log_probs_stride] * logit_scale;
      if (ENTROPY) {
        hs = d_entropy[t * d_entropy_stride] * logit_scale;
        H = entropy[t];
      }
    }
  }
  const bool zero = gs == 0.f && hs == 0.f;
  const float* x = logits + (long long)r * ldl;
  __nv_bfloat16* out = grad + (long long)r * ldg;
  const int i0 = chunk * (GRAD_THREADS * GRAD_UNROLL) + threadIdx.x;
  uint4 v[GRAD_UNROLL][2];
  const bool whole = ((int)chunk + 1) * (GRAD_THREADS * GRAD_UNROLL * 8) <= V;
  if (whole && !zero) {
#pragma unroll
    for (int k = 0; k < GRAD_UNROLL; ++k) {
      const uint4* q = reinterpret_cast<const uint4*>(x + (long long)(i0 + k * GRAD_THREADS) * 8);
      v[k][0] = __ldg(q);
      v[k][1] = __ldg(q + 1);
    }
  } else {
#pragma unroll
    for (int k = 0; k < GRAD_UNROLL; ++k) {
      uint32_t w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int j = (i0 + k * GRAD_THREADS) * 8 + e;
        w[e] = !zero && j < V ? __float_as_uint(x[j]) : 0u;
      }
      v[k][0] = make_uint4(w[0], w[1], w[2], w[3]);
      v[k][1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
  }
  const F2 c2 = pack2(scale2, scale2), off2 = pack2(-L.x, -L.x), log2_s = pack2(-L.y, -L.y), gs2 = pack2(-gs, -gs);
#pragma unroll
  for (int k = 0; k < GRAD_UNROLL; ++k) {
    const int i = i0 + k * GRAD_THREADS;
    if (i * 8 >= V) return;
    F2 f[4];
    Vec<float>::unpack(v[k][0], f);
    Vec<float>::unpack(v[k][1], f + 2);
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 d = unpack2(fma2(add2(f[j], off2), c2, log2_s));
      const F2 p = pack2(fast_exp2(d.x), fast_exp2(d.y));
      float2 y;
      if (ENTROPY) y = unpack2(mul2(p, pack2(-fmaf(hs, fmaf(fmaxf(d.x, kFloor2), kLn2, H), gs),
          -fmaf(hs, fmaf(fmaxf(d.y, kFloor2), kLn2, H), gs))));
      else y = unpack2(mul2(p, gs2));
      w[j] = zero ? 0u : pack_bf16x2(y.x, y.y);
    }
    if ((i + 1) * 8 <= V) {
      *reinterpret_cast<uint4*>(out + (long long)i * 8) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (i * 8 + e < V) reinterpret_cast<uint16_t*>(out)[i * 8 + e] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
    }
    // the label's own gradient, over the vector just written by this thread
    if (!zero && label >> 3 == i) out[label] = __float2bfloat16(gs + score_gradient<ENTROPY>(log2_prob(x[label], L, scale2), gs, hs, H));
  }
}

}  // namespace

void token_log_probs_grad_rows(const float* logits, long long ldl, const void* labels, bool labels64, const float2* lse,
    const float* entropy, const float* d_log_probs, long long d_log_probs_stride, const float* d_entropy, long long d_entropy_stride,
    void* grad, long long ldg, LiveRows live, int N, float logit_scale, long long ignore_index, cudaStream_t stream) {
  if (live.rows <= 0) return;
  constexpr int kColumns = GRAD_THREADS * GRAD_UNROLL * 8;
  const unsigned chunks = (unsigned)((N + kColumns - 1) / kColumns);
  auto kernel = d_entropy != nullptr ? grad_rows_kernel<true> : grad_rows_kernel<false>;
  kernel<<<(unsigned)live.rows * chunks, GRAD_THREADS, 0, stream>>>(logits, ldl, labels, labels64, lse, entropy, d_log_probs,
      d_log_probs_stride, d_entropy, d_entropy_stride, reinterpret_cast<__nv_bfloat16*>(grad), ldg, live, N, logit_scale,
      logit_scale * kLog2e, ignore_index, chunks);
  count_launch();
  check_cuda(cudaGetLastError(), "kept logits gradient launch");
}

// ------------------------------------------------------------------------- live rows of a batch
namespace {

// A block takes `share` consecutive rows of the batch: it counts the live rows before them (all of the earlier labels, from L2), which
// gives its rows their places, and copies the live ones there, a warp per row. The d-th row that does not count clears compact row
// T - 1 - d, so that all rows behind the live ones are zeros.
constexpr int COMPACT_THREADS = 256;

__global__ void __launch_bounds__(COMPACT_THREADS)
    compact_rows_kernel(const void* __restrict__ labels, bool labels64, long long ignore_index, int T, int V,
        const __nv_bfloat16* __restrict__ x, long long ldx, int H, int share, int* __restrict__ index, int* __restrict__ count,
        __nv_bfloat16* __restrict__ compact, float* __restrict__ log_probs, float* __restrict__ entropy, float2* __restrict__ lse) {
  __shared__ int warp_count[COMPACT_THREADS / 32], place[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int first = blockIdx.x * share, end = min(T, first + share);
  auto is_live = [&](int t) {
    const long long l = load_label(labels, labels64, t);
    return l != ignore_index && l >= 0 && l < V;
  };
  int n = 0;
#pragma unroll 4
  for (int t = threadIdx.x; t < first; t += COMPACT_THREADS) n += is_live(t) ? 1 : 0;
  n = __reduce_add_sync(0xffffffffu, n);
  if (lane == 0) warp_count[warp] = n;
  __syncthreads();
  int before = 0;
#pragma unroll
  for (int w = 0; w < COMPACT_THREADS / 32; ++w) before += warp_count[w];
  for (int t0 = first; t0 < end; t0 += 32) {
    if (warp == 0) {
      const int t = t0 + lane;
      const bool live = t < end && is_live(t);
      const unsigned votes = __ballot_sync(0xffffffffu, live);
      const int p = before + __popc(votes & ((1u << lane) - 1));  // live rows before t
      before += __popc(votes);
      if (t < end) {
        if (live) {
          index[p] = t;
        } else {
          log_probs[t] = 0.f;
          lse[t] = make_float2(0.f, 0.f);
          if (entropy != nullptr) entropy[t] = 0.f;
        }
        if (t == T - 1) *count = p + (live ? 1 : 0);
        place[lane] = live ? p : -(T - 1 - (t - p)) - 1;
      }
    }
    __syncthreads();
    for (int k = warp; k < 32 && t0 + k < end; k += COMPACT_THREADS / 32) {
      const int p = place[k];
      uint4* dst = reinterpret_cast<uint4*>(compact + (long long)(p >= 0 ? p : -p - 1) * H);
      const uint4* src = reinterpret_cast<const uint4*>(x + (long long)(t0 + k) * ldx);
      if (p >= 0) {
#pragma unroll 8
        for (int i = lane; i < H / 8; i += 32) dst[i] = src[i];
      } else {
        for (int i = lane; i < H / 8; i += 32) dst[i] = make_uint4(0, 0, 0, 0);
      }
    }
    __syncthreads();
  }
}

}  // namespace

void vocab_compact_rows(const void* labels, bool labels64, long long ignore_index, int T, int V, const void* x, long long ldx, int H,
    int* index, int* count, void* compact, float* log_probs, float* entropy, float2* lse, cudaStream_t stream) {
  // a row per warp as long as that makes at most 1024 blocks (each of them reads all labels before its rows)
  int share = 8;
  while ((T + share - 1) / share > 1024) share *= 2;
  compact_rows_kernel<<<(T + share - 1) / share, COMPACT_THREADS, 0, stream>>>(labels, labels64, ignore_index, T, V,
      reinterpret_cast<const __nv_bfloat16*>(x), ldx, H, share, index, count, reinterpret_cast<__nv_bfloat16*>(compact), log_probs,
      entropy, lse);
  count_launch();
  check_cuda(cudaGetLastError(), "compact rows launch");
}

}  // namespace b200
