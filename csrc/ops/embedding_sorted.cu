// Embedding lookup, out[t] = scale * W[id_t], and its gradient summed in sorted token order:
//   dW[v] = scale * sum over t with id_t = v of dout[t]
//
// The gradient sorts the pairs (id, t) as 64-bit keys, which are distinct, so their order is unique and every sum is taken in
// the same order on every run, one fixed by the ids and the sizes: ascending t inside of a chunk, and the chunks' parts by every fourth on four
// lanes, lane after lane; nothing is added atomically. Sorting: runs of 1024 keys in shared memory (bitonic), then
// levels that merge 16 runs at a time by rank: a key's place is its place in its own run plus the number of smaller keys in
// each of the 15 others (independent binary searches, 16 loads in flight). Summing: a block takes 8 to 128 consecutive sorted
// tokens (a chunk) and a slab of columns and reads each dout row once; a run of equal ids inside of the chunk goes straight to its row of
// dW, a run that crosses the border to the next chunk leaves fp32 partial sums, which a last kernel joins in order. A chunk of fp32 rows and
// the parts of a run are added in 64 bits, a chunk of 16-bit rows in 32 (at most 128 values of 8 or 11 bits): what is rounded is a part, once, and
// the row of dW, once. In 32 bits throughout the error of a frequent token grew with its rows (relative, fp32: 5e-8 at 1000 rows, 3e-7 at 1e6,
// now 2e-8 at either) and 10001 x 1536 fp32, both directions, took 96.5 us instead of 98.5.
//
// Bound by HBM: dout is read once, the rows of dW are written once (read and written when they are accumulated into).
#include <cuda_fp16.h>

#include "../common/launch.h"
#include "../common/ptx.cuh"
#include "vocabulary.h"

namespace b200 {

namespace {

constexpr int LOG_RUN = 10, RUN = 1 << LOG_RUN;  // keys sorted by one block
constexpr int LOG_FAN = 4, FAN = 1 << LOG_FAN;  // runs merged per level
constexpr int MAX_CHUNK = 128;   // sorted tokens summed by one block, at most
constexpr int SUM_THREADS = 128;
constexpr uint64_t kNoKey = ~0ull;
constexpr uint32_t kNoId = 0x7fffffffu;  // ids outside of the table, sorted behind all others

__device__ __forceinline__ uint32_t key_id(uint64_t key) { return (uint32_t)(key >> 32); }

__device__ __forceinline__ long long load_id(const void* ids, bool ids64, long long t) {
  return ids64 ? reinterpret_cast<const long long*>(ids)[t] : reinterpret_cast<const int*>(ids)[t];
}

// ------------------------------------------------------------------------- element types
template <typename T, int N>
struct Pack;
template <typename T>
struct Pack<T, 1> {
  T v;
};
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16(x); }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T* p) {
  return *reinterpret_cast<const Pack<T, N>*>(p);
}
template <typename T, int N>
__device__ __forceinline__ float element(const Pack<T, N>& p, int i) {
  if constexpr (N == 1) return to_float(p.v);
  else return to_float(p.v[i]);
}
template <typename T, int N>
__device__ __forceinline__ void set_element(Pack<T, N>& p, int i, float f) {
  if constexpr (N == 1) p.v = from_float<T>(f);
  else p.v[i] = from_float<T>(f);
}

// ------------------------------------------------------------------------- lookup
constexpr int LOOKUP_ROWS = 4;
constexpr int LOOKUP_THREADS = 128;

template <typename T, int N>
__global__ void __launch_bounds__(LOOKUP_THREADS)
    embedding_lookup_kernel(const T* __restrict__ weight, const void* __restrict__ ids, bool ids64, T* __restrict__ out, long long tokens,
                            long long V, int H, float scale, int* status) {
  const long long t0 = (long long)blockIdx.x * LOOKUP_ROWS;
  long long id[LOOKUP_ROWS];
  bool live[LOOKUP_ROWS], good[LOOKUP_ROWS];
#pragma unroll
  for (int k = 0; k < LOOKUP_ROWS; ++k) {
    live[k] = t0 + k < tokens;
    id[k] = live[k] ? load_id(ids, ids64, t0 + k) : 0;
    good[k] = live[k] && id[k] >= 0 && id[k] < V;
    if (live[k] && !good[k] && threadIdx.x == 0 && blockIdx.y == 0 && status != nullptr) atomicCAS(status, 0, kStatusBadTokenId);
  }
  const int c = (blockIdx.y * LOOKUP_THREADS + threadIdx.x) * N;
  if (c >= H) return;
  Pack<T, N> v[LOOKUP_ROWS];
#pragma unroll
  for (int k = 0; k < LOOKUP_ROWS; ++k) {
    if (good[k]) {
      v[k] = load_pack<T, N>(weight + id[k] * H + c);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) set_element<T, N>(v[k], e, 0.f);
    }
  }
#pragma unroll
  for (int k = 0; k < LOOKUP_ROWS; ++k) {
    if (!live[k]) break;
    if (scale != 1.f) {
#pragma unroll
      for (int e = 0; e < N; ++e) set_element<T, N>(v[k], e, element<T, N>(v[k], e) * scale);
    }
    *reinterpret_cast<Pack<T, N>*>(out + (t0 + k) * H + c) = v[k];
  }
}

// ------------------------------------------------------------------------- zeros
// A share of the zero fill of a new gradient, carried by the blocks of a kernel behind those that do its own work: sorting is a chain of
// latencies on few SMs, filling is all bandwidth, and together they take the longer of the two (32768 x 4096 of 128256:
// 141 us of fill and 27 of sorting become 148).
struct Fill {
  uint4* p;
  long long n;  // 16-byte words
  int tail;     // bytes behind them
};
constexpr int FILL_WORDS = 8;  // per thread

__device__ __forceinline__ void fill_zero(const Fill& f, long long block) {
  if (block == 0 && threadIdx.x < f.tail) reinterpret_cast<unsigned char*>(f.p + f.n)[threadIdx.x] = 0;
  const long long base = block * (FILL_WORDS * blockDim.x) + threadIdx.x;
#pragma unroll
  for (int k = 0; k < FILL_WORDS; ++k) {
    const long long i = base + k * blockDim.x;
    if (i < f.n) f.p[i] = make_uint4(0, 0, 0, 0);
  }
}

// ------------------------------------------------------------------------- sort
// Each thread owns one pair of a compare-exchange step. Steps of distance <= 32 stay inside of the 64 keys of a warp.
__global__ void __launch_bounds__(RUN / 2)
    sort_runs_kernel(const void* __restrict__ ids, bool ids64, uint64_t* __restrict__ keys, long long T, long long V, int runs, Fill fill) {
  __shared__ uint64_t s[RUN];
  if (blockIdx.x >= runs) {
    fill_zero(fill, blockIdx.x - runs);
    return;
  }
  const long long base = (long long)blockIdx.x * RUN;
  const int size = 2 * blockDim.x;  // a power of two above 64
  for (int i = threadIdx.x; i < size; i += blockDim.x) {
    const long long t = base + i;
    uint64_t key = kNoKey;
    if (t < T) {
      const long long id = load_id(ids, ids64, t);
      key = (uint64_t)(id >= 0 && id < V ? (uint32_t)id : kNoId) << 32 | (uint32_t)t;
    }
    s[i] = key;
  }
  __syncthreads();
  for (int k = 2; k <= size; k <<= 1) {
    for (int j = k >> 1; j > 0; j >>= 1) {
      const int low = threadIdx.x & (j - 1);
      const int i = 2 * (threadIdx.x - low) + low;
      const uint64_t a = s[i], b = s[i + j];
      const bool up = (i & k) == 0;
      if ((a > b) == up) {
        s[i] = b;
        s[i + j] = a;
      }
      // the next step's distance is j / 2, or k when this was the last of its stage
      const int next = j > 1 ? j >> 1 : k;
      if (j > 32 || next > 32) __syncthreads();
      else __syncwarp();
    }
  }
  for (int i = threadIdx.x; i < size; i += blockDim.x)
    if (base + i < T) keys[base + i] = s[i];
}

// One level: groups of FAN sorted runs of `length` keys (a power of two; the last run may be short) become one sorted run each.
__global__ void __launch_bounds__(128) merge_runs_kernel(const uint64_t* __restrict__ in, uint64_t* __restrict__ out, int T,
    int log_length, int blocks, Fill fill) {
  if (blockIdx.x >= blocks) {
    fill_zero(fill, blockIdx.x - blocks);
    return;
  }
  const int i = blockIdx.x * 128 + threadIdx.x;
  if (i >= T) return;
  const uint64_t key = in[i];
  const int first = (i >> log_length) / FAN * FAN;          // first run of the group
  const int begin = first << log_length;
  int pos[FAN], end[FAN];                                  // pos: keys before it, in its run, are smaller
#pragma unroll
  for (int r = 0; r < FAN; ++r) {
    const long long b = ((long long)(first + r)) << log_length;
    pos[r] = (int)min((long long)T, b);
    end[r] = (int)min((long long)T, b + (1LL << log_length));
  }
  int place = begin;
#pragma unroll
  for (int r = 0; r < FAN; ++r) place -= pos[r];
  for (int step = 1 << log_length; step > 0; step >>= 1) {
#pragma unroll
    for (int r = 0; r < FAN; ++r)
      if (step <= end[r] - pos[r] && in[pos[r] + step - 1] < key) pos[r] += step;
  }
#pragma unroll
  for (int r = 0; r < FAN; ++r) place += pos[r];
  out[place] = key;
}

// ------------------------------------------------------------------------- sums
// Type of a chunk's sums.
template <typename T>
struct Sum {
  using type = float;
};
template <>
struct Sum<float> {
  using type = double;
};

template <typename D, int N, bool ACC, typename A>
__device__ __forceinline__ void write_row(D* dst, const A* acc, float scale) {
  if constexpr (ACC) {
    constexpr int W = N >= 4 ? 4 : 1;
    float* d = reinterpret_cast<float*>(dst);
#pragma unroll
    for (int e = 0; e < N; e += W) {
      Pack<float, W> v = load_pack<float, W>(d + e);
#pragma unroll
      for (int k = 0; k < W; ++k) set_element<float, W>(v, k, (float)(element<float, W>(v, k) + acc[e + k] * scale));
      *reinterpret_cast<Pack<float, W>*>(d + e) = v;
    }
  } else {
    Pack<D, N> v;
#pragma unroll
    for (int e = 0; e < N; ++e) set_element<D, N>(v, e, (float)(acc[e] * scale));
    *reinterpret_cast<Pack<D, N>*>(dst) = v;
  }
}

// D: type of a dweight row (float when accumulating)
template <typename T, typename D, int N, bool ACC>
__global__ void __launch_bounds__(SUM_THREADS)
    sum_tokens_kernel(const T* __restrict__ dout, const uint64_t* __restrict__ keys, D* __restrict__ dweight, float* __restrict__ partials,
                      long long tokens, int chunk_tokens, int H, float scale) {
  __shared__ uint32_t ids[MAX_CHUNK + 2], rows[MAX_CHUNK];
  const long long chunk = blockIdx.x, base = chunk * chunk_tokens;
  for (int k = threadIdx.x; k < chunk_tokens + 2; k += SUM_THREADS) {
    const long long i = base + k - 1;
    const uint64_t key = i >= 0 && i < tokens ? keys[i] : kNoKey;  // kNoKey's id is no key's
    ids[k] = key_id(key);
    // places without a token read row 0, so that a batch of loads has no condition in it and stays in flight together
    if (k > 0 && k <= chunk_tokens) rows[k - 1] = key == kNoKey ? 0u : (uint32_t)key;
  }
  __syncthreads();
  const int c = (blockIdx.y * SUM_THREADS + threadIdx.x) * N;
  if (c >= H) return;
  const int count = (int)min((long long)chunk_tokens, tokens - base);
  typename Sum<T>::type acc[N];
#pragma unroll
  for (int e = 0; e < N; ++e) acc[e] = 0;
  bool from_before = ids[0] == ids[1];
  constexpr int UNROLL = 8;  // divides every chunk size
  for (int i0 = 0; i0 < count; i0 += UNROLL) {
    Pack<T, N> v[UNROLL];
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) v[k] = load_pack<T, N>(dout + (long long)rows[i0 + k] * H + c);
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) {
      const int i = i0 + k;
      const uint32_t id = ids[1 + i];
      if (i >= count || id == kNoId) break;
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] += element<T, N>(v[k], e);
      const bool ends = ids[2 + i] != id;
      if (ends || i == count - 1) {
        if (ends && !from_before) {
          write_row<D, N, ACC>(dweight + (long long)id * H + c, acc, scale);
        } else {
          // slot 0: the part of a run that began in an earlier chunk, slot 1: the head of a run that goes on
          float* p = partials + (2 * chunk + (from_before ? 0 : 1)) * H + c;
#pragma unroll
          for (int e = 0; e < N; ++e) p[e] = (float)acc[e];
        }
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] = 0;
        from_before = false;
      }
    }
  }
}

// Joins the partial sums of runs that cross chunk borders: the block of the chunk in which the run begins adds its head and the
// parts of the following chunks. Four threads share a column's parts, every fourth one each, and their sums are added in order.
constexpr int JOIN_LANES = 4;
constexpr int JOIN_COLUMNS = 64;
constexpr int JOIN_THREADS = JOIN_LANES * JOIN_COLUMNS;

template <typename D, int N, bool ACC>
__global__ void __launch_bounds__(JOIN_THREADS)
    join_runs_kernel(const uint64_t* __restrict__ keys, D* __restrict__ dweight, const float* __restrict__ partials, int tokens,
        int chunk_tokens, int H, float scale) {
  __shared__ double s[JOIN_LANES][N][JOIN_COLUMNS];
  const int chunks = (tokens + chunk_tokens - 1) / chunk_tokens, chunk = blockIdx.x;
  const int first = chunk * chunk_tokens, next = first + chunk_tokens;  // next < tokens: the last chunk has no block
  const uint32_t id = key_id(keys[next - 1]), after = key_id(keys[next]), here = key_id(keys[first]),
      before = first > 0 ? key_id(keys[first - 1]) : ~0u;
  if (id == kNoId || after != id) return;          // no run crosses this border
  if (here == id && before == id) return;          // it began in an earlier chunk
  // chunks behind this one that the run fills to their last token, and one more in which it ends
  int parts = 0;
  for (;;) {
    const long long c = (long long)chunk + 1 + parts + threadIdx.x;
    const long long last = (c + 1) * chunk_tokens - 1;
    const bool through = c < chunks && last + 1 < tokens && key_id(keys[last]) == id && key_id(keys[last + 1]) == id;
    // runs are contiguous: the threads that see it pass through are the first ones
    const int n = __syncthreads_count(through);
    parts += n;
    if (n < JOIN_THREADS) break;
  }
  ++parts;
  const int column = threadIdx.x % JOIN_COLUMNS, lane = threadIdx.x / JOIN_COLUMNS;
  const int c = (blockIdx.y * JOIN_COLUMNS + column) * N;
  double acc[N];
#pragma unroll
  for (int e = 0; e < N; ++e) acc[e] = 0;
  if (c < H) {
    if (lane == 0) {
      const Pack<float, N> v = load_pack<float, N>(partials + (2LL * chunk + 1) * H + c);
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] = element<float, N>(v, e);
    }
    constexpr int BATCH = 8;
    for (int k0 = lane; k0 < parts; k0 += BATCH * JOIN_LANES) {
      Pack<float, N> v[BATCH];
#pragma unroll
      for (int b = 0; b < BATCH; ++b) {
        const int k = min(k0 + b * JOIN_LANES, parts - 1);
        v[b] = load_pack<float, N>(partials + 2LL * (chunk + 1 + k) * H + c);
      }
#pragma unroll
      for (int b = 0; b < BATCH; ++b) {
        if (k0 + b * JOIN_LANES >= parts) break;
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] += element<float, N>(v[b], e);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < N; ++e) s[lane][e][column] = acc[e];
  __syncthreads();
  if (lane == 0 && c < H) {
#pragma unroll
    for (int l = 1; l < JOIN_LANES; ++l)
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] += s[l][e][column];
    write_row<D, N, ACC>(dweight + (long long)id * H + c, acc, scale);
  }
}

template <typename T>
bool wide_rows(int H, const void* a, const void* b) {
  return (long long)H * sizeof(T) % 16 == 0 && reinterpret_cast<uintptr_t>(a) % 16 == 0 && reinterpret_cast<uintptr_t>(b) % 16 == 0;
}

template <typename T>
void lookup(const void* weight, const void* ids, bool ids64, void* out, long long tokens, long long V, int H, float scale, int* status,
    cudaStream_t stream) {
  constexpr int N = 16 / sizeof(T);
  const bool wide = wide_rows<T>(H, weight, out);
  const int per_block = LOOKUP_THREADS * (wide ? N : 1);
  const dim3 grid((unsigned)((tokens + LOOKUP_ROWS - 1) / LOOKUP_ROWS), (unsigned)((H + per_block - 1) / per_block));
  if (wide)
    embedding_lookup_kernel<T, N><<<grid, LOOKUP_THREADS, 0, stream>>>(reinterpret_cast<const T*>(weight), ids, ids64,
        reinterpret_cast<T*>(out), tokens, V, H, scale, status);
  else
    embedding_lookup_kernel<T, 1><<<grid, LOOKUP_THREADS, 0, stream>>>(reinterpret_cast<const T*>(weight), ids, ids64,
        reinterpret_cast<T*>(out), tokens, V, H, scale, status);
}

// Tokens of one chunk: as many as leave about four blocks per SM, at most 128 (fewer and longer chunks mean fewer partial sums; with
// fewer blocks the chains of loads of a chunk are not covered). A rule on the sizes and the type alone, not on the addresses that decide how
// wide the loads are, so that the order of additions does not depend on them either.
template <typename E>
int chunk_tokens(long long T, int H) {
  constexpr int columns = SUM_THREADS * 16 / (int)sizeof(E);
  const long long slabs = (H + columns - 1) / columns;
  int n = 8;
  while (n < MAX_CHUNK && (T + 2 * n - 1) / (2 * n) * slabs >= 592) n *= 2;
  return n;
}

template <typename T, typename D, int N, bool ACC>
void sums(const void* dout, const uint64_t* keys, void* dweight, float* partials, long long tokens, int H, float scale,
    cudaStream_t stream) {
  const int columns = SUM_THREADS * N, n = chunk_tokens<T>(tokens, H);
  const long long chunks = (tokens + n - 1) / n;
  const dim3 grid((unsigned)chunks, (unsigned)((H + columns - 1) / columns));
  sum_tokens_kernel<T, D, N, ACC><<<grid, SUM_THREADS, 0, stream>>>(reinterpret_cast<const T*>(dout), keys,
      reinterpret_cast<D*>(dweight), partials, tokens, n, H, scale);
  count_launch();
  check_cuda(cudaGetLastError(), "embedding gradient sum launch");
  if (chunks > 1) {
    constexpr int J = N == 1 ? 1 : 4;  // partial sums are fp32: 16 bytes are four columns
    const dim3 join((unsigned)(chunks - 1), (unsigned)((H + J * JOIN_COLUMNS - 1) / (J * JOIN_COLUMNS)));
    join_runs_kernel<D, J, ACC><<<join, JOIN_THREADS, 0, stream>>>(keys, reinterpret_cast<D*>(dweight), partials, (int)tokens, n, H, scale);
    count_launch();
    check_cuda(cudaGetLastError(), "embedding gradient join launch");
  }
}

template <typename T>
void gradient(const void* dout, const uint64_t* keys, void* dweight, bool accumulate, float* partials, long long tokens, int H,
    float scale, cudaStream_t stream) {
  constexpr int N = 16 / sizeof(T);
  const bool wide = wide_rows<T>(H, dout, dweight);
  if (accumulate) {
    if (wide) sums<T, float, N, true>(dout, keys, dweight, partials, tokens, H, scale, stream);
    else sums<T, float, 1, true>(dout, keys, dweight, partials, tokens, H, scale, stream);
  } else {
    if (wide) sums<T, T, N, false>(dout, keys, dweight, partials, tokens, H, scale, stream);
    else sums<T, T, 1, false>(dout, keys, dweight, partials, tokens, H, scale, stream);
  }
}

long long key_bytes(long long T) { return (T * 8 + 255) / 256 * 256; }

}  // namespace

void embedding_lookup(const void* weight, Scalar type, const void* ids, bool ids64, void* out, long long T, long long V, int H,
                      float scale, int* status, cudaStream_t stream) {
  if (T == 0 || H == 0) return;
  auto launch = type == Scalar::kBf16 ? lookup<__nv_bfloat16> : type == Scalar::kF16 ? lookup<__half> : lookup<float>;
  launch(weight, ids, ids64, out, T, V, H, scale, status, stream);
  count_launch();
  check_cuda(cudaGetLastError(), "embedding lookup launch");
}

long long embedding_gradient_workspace(long long T, int H, Scalar type) {
  const int n = type == Scalar::kF32 ? chunk_tokens<float>(T, H) : chunk_tokens<__nv_bfloat16>(T, H);
  const long long chunks = (T + n - 1) / n;
  return 2 * key_bytes(T) + (chunks > 1 ? 2 * chunks * H * 4 : 0);
}

void embedding_gradient(const void* dout, Scalar type, const void* ids, bool ids64, void* dweight, bool accumulate, void* workspace,
                        long long T, long long V, int H, float scale, cudaStream_t stream) {
  if (H == 0 || (T == 0 && (accumulate || V == 0))) return;  // nothing to add and nothing to clear
  uint64_t* keys = reinterpret_cast<uint64_t*>(workspace);
  uint64_t* other = reinterpret_cast<uint64_t*>(reinterpret_cast<char*>(workspace) + key_bytes(T));
  float* partials = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + 2 * key_bytes(T));
  // two keys each; not fewer than 128, for the blocks that fill
  const int threads = T <= RUN / 4 ? RUN / 8 : T <= RUN / 2 ? RUN / 4 : RUN / 2;
  int kernels = 1;
  for (int log_length = LOG_RUN; (1LL << log_length) < T; log_length += LOG_FAN) ++kernels;
  // every kernel of the sort carries the same share of the zeros of a new gradient
  const long long size = type == Scalar::kF32 ? 4 : 2, bytes = accumulate ? 0 : V * H * size, words = bytes / 16;
  auto share = [&](int k) {
    const long long begin = words * k / kernels, end = words * (k + 1) / kernels;
    return Fill{reinterpret_cast<uint4*>(dweight) + begin, end - begin, k + 1 == kernels ? (int)(bytes % 16) : 0};
  };
  auto fill_blocks = [](const Fill& f, int block) {
    const int words = FILL_WORDS * block;
    return (unsigned)((f.n + words - 1) / words + (f.n == 0 && f.tail > 0 ? 1 : 0));
  };
  const unsigned runs = (unsigned)((T + RUN - 1) / RUN), blocks = (unsigned)((T + 127) / 128);
  Fill fill = share(0);
  sort_runs_kernel<<<runs + fill_blocks(fill, threads), threads, 0, stream>>>(ids, ids64, keys, T, V, (int)runs, fill);
  count_launch();
  check_cuda(cudaGetLastError(), "embedding gradient sort launch");
  int k = 1;
  for (int log_length = LOG_RUN; (1LL << log_length) < T; log_length += LOG_FAN, ++k) {
    fill = share(k);
    merge_runs_kernel<<<blocks + fill_blocks(fill, 128), 128, 0, stream>>>(keys, other, (int)T, log_length, (int)blocks, fill);
    count_launch();
    check_cuda(cudaGetLastError(), "embedding gradient merge launch");
    uint64_t* t = keys;
    keys = other;
    other = t;
  }
  auto launch = type == Scalar::kBf16 ? gradient<__nv_bfloat16> : type == Scalar::kF16 ? gradient<__half> : gradient<float>;
  if (T > 0) launch(dout, keys, dweight, accumulate, partials, T, H, scale, stream);
}

}  // namespace b200
