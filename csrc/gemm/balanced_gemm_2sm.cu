// C [M, N] = A [M, K] B [K, N] for few output tiles and a long K: the data gradient of the output projection, where K is the
// vocabulary. bf16 operands (A K-major, B row-major), fp32 accumulation, bf16 result.
//
// A 256 x 256 output tile on a CTA pair takes K / 64 steps, and M N / 65536 tiles seldom divide by the 74 pairs: 14 x 16 tiles take
// four waves where 3.03 would do, 1 x 16 tiles leave 58 pairs idle. So the waves that occupy every pair are worked on tile by tile (the
// pairs walk K together and share their operands in L2), and when at most half of the pairs would have a tile in the last wave, the
// steps of its tiles, tile after tile, are cut into equal ranges, one per pair. A tile that lies in one range is stored as bf16; of a
// tile that is cut, every pair that worked on it leaves an fp32 partial tile (at most two per pair: the tile its range begins in and the
// one it ends in), and balanced_rows adds them in the order of the pairs, so the result does not depend on the order of execution.
// The number of rows may be known on the device only (LiveRows): the cut is computed there, the same way by both kernels.
//
// A tile's K products stay in the tensor cores' accumulator throughout, unlike those of vocab_gemm_2sm.cu: its truncation is of no account next
// to the result's bf16 (256 x 256 x 128256, all products of one sign, the worst case: 5e-6 of the result too little, a rounding to
// bf16 is up to 3.9e-3).
//
// Staging and synchronisation are those of the pair GEMM of gemm_bf16_2sm.cu. 3584 live rows x 4096 x 128256: 3.23 ms with whole
// tiles, 2.61 ms cut. Bound by the tensor cores and the L2 -> SM traffic of its operands (64 bytes a cycle and SM).
#include <cuda.h>

#include "../common/cta_pair.cuh"
#include "../common/launch.h"
#include "../common/ptx.cuh"
#include "../common/tensor_map.h"
#include "../ops/vocabulary.h"

namespace b200 {

namespace {

constexpr int BM = 128;       // rows per CTA (256 per pair)
constexpr int BN = 256;       // columns per pair
constexpr int BN_HALF = 128;  // B columns staged per CTA
constexpr int BK = 64;
constexpr int STAGES = 6;
constexpr int A_STAGE_BYTES = BM * BK * 2;
constexpr int B_STAGE_BYTES = BN_HALF * BK * 2;
constexpr int THREADS = 192;
constexpr int TMEM_COLS = 512;
constexpr int BOX_BYTES = 32 * 128;
constexpr int STAGING_BYTES = 4 * 2 * BOX_BYTES;
constexpr int SMEM_BYTES = STAGES * (A_STAGE_BYTES + B_STAGE_BYTES) + STAGING_BYTES + 1024 + 256;
constexpr int MIN_STEPS = 8;  // steps that a range has at least: shorter ones cost more in partial tiles than they save

// The division of a product among the pairs: tiles [0, whole) tile by tile, the steps of the others cut into `ranges` ranges.
struct Cut {
  int m_tiles, n_tiles, steps, grid_pairs, whole, ranges;
  long long total;  // steps of the tiles that are cut

  __device__ Cut(int live_rows, int N, int K, int pairs) : grid_pairs(pairs) {
    m_tiles = max(1, (live_rows + 2 * BM - 1) / (2 * BM));
    n_tiles = (N + BN - 1) / BN;
    steps = (K + BK - 1) / BK;
    const int tiles = m_tiles * n_tiles, rest = tiles % pairs;
    const bool cut = 2 * rest <= pairs;
    whole = cut ? tiles - rest : tiles;
    total = cut ? (long long)rest * steps : 0;
    ranges = (int)min((long long)pairs, max(1LL, total / MIN_STEPS));
  }
  __device__ long long begin(int range) const { return range < ranges ? total * range / ranges : total; }
  // the range that holds step u
  __device__ int range_of(long long u) const {
    int p = (int)(u * ranges / total);
    while (p + 1 < ranges && begin(p + 1) <= u) ++p;
    while (p > 0 && begin(p) > u) --p;
    return p;
  }
};

// What one pair works on, in order. Every role of both CTAs walks the same list.
struct Walk {
  const Cut& cut;
  int pair, next_tile;
  long long u, first, last;
  // the present item
  int tile, kb0, kb1, slot;
  bool complete;  // the tile is computed whole

  __device__ Walk(const Cut& c, int p) : cut(c), pair(p), next_tile(p), u(c.begin(p)), first(c.begin(p)), last(c.begin(p + 1)), tile(0),
      kb0(0), kb1(0), slot(0), complete(true) {}
  __device__ bool next() {
    if (next_tile < cut.whole) {
      tile = next_tile;
      next_tile += cut.grid_pairs;
      kb0 = 0;
      kb1 = cut.steps;
      complete = true;
      return true;
    }
    if (u >= last) return false;
    const int t = (int)(u / cut.steps);
    kb0 = (int)(u - (long long)t * cut.steps);
    kb1 = (int)min((long long)cut.steps, kb0 + (last - u));
    tile = cut.whole + t;
    slot = 2 * pair + (u == first ? 0 : 1);
    complete = kb0 == 0 && kb1 == cut.steps;
    u += kb1 - kb0;
    return true;
  }
};

__device__ __forceinline__ int live_count(const LiveRows& live) {
  return live.count == nullptr ? live.rows : max(0, min(live.rows, *live.count - live.base));
}

__global__ void __launch_bounds__(THREADS, 1)
    balanced_gemm_2sm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmA1,
        const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmC, const __grid_constant__ CUtensorMap tmP,
        int N, int K, RowBoxes rows, LiveRows live, int* status) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * A_STAGE_BYTES;
  uint8_t* sStage = smem + STAGES * (A_STAGE_BYTES + B_STAGE_BYTES);
  uint64_t* bars = reinterpret_cast<uint64_t*>(sStage + STAGING_BYTES);
  uint64_t* full = bars;
  uint64_t* empty = bars + STAGES;
  uint64_t* acc_full = bars + 2 * STAGES;
  uint64_t* acc_empty = bars + 2 * STAGES + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t cta_rank = cluster_ctarank();  // 0 = leader
  const bool leader = cta_rank == 0;
  const int pair = blockIdx.x >> 1;
  const Cut cut(live_count(live), N, K, gridDim.x >> 1);
  const int group = min(cut.m_tiles, 8);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 8);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  clear_rows(sA, STAGES, A_STAGE_BYTES, cta_rank == 0 ? rows.rows0 : rows.rows1);
  __syncthreads();
  if (warp == 1) {
    tmem_alloc_2sm(tmem_slot, TMEM_COLS);
    tmem_relinquish_2sm();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers are initialised before anything remote touches them
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer (both CTAs)
    if (lane == 0) {
      tma_prefetch_desc(leader ? &tmA : &tmA1);
      tma_prefetch_desc(&tmB);
      uint32_t it = 0;
      bool ok = true;
      Walk walk(cut, pair);
      while (ok && walk.next()) {
        const TileCoord tc = tile_coord(walk.tile, cut.m_tiles, cut.n_tiles, group);
        const int m0 = tc.mi * (2 * BM) + (int)cta_rank * BM;
        const int n0 = tc.ni * BN + (int)cta_rank * BN_HALF;
        for (int kb = walk.kb0; kb < walk.kb1; ++kb, ++it) {
          const uint32_t s = it % STAGES;
          const uint32_t ph = (it / STAGES) & 1;
          if (!mbar_wait(&empty[s], ph ^ 1, abort_flag)) {
            raise_status(status, kStatusWaitTimeoutProducer, abort_flag);
            ok = false;
            break;
          }
          const uint32_t full_leader = map_to_cta(smem_u32(&full[s]), 0);
          if (leader) mbar_arrive_expect_tx(&full[s], (rows.rows0 + rows.rows1) * (BK * 2) + 2 * B_STAGE_BYTES);
          uint8_t* b_dst = sB + s * B_STAGE_BYTES;
          if (leader) tma_load_2d_pair(sA + s * A_STAGE_BYTES, &tmA, full_leader, kb * BK, m0);
          else if (rows.rows1 > 0) tma_load_2d_pair(sA + s * A_STAGE_BYTES, &tmA1, full_leader, kb * BK, m0);
#pragma unroll
          for (int j = 0; j < BN_HALF / 64; ++j) tma_load_2d_pair(b_dst + j * (BK * 128), &tmB, full_leader, n0 + j * 64, kb * BK);
        }
      }
      if (!ok) {
        for (int i = 0; i < 64; ++i) __nanosleep(1000);  // copies in flight land before the CTA may exit
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer (leader CTA only)
    if (leader && lane == 0) {
      constexpr uint32_t idesc = umma_idesc_bf16(2 * BM, BN, 0, 1);
      uint32_t it = 0, tcount = 0;
      bool ok = true;
      Walk walk(cut, pair);
      for (; ok && walk.next(); ++tcount) {
        const uint32_t buf = tcount & 1;
        const uint32_t aph = (tcount >> 1) & 1;
        if (!mbar_wait(&acc_empty[buf], aph ^ 1, abort_flag)) {
          raise_status(status, kStatusWaitTimeoutMma, abort_flag);
          break;
        }
        tc_fence_after_sync();
        const uint32_t d_tmem = tmem_base + buf * BN;
        for (int kb = walk.kb0; kb < walk.kb1; ++kb, ++it) {
          const uint32_t s = it % STAGES;
          const uint32_t ph = (it / STAGES) & 1;
          if (!mbar_wait(&full[s], ph, abort_flag)) {
            raise_status(status, kStatusWaitTimeoutMma, abort_flag);
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t a_base = smem_u32(sA + s * A_STAGE_BYTES);
          const uint32_t b_base = smem_u32(sB + s * B_STAGE_BYTES);
#pragma unroll
          for (int k = 0; k < BK / 16; ++k) {
            umma_f16_ss_2sm(d_tmem, umma_smem_desc_sw128(a_base + k * 32, 16, 1024),
                umma_smem_desc_sw128(b_base + k * 16 * 128, BK * 128, 1024), idesc, (kb != walk.kb0 || k != 0) ? 1u : 0u);
          }
          const uint32_t e_local = smem_u32(&empty[s]);  // release the stage in both CTAs
          umma_commit_2sm(map_to_cta(e_local, 0));
          umma_commit_2sm(map_to_cta(e_local, 1));
        }
        if (ok) {
          const uint32_t f_local = smem_u32(&acc_full[buf]);
          umma_commit_2sm(map_to_cta(f_local, 0));
          umma_commit_2sm(map_to_cta(f_local, 1));
        }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ epilogue: this CTA's 128 x 256 half
    const int q = warp & 3;
    uint8_t* stage0 = sStage + q * (2 * BOX_BYTES);
    uint32_t tcount = 0, nstore = 0;
    Walk walk(cut, pair);
    for (; walk.next(); ++tcount) {
      const bool whole = walk.complete;
      const TileCoord tc = tile_coord(walk.tile, cut.m_tiles, cut.n_tiles, group);
      const uint32_t buf = tcount & 1;
      const uint32_t aph = (tcount >> 1) & 1;
      if (!mbar_wait(&acc_full[buf], aph, abort_flag)) {
        raise_status(status, kStatusWaitTimeoutEpilogue, abort_flag);
        break;
      }
      tc_fence_after_sync();
      const int tile_row0 = (int)cta_rank * BM + q * 32;
      const int row0 = tc.mi * (2 * BM) + tile_row0;
      const uint32_t t_row = tmem_base + (uint32_t(q * 32) << 16) + buf * BN;
      const int columns = min(BN, N - tc.ni * BN);
      const int boxes = whole ? (columns + 63) / 64 : (columns + 31) / 32;
#pragma unroll 1
      for (int c = 0; c < boxes; ++c, ++nstore) {
        uint8_t* box = stage0 + (nstore & 1) * BOX_BYTES;
        if (lane == 0) tma_store_wait_read<1>();  // the store that used this box two boxes ago has read it
        __syncwarp();
        if (whole) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint32_t v[32];
            B200_TMEM_LD_32(v, t_row + c * 64 + half * 32);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              box_write(box, lane, half * 4 + j, make_uint4(pack_bf16x2(__uint_as_float(v[8 * j]), __uint_as_float(v[8 * j + 1])),
                  pack_bf16x2(__uint_as_float(v[8 * j + 2]), __uint_as_float(v[8 * j + 3])),
                  pack_bf16x2(__uint_as_float(v[8 * j + 4]), __uint_as_float(v[8 * j + 5])),
                  pack_bf16x2(__uint_as_float(v[8 * j + 6]), __uint_as_float(v[8 * j + 7]))));
            }
          }
        } else {
          uint32_t v[32];
          B200_TMEM_LD_32(v, t_row + c * 32);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 8; ++j) box_write(box, lane, j, make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]));
        }
        if (c == boxes - 1) {
          // last read of this accumulator: hand the TMEM buffer back before the stores drain
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(map_to_cta(smem_u32(&acc_empty[buf]), 0));
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0 && row0 < live.rows) {
          if (whole) tma_store_2d(&tmC, box, tc.ni * BN + c * 64, row0);
          else tma_store_2d(&tmP, box, c * 32, walk.slot * (2 * BM) + tile_row0);
          tma_store_commit();
        }
      }
    }
    // every bulk store of this warp has left shared memory and reached global memory before the CTA exits
    if (lane == 0) tma_store_wait<0>();
    __syncwarp();
  }

  // Neither CTA may free its TMEM or exit while the other can still reach into it.
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_2sm(tmem_base, TMEM_COLS);
  }
}

// The product's live rows at their places in the batch: out[t] (bf16, N columns, a multiple of 8) is the row of C where the tile was
// computed whole, and the sum of its partial tiles in the order of the pairs where it was cut. One block per row and 1024 columns.
__global__ void __launch_bounds__(128)
    balanced_rows_kernel(const __nv_bfloat16* __restrict__ C, const float* __restrict__ partials, LiveRows live,
        __nv_bfloat16* __restrict__ out, int N, int K, int pairs) {
  const int r = blockIdx.x, rows = live_count(live);
  if (r >= rows) return;
  const long long t = live.index != nullptr ? live.index[live.base + r] : live.base + r;
  const Cut cut(rows, N, K, pairs);
  const int group = min(cut.m_tiles, 8);
  const int mi = r / (2 * BM), row = r % (2 * BM);
  const int panel = mi / group, panel_rows = min(cut.m_tiles - panel * group, group);
  const int c = (blockIdx.y * 128 + threadIdx.x) * 8;
  if (c < N) {
    const int ni = c / BN, col = c % BN;
    const int tile = panel * group * cut.n_tiles + ni * panel_rows + (mi - panel * group);  // inverse of tile_coord
    uint4 v;
    int p0 = 0, p1 = 0;
    const long long begin = (long long)(tile - cut.whole) * cut.steps;
    if (tile >= cut.whole) {
      p0 = cut.range_of(begin);
      p1 = cut.range_of(begin + cut.steps - 1);
    }
    if (p0 == p1) {
      v = *reinterpret_cast<const uint4*>(C + (long long)r * N + c);
    } else {
      float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
      for (int p = p0; p <= p1; ++p) {
        const int slot = 2 * p + (cut.begin(p) >= begin ? 0 : 1);  // the tile its range begins in, or the one it ends in
        const float4* q = reinterpret_cast<const float4*>(partials + ((long long)slot * (2 * BM) + row) * BN + col);
        const float4 a = q[0], b = q[1];
        f[0] += a.x; f[1] += a.y; f[2] += a.z; f[3] += a.w;
        f[4] += b.x; f[5] += b.y; f[6] += b.z; f[7] += b.w;
      }
      v = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
    }
    *reinterpret_cast<uint4*>(out + t * N + c) = v;
  }
}

int grid_pairs() { return sm_count() / 2; }

}  // namespace

long long balanced_partials() { return 2LL * grid_pairs() * (2 * BM) * BN; }

void balanced_gemm(const void* A, const void* B, void* C, float* partials, LiveRows live, int N, int K, long long lda, long long ldb,
    int* status, cudaStream_t stream) {
  if (live.rows <= 0) return;
  const RowBoxes rows(live.rows);
  const CUtensorMap tmA = make_tensor_map_2d_b16(A, K, live.rows, lda, BK, rows.rows0);
  const CUtensorMap tmA1 = make_tensor_map_2d_b16(A, K, live.rows, lda, BK, rows.rows1 > 0 ? rows.rows1 : rows.rows0);
  const CUtensorMap tmB = make_tensor_map_2d_b16(B, N, K, ldb, 64, BK);
  const CUtensorMap tmC = make_tensor_map_2d_b16(C, N, live.rows, N, 64, 32);
  const CUtensorMap tmP = make_tensor_map_2d_f32(partials, BN, 2LL * grid_pairs() * (2 * BM), BN, 32, 32);
  check_cuda(cudaFuncSetAttribute(balanced_gemm_2sm_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES),
      "balanced gemm smem attr");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * grid_pairs(), 1, 1);
  cfg.blockDim = dim3(THREADS, 1, 1);
  cfg.dynamicSmemBytes = SMEM_BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  check_cuda(cudaLaunchKernelEx(&cfg, balanced_gemm_2sm_kernel, tmA, tmA1, tmB, tmC, tmP, N, K, rows, live, status),
      "balanced gemm launch");
  count_launch();
}

void balanced_rows(const void* C, const float* partials, LiveRows live, void* out, int N, int K, cudaStream_t stream) {
  if (live.rows <= 0) return;
  const dim3 grid((unsigned)live.rows, (unsigned)((N + 1023) / 1024));
  balanced_rows_kernel<<<grid, 128, 0, stream>>>(reinterpret_cast<const __nv_bfloat16*>(C), partials, live,
      reinterpret_cast<__nv_bfloat16*>(out), N, K, grid_pairs());
  count_launch();
  check_cuda(cudaGetLastError(), "balanced rows launch");
}

}  // namespace b200
