// Output projection fused with the softmax that follows it: logits = x [M, K] W [N, K]^T are formed on CTA pairs in 256 x 256
// tiles (tcgen05 cta_group::2) and are reduced, or turned into their gradient, on the way out of tensor memory.
//
//   statistics: the epilogue reduces each row of a tile to (m, s, u, x[label]): largest logit, sums of softmax_stats.cuh
//               relative to it, and the label's logit if it lies in the tile's columns; 16 bytes per row and tile go to
//               stats[slice][row] for every 128 columns instead of 256 bytes of logits. token_log_probs_join combines them.
//   statistics, logits kept: the same, and the fp32 logits leave through shared memory and bulk tensor stores, for a backward
//               pass that has the memory for them: 2.1 GB of stores hide under 2.7 ms of MMAs (4096 x 4096 x 128256), and what
//               the gradient mode would take, 2.7 ms, becomes a pass over memory (0.42 ms).
//   gradient:   the logits are formed again, and the epilogue writes d(logits) in bf16, the operand type of the two products
//               that follow (d(x) = d(logits) W, dW = d(logits)^T x); the factor 1[label] - p is formed in fp32 from the fp32
//               logits, so the one rounding is that of the stored operand.
//
// Same staging and synchronisation as the pair GEMM of gemm_bf16_2sm.cu (six 32 KB stages per CTA filled by TMA without
// multicast, one issuing thread in the even CTA, two accumulators of 256 TMEM columns so that the epilogue of one tile runs
// under the MMAs of the next). An epilogue thread owns one row of 128 columns, so the statistics need no exchange between
// threads. Eight epilogue warps, two per quarter of the tensor memory's lanes, each with half of the columns: with four, one per
// scheduler and each instruction waiting for the one before, the epilogue of a tile with entropy took about 20000 cycles and
// bounded the kernel up to K = 2048 (16384 cycles of MMAs a tile).
//
// The tensor cores' fp32 accumulator is truncated at every step of 16 products, an error that grows with K and always points the same way.
// So K is taken in parts of 1024: the epilogue threads add the parts up in registers, 128 columns a thread, rounding to nearest, while
// the tensor cores work on the next part (about 700 cycles against 8192). Log-probabilities at K = 4096 against 64 bits, relative:
// 1.5e-6 in one part, 3.5e-7 in parts of 1024 (at every larger K), 1.8e-7 in parts of 512. 4096 x 4096 x 128256 takes the same time either way;
// 777 x 2048 x 49152, whose last epilogue is not covered, 145 us in one part, 153 in parts of 1024, 158 in parts of 512.
//
// Rows whose label does not count are left out of all products: the batch is compacted to its live rows beforehand, whose number only
// the device knows (LiveRows), so the kernel takes its row count from memory and the grid is sized for the whole batch.
#include <cuda.h>

#include "../common/cta_pair.cuh"
#include "../common/launch.h"
#include "../common/ptx.cuh"
#include "../common/tensor_map.h"
#include "../ops/softmax_stats.cuh"
#include "../ops/vocabulary.h"

namespace b200 {

namespace {

constexpr int BM = 128;       // rows per CTA (256 per pair)
constexpr int BN = 256;       // columns per pair
constexpr int SLICES = BN / kVocabSlice;
constexpr int BN_HALF = 128;  // W rows staged per CTA
constexpr int BK = 64;
constexpr int PART = 16;      // k-blocks whose products stay in the tensor cores' accumulator
constexpr int STAGES = 6;
constexpr int A_STAGE_BYTES = BM * BK * 2;
constexpr int B_STAGE_BYTES = BN_HALF * BK * 2;
constexpr int EPI_WARPS = 8;
constexpr int THREADS = 64 + 32 * EPI_WARPS;
constexpr int TMEM_COLS = 512;
constexpr int BOX_BYTES = 32 * 128;               // one epilogue box: 32 rows x 64 bf16
constexpr int STAGING_BYTES = EPI_WARPS * BOX_BYTES;
constexpr int SMEM_BYTES = STAGES * (A_STAGE_BYTES + B_STAGE_BYTES) + STAGING_BYTES + 1024 + 256;

struct RowArgs {
  const void* labels;
  bool labels64;
  float4* stats;  // statistics: [slices][live.rows]
  LiveRows live;
  const float2* lse;
  const float* entropy;
  const float* d_log_probs;
  long long d_log_probs_stride;
  const float* d_entropy;
  long long d_entropy_stride;
  float logit_scale;
  long long ignore_index;
};

// 16 columns of this warp's 32 lanes (with 32 at a time the accumulators of a thread no longer fit its registers).
__device__ __forceinline__ void tmem_load_16(uint32_t (&v)[16], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
        "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(addr)
      : "memory");
}

enum class Mode : int { kStats, kStatsKeep, kGrad };

// x[i] of 32 registers for a lane's own i: halved five times, so that the array stays in registers.
__device__ __forceinline__ float select32(const float (&x)[32], int i) {
  float t[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) t[k] = (i & 16) ? x[k + 16] : x[k];
#pragma unroll
  for (int k = 0; k < 8; ++k) t[k] = (i & 8) ? t[k + 8] : t[k];
#pragma unroll
  for (int k = 0; k < 4; ++k) t[k] = (i & 4) ? t[k + 4] : t[k];
#pragma unroll
  for (int k = 0; k < 2; ++k) t[k] = (i & 2) ? t[k + 2] : t[k];
  return (i & 1) ? t[1] : t[0];
}

template <Mode MODE, bool ENTROPY>
__global__ void __launch_bounds__(THREADS, 1)
    vocab_gemm_2sm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmA1,
        const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmOut, int N, int K, RowBoxes box, int* status,
        RowArgs rows) {
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
  const int num_pairs = gridDim.x >> 1;
  // rows of this launch that count; at least one tile is worked on, so that a batch without any leaves zeros behind
  const int live = rows.live.count == nullptr ? rows.live.rows : max(0, min(rows.live.rows, *rows.live.count - rows.live.base));
  const int m_tiles = max(1, (live + 2 * BM - 1) / (2 * BM));
  const int n_tiles = (N + BN - 1) / BN;
  const int k_blocks = (K + BK - 1) / BK;
  const int total = m_tiles * n_tiles;
  // Row panels of up to eight tiles: the pairs that run at a time share their A rows within a panel column and their W rows
  // across the panel (the raster of the plain pair GEMM).
  const int group = min(m_tiles, 8);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 2 * EPI_WARPS);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  clear_rows(sA, STAGES, A_STAGE_BYTES, cta_rank == 0 ? box.rows0 : box.rows1);
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
      for (int tile = pair; tile < total && ok; tile += num_pairs) {
        const TileCoord tc = tile_coord(tile, m_tiles, n_tiles, group);
        const int m0 = tc.mi * (2 * BM) + (int)cta_rank * BM;
        const int n0 = tc.ni * BN + (int)cta_rank * BN_HALF;
        for (int kb = 0; kb < k_blocks; ++kb, ++it) {
          const uint32_t s = it % STAGES;
          const uint32_t ph = (it / STAGES) & 1;
          if (!mbar_wait(&empty[s], ph ^ 1, abort_flag)) {
            raise_status(status, kStatusWaitTimeoutProducer, abort_flag);
            ok = false;
            break;
          }
          const uint32_t full_leader = map_to_cta(smem_u32(&full[s]), 0);
          if (leader) mbar_arrive_expect_tx(&full[s], (box.rows0 + box.rows1) * (BK * 2) + 2 * B_STAGE_BYTES);
          if (leader) tma_load_2d_pair(sA + s * A_STAGE_BYTES, &tmA, full_leader, kb * BK, m0);
          else if (box.rows1 > 0) tma_load_2d_pair(sA + s * A_STAGE_BYTES, &tmA1, full_leader, kb * BK, m0);
          tma_load_2d_pair(sB + s * B_STAGE_BYTES, &tmB, full_leader, kb * BK, n0);
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
      constexpr uint32_t idesc = umma_idesc_bf16(2 * BM, BN, 0, 0);
      uint32_t it = 0, tcount = 0;
      bool ok = true;
      for (int tile = pair; tile < total && ok; tile += num_pairs) {
        for (int part = 0; part < k_blocks && ok; part += PART, ++tcount) {
          const uint32_t buf = tcount & 1;
          const uint32_t aph = (tcount >> 1) & 1;
          if (!mbar_wait(&acc_empty[buf], aph ^ 1, abort_flag)) {
            raise_status(status, kStatusWaitTimeoutMma, abort_flag);
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t d_tmem = tmem_base + buf * BN;
          const int part_end = min(k_blocks, part + PART);
          for (int kb = part; kb < part_end; ++kb, ++it) {
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
              umma_f16_ss_2sm(d_tmem, umma_smem_desc_sw128(a_base + k * 32, 16, 1024), umma_smem_desc_sw128(b_base + k * 32, 16, 1024),
                              idesc, (kb != part || k != 0) ? 1u : 0u);
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
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ epilogue: 32 rows x 128 columns of this CTA's 128 x 256 half
    const int q = warp & 3;             // the quarter of the lanes that this warp can read
    const int half = (warp - 2) >> 2;   // its half of the columns
    uint8_t* store_box = sStage + (warp - 2) * BOX_BYTES;
    const float scale2 = rows.logit_scale * kLog2e;
    uint32_t tcount = 0;
    bool ok = true;
    for (int tile = pair; tile < total && ok; tile += num_pairs) {
      const TileCoord tc = tile_coord(tile, m_tiles, n_tiles, group);
      const int row0 = tc.mi * (2 * BM) + (int)cta_rank * BM + q * 32;
      const int row = row0 + lane;
      const int slice_col0 = tc.ni * BN + half * kVocabSlice;
      // the label's column relative to the slice; -1: not here
      int label = -1;
      bool ignored = true;
      int t = 0;  // the row's place in the batch
      if (row < live) {
        t = rows.live.index != nullptr ? rows.live.index[rows.live.base + row] : rows.live.base + row;
        const long long l = load_label(rows.labels, rows.labels64, t);
        ignored = l == rows.ignore_index || l < 0 || l >= N;
        if (!ignored && l >= slice_col0 && l < slice_col0 + kVocabSlice) label = (int)(l - slice_col0);
      }
      float2 L = make_float2(0.f, 0.f);
      float gs = 0.f, hs = 0.f, H = 0.f;
      bool zero = true;
      if (MODE == Mode::kGrad && !ignored) {
        L = rows.lse[t];
        gs = rows.d_log_probs[(long long)t * rows.d_log_probs_stride] * rows.logit_scale;
        if (ENTROPY) {
          hs = rows.d_entropy[(long long)t * rows.d_entropy_stride] * rows.logit_scale;
          H = rows.entropy[t];
        }
        zero = gs == 0.f && hs == 0.f;
      }
      // the parts of K, added up
      float acc[kVocabSlice];
#pragma unroll
      for (int e = 0; e < kVocabSlice; ++e) acc[e] = 0.f;
#pragma unroll 1
      for (int part = 0; part < k_blocks; part += PART, ++tcount) {
        const uint32_t buf = tcount & 1;
        const uint32_t aph = (tcount >> 1) & 1;
        if (!mbar_wait(&acc_full[buf], aph, abort_flag)) {
          raise_status(status, kStatusWaitTimeoutEpilogue, abort_flag);
          ok = false;
          break;
        }
        tc_fence_after_sync();
        const uint32_t t_row = tmem_base + (uint32_t(q * 32) << 16) + buf * BN + half * kVocabSlice;
#pragma unroll
        for (int c = 0; c < kVocabSlice / 16; ++c) {
          uint32_t v[16];
          tmem_load_16(v, t_row + c * 16);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[c * 16 + e] += __uint_as_float(v[e]);
        }
        // hand the TMEM buffer back
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(map_to_cta(smem_u32(&acc_empty[buf]), 0));
      }
      if (!ok || slice_col0 >= N) continue;  // nothing of the vocabulary here

      if (MODE != Mode::kGrad) {
        Stats st = empty_stats();
        float x_label = 0.f;
#pragma unroll
        for (int c = 0; c < kVocabSlice / 32; ++c) {
          const int col0 = slice_col0 + c * 32;
          if (col0 >= N) break;
          float(&x)[32] = *reinterpret_cast<float(*)[32]>(acc + c * 32);
          if (MODE == Mode::kStatsKeep) {
            if (lane == 0) tma_store_wait_read<0>();  // the store that used the box before has read it
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 8; ++j)
              box_write(store_box, lane, j, make_uint4(__float_as_uint(x[4 * j]), __float_as_uint(x[4 * j + 1]),
                  __float_as_uint(x[4 * j + 2]), __float_as_uint(x[4 * j + 3])));
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0 && row0 < live) {
              tma_store_2d(&tmOut, store_box, col0, row0);
              tma_store_commit();
            }
          }
          if (col0 + 32 > N) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (col0 + e >= N) x[e] = -INFINITY;
          }
          if ((label >> 5) == c) x_label = select32(x, label & 31);
          float top = x[0];
          F2 f[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            top = fmaxf(top, fmaxf(x[2 * e], x[2 * e + 1]));
            f[e] = pack2(x[2 * e], x[2 * e + 1]);
          }
          accumulate<ENTROPY, 32>(st, f, top, scale2);
        }
        if (row < live) rows.stats[(long long)(tc.ni * SLICES + half) * rows.live.rows + row] = make_float4(st.m, st.s, st.u, x_label);
      } else {
#pragma unroll
        for (int c = 0; c < kVocabSlice / 64; ++c) {
          const int col0 = slice_col0 + c * 64;
          if (col0 >= N) break;
          if (lane == 0) tma_store_wait_read<0>();  // the store that used the box before has read it
          __syncwarp();
#pragma unroll
          for (int part = 0; part < 2; ++part) {
            const float(&x)[32] = *reinterpret_cast<const float(*)[32]>(acc + c * 64 + part * 32);
            uint32_t w[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float a = score_gradient<ENTROPY>(log2_prob(x[2 * e], L, scale2), gs, hs, H);
              const float b = score_gradient<ENTROPY>(log2_prob(x[2 * e + 1], L, scale2), gs, hs, H);
              w[e] = zero ? 0u : pack_bf16x2(a, b);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
              box_write(store_box, lane, part * 4 + j, make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]));
            if ((label >> 5) == 2 * c + part && !zero) {
              // the label's own gradient, over the element of the row just written
              const float d = log2_prob(select32(x, label & 31), L, scale2);
              const int e = label & 63;
              *reinterpret_cast<__nv_bfloat16*>(store_box + lane * 128 + (((e >> 3) ^ (lane & 7)) << 4) + (e & 7) * 2) =
                  __float2bfloat16(gs + score_gradient<ENTROPY>(d, gs, hs, H));
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0 && row0 < rows.live.rows) {
            tma_store_2d(&tmOut, store_box, col0, row0);
            tma_store_commit();
          }
        }
      }
    }
    if (MODE != Mode::kStats) {
      // every bulk store of this warp has left shared memory and reached global memory before the CTA exits
      if (lane == 0) tma_store_wait<0>();
      __syncwarp();
    }
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

template <Mode MODE, bool ENTROPY>
void launch(const void* x, long long ldx, const CUtensorMap& tmB, const CUtensorMap* out, int N, int K, int* status,
    const RowArgs& rows, cudaStream_t stream) {
  auto kernel = vocab_gemm_2sm_kernel<MODE, ENTROPY>;
  check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES), "vocab gemm smem attr");
  const RowBoxes box(rows.live.rows);
  const CUtensorMap tmA = make_tensor_map_2d_b16(x, K, rows.live.rows, ldx, BK, box.rows0);
  const CUtensorMap tmA1 = make_tensor_map_2d_b16(x, K, rows.live.rows, ldx, BK, box.rows1 > 0 ? box.rows1 : box.rows0);
  const CUtensorMap& tmOut = out != nullptr ? *out : tmA;
  const int m_tiles = (rows.live.rows + 2 * BM - 1) / (2 * BM), n_tiles = (N + BN - 1) / BN;
  int pairs = sm_count() / 2;
  if ((long long)m_tiles * n_tiles < pairs) pairs = m_tiles * n_tiles;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * pairs, 1, 1);
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
  check_cuda(cudaLaunchKernelEx(&cfg, kernel, tmA, tmA1, tmB, tmOut, N, K, box, status, rows), "vocab gemm launch");
  count_launch();
}

}  // namespace

void vocab_gemm_stats(const void* x, const void* w, const void* labels, bool labels64, float* stats, float* logits, long long ldl,
    bool entropy, LiveRows live, int N, int K, long long ldx, long long ldw, float logit_scale, int* status, cudaStream_t stream) {
  if (live.rows <= 0) return;
  const CUtensorMap tmB = make_tensor_map_2d_b16(w, K, N, ldw, BK, BN_HALF);
  RowArgs rows = {};
  rows.live = live;
  rows.labels = labels;
  rows.labels64 = labels64;
  rows.stats = reinterpret_cast<float4*>(stats);
  rows.logit_scale = logit_scale;
  rows.ignore_index = -1;  // every label outside of [0, N) counts as none here
  if (logits != nullptr) {
    const CUtensorMap tmL = make_tensor_map_2d_f32(logits, N, live.rows, ldl, 32, 32);
    if (entropy) launch<Mode::kStatsKeep, true>(x, ldx, tmB, &tmL, N, K, status, rows, stream);
    else launch<Mode::kStatsKeep, false>(x, ldx, tmB, &tmL, N, K, status, rows, stream);
  } else if (entropy) {
    launch<Mode::kStats, true>(x, ldx, tmB, nullptr, N, K, status, rows, stream);
  } else {
    launch<Mode::kStats, false>(x, ldx, tmB, nullptr, N, K, status, rows, stream);
  }
}

void vocab_gemm_grad(const void* x, const void* w, const void* labels, bool labels64, const float2* lse, const float* entropy,
                     const float* d_log_probs, long long d_log_probs_stride, const float* d_entropy, long long d_entropy_stride,
                     void* grad, LiveRows live, int N, int K, long long ldx, long long ldw, long long ldg, float logit_scale,
                     long long ignore_index, int* status, cudaStream_t stream) {
  if (live.rows <= 0) return;
  const CUtensorMap tmB = make_tensor_map_2d_b16(w, K, N, ldw, BK, BN_HALF);
  const CUtensorMap tmG = make_tensor_map_2d_b16(grad, N, live.rows, ldg, 64, 32);
  RowArgs rows = {};
  rows.live = live;
  rows.labels = labels;
  rows.labels64 = labels64;
  rows.lse = lse;
  rows.entropy = entropy;
  rows.d_log_probs = d_log_probs;
  rows.d_log_probs_stride = d_log_probs_stride;
  rows.d_entropy = d_entropy;
  rows.d_entropy_stride = d_entropy_stride;
  rows.logit_scale = logit_scale;
  rows.ignore_index = ignore_index;
  if (d_entropy != nullptr) launch<Mode::kGrad, true>(x, ldx, tmB, &tmG, N, K, status, rows, stream);
  else launch<Mode::kGrad, false>(x, ldx, tmB, &tmG, N, K, status, rows, stream);
}

}  // namespace b200
