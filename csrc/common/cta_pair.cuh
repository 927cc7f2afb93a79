// Device primitives of kernels that run on CTA pairs (clusters of two, tcgen05 cta_group::2): cluster barriers and
// remote mbarriers, TMEM and MMA in their two-SM forms, and the raster and epilogue boxes that the pair GEMMs share.
#pragma once

#include <cuda.h>

#include "ptx.cuh"

namespace b200 {

__device__ __forceinline__ uint32_t cluster_ctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// shared::cluster address of `local` in CTA `rank` of this cluster
__device__ __forceinline__ uint32_t map_to_cta(uint32_t local, uint32_t rank) {
  uint32_t out;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(out) : "r"(local), "r"(rank));
  return out;
}

__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

__device__ __forceinline__ void tmem_alloc_2sm(uint32_t* smem_result, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(smem_result)), "r"(ncols) : "memory");
}
__device__ __forceinline__ void tmem_relinquish_2sm() {
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_2sm(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}

// Copy into this CTA's shared memory; completion bytes are credited to the barrier at `bar_cluster_addr`, which may
// belong to the other CTA of the pair.
__device__ __forceinline__ void tma_load_2d_pair(void* smem_dst, const CUtensorMap* desc, uint32_t bar_cluster_addr, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      :
      : "r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(desc)), "r"(bar_cluster_addr), "r"(x), "r"(y)
      : "memory");
}

__device__ __forceinline__ void umma_f16_ss_2sm(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t"
      "}\n"
      :
      : "r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Arrive on the barrier at a shared::cluster address once all MMAs issued so far by this thread have retired.
__device__ __forceinline__ void umma_commit_2sm(uint32_t bar_cluster_addr) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar_cluster_addr) : "memory");
}

struct TileCoord {
  int mi, ni;  // tile indices (256-row, 256-column units)
};

__device__ __forceinline__ TileCoord tile_coord(int tile, int m_tiles, int n_tiles, int group) {
  if (group > 0) {
    const int per_group = group * n_tiles;
    const int g = tile / per_group;
    const int first = g * group;
    const int gsize = min(m_tiles - first, group);
    const int r = tile - g * per_group;
    return {first + r % gsize, r / gsize};
  }
  group = -group;
  const int per_group = group * m_tiles;
  const int g = tile / per_group;
  const int first = g * group;
  const int gsize = min(n_tiles - first, group);
  const int r = tile - g * per_group;
  return {r / gsize, first + r % gsize};
}

// Row `lane` of a swizzled 32 x 128-byte box: 16-byte chunk `c` of the row lands at chunk `c ^ (lane & 7)`.
__device__ __forceinline__ void box_write(uint8_t* box, int lane, int chunk, uint4 v) {
  *reinterpret_cast<uint4*>(box + lane * 128 + ((chunk ^ (lane & 7)) << 4)) = v;
}

// Rows of the K-major A operand that the two CTAs of a pair fetch per k-block. A batch of at most one tile fetches the rows that it has
// (a multiple of eight): rows of a box that lie outside of the matrix are zeros, but they are asked for all the same, all at
// one address, and with a single row the pairs queued up there (scores of 1 x 4096 x 128256: 262 to 300 us, depending on where the
// row lay; 204 with boxes of eight rows).
struct RowBoxes {
  int rows0, rows1;

  explicit RowBoxes(int rows) : rows0(128), rows1(128) {
    if (rows <= 128) {
      rows0 = (rows + 7) / 8 * 8;
      rows1 = 0;
    } else if (rows <= 256) {
      rows1 = (rows - 128 + 7) / 8 * 8;
    }
  }
};

// Zeros in the rows of each stage that no copy fills (whole block; 128 rows of 128 bytes per stage).
__device__ __forceinline__ void clear_rows(uint8_t* stages, int count, int stage_bytes, int filled) {
  const int words = (128 - filled) * 8;
  for (int i = threadIdx.x; i < count * words; i += blockDim.x) {
    const int s = i / words;
    *reinterpret_cast<uint4*>(stages + s * stage_bytes + filled * 128 + (i - s * words) * 16) = make_uint4(0, 0, 0, 0);
  }
  if (words > 0) fence_proxy_async_smem();  // the tensor cores read them through the async proxy
}

}  // namespace b200
