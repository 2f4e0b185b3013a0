// tcgen05 building blocks of products of two microscaled 4-bit operands: block-scaled MMA, scales into tensor memory,
// tensor-map loads.
#pragma once

#include "fp4.cuh"
#include "umma_common.cuh"

namespace rb200 {
namespace f4 {

constexpr int kStageK = 256;  // k of a pipeline stage: a 128-byte row of codes
constexpr int kMmaK = 64;     // k of one MMA

// 512-byte scale tiles a stage has for 128 rows
__host__ __device__ constexpr int stage_tiles(int fmt) { return kStageK / block_of(fmt) / 4; }

#ifdef __CUDACC__

// Instruction descriptor of the block-scaled kinds: e2m1 operands, both K-major; n columns, m rows.
// Bits: [4,6) which half of the word B's scales start in, [7,10) and [10,13) operand types, [17,23) n / 8, 23 scale type
// (1: powers of two), [24,29) m / 16, [29,31) as [4,6) for A.
template <int FMT>
__device__ __forceinline__ uint32_t mma_desc(int m, int n) {
  return (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((FMT == kMx ? 1u : 0u) << 23) | ((uint32_t)(m >> 4) << 24);
}
// kMx: an MMA's 64 k are two blocks, so every other MMA starts in the upper half of its scale words.
__device__ __forceinline__ uint32_t upper_half(uint32_t idesc) { return idesc | (2u << 4) | (2u << 29); }

template <int FMT>
__device__ __forceinline__ void mma_scaled(uint32_t d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t a_scales,
                                           uint32_t b_scales, uint32_t accumulate) {
  if (FMT == kMx)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(a_scales), "r"(b_scales), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(a_scales), "r"(b_scales), "r"(accumulate)
        : "memory");
}

// A 512-byte scale tile from shared memory into four columns of tensor memory, repeated in the four groups of 32 lanes.
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// its descriptor: no swizzle, 8 rows x 16 bytes after one another
__device__ __forceinline__ uint64_t scale_desc(uint32_t smem_addr) {
  return (uint64_t)((smem_addr & 0x3FFFFu) >> 4) | ((uint64_t)1 << 16) | ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
}

__device__ __forceinline__ void tma_load(void* smem_dst, const CUtensorMap* map, int c0, int c1, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          smem_u32(smem_dst)),
      "l"(map), "r"(c0), "r"(c1), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tma_prefetch(const CUtensorMap* map, int c0, int c1) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(map), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void tma_prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t at_rank(uint32_t addr, int rank) {  // a shared-memory address in another CTA of the cluster
  uint32_t to;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(addr), "r"(rank));
  return to;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_cluster(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

#endif  // __CUDACC__

}  // namespace f4
}  // namespace rb200
