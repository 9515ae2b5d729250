// Pieces shared by the 8-bit contraction kernels: the scaled epilogue, and the
// 2-D TMA loads and integer tensor-core instructions of the tcgen05 kernels.
#pragma once

#include "eir_common.cuh"
#include "op_common.cuh"
#include "op_params.h"

namespace eir {

// z = acc sa sb + bias in FP32 (the integer rounds to 24 bits, then one rounding each)
__device__ __forceinline__ float i8_scaled(int32_t acc, float sa, float sb, float bias) {
  return fmaf((float)acc, sa * sb, bias);
}
// two of them in packed FP32 arithmetic (the same roundings)
__device__ __forceinline__ float2 scaled2(int32_t a0, int32_t a1, float2 sa, float sb, float bias) {
  return fma2(make_float2((float)a0, (float)a1), mul2(sa, make_float2(sb, sb)), make_float2(bias, bias));
}
// silu(z) = z / (1 + e^-z) with the hardware's exponential and reciprocal: off
// by about (|z| + 4) 2^-24 of itself, under the rounding of the sum that gave z
__device__ __forceinline__ float silu(float z) { return __fdividef(z, 1.f + __expf(-z)); }
// ReLU that keeps a NaN; `low` = 0, or -infinity for no activation
__device__ __forceinline__ float relu_from(float z, float low) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(z), "f"(low));
  return r;
}

// 2-D tiled TMA load global -> shared, completion on an mbarrier (no multicast)
__device__ __forceinline__ void tma_load_2d(void *dst, void const *map, uint64_t *bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1)
      : "memory");
}
// the same with the completion counted on an mbarrier of either CTA of the pair
__device__ __forceinline__ void tma_load_2d_pair(void *dst, void const *map, uint32_t bar_cluster, int c0,
                                                 int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(bar_cluster), "r"(c0), "r"(c1)
      : "memory");
}

__device__ __forceinline__ void tma_load_3d(void *dst, void const *map, uint64_t *bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair(void *dst, void const *map, uint32_t bar_cluster, int c0, int c1,
                                                 int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(bar_cluster), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

// the same boxes into L2 only. L2 is where all of the GPU's writes meet, so what a kernel that
// still runs writes afterwards is what a later load reads
__device__ __forceinline__ void tma_prefetch_2d(void const *map, int c0, int c1) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];" ::"l"(map), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void tma_prefetch_3d(void const *map, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global [%0, {%1, %2, %3}];" ::"l"(map), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}

// arrive on an mbarrier of any CTA of the cluster without ordering earlier memory accesses
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t bar_cluster) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar_cluster) : "memory");
}

// instruction descriptor of kind::i8: signed 8-bit operands, both K-major, 32-bit integer accumulate
__host__ __device__ constexpr uint32_t i8_idesc(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

__device__ __forceinline__ void umma_i8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_i8_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 32 lanes x 16 columns of 32-bit TMEM -> 16 registers per thread (row = lane)
__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
        "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
        "=r"(v[14]), "=r"(v[15])
      : "r"(taddr));
}

}  // namespace eir
