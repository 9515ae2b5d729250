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
__device__ __forceinline__ float silu(float z) { return z / (1.f + expf(-z)); }
// ReLU that keeps a NaN; `low` = 0, or -infinity for no activation
__device__ __forceinline__ float relu_from(float z, float low) { return z < low ? low : z; }

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

// The channel side of the epilogue, held by the thread that owns the channel:
// its scale and bias (gated: the gate's and the value's)
struct I8Channel {
  float sb, bias, sb2, bias2;
};
__device__ __forceinline__ I8Channel i8_channel(I8Params const &p, I8Ptrs const &a, int64_t c, int64_t n_out,
                                                bool gated) {
  I8Channel h{1.f, 0.f, 1.f, 0.f};
  if (c >= n_out) return h;
  if (a.scale_r) h.sb = a.scale_r[c];
  if (a.bias) h.bias = a.bias[c];
  if (gated) {
    if (a.scale_r) h.sb2 = a.scale_r[c + n_out];
    if (a.bias) h.bias2 = a.bias[c + n_out];
  }
  return h;
}
// one output value from its accumulator(s)
template <bool GATED>
__device__ __forceinline__ float i8_value(int32_t acc, int32_t acc2, float sa, I8Channel const &h, float low) {
  const float z = i8_scaled(acc, sa, h.sb, h.bias);
  if (GATED) return silu(z) * i8_scaled(acc2, sa, h.sb2, h.bias2);
  return relu_from(z, low);
}

}  // namespace eir
