// Device helpers shared by the row operators and the 8-bit contraction.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include "eir_cuda.h"
#include "eir_operators.h"

namespace eir {

// below this row maximum (2^-100) 127 / m nears the end of the FP32 range: the
// row counts as zeros
constexpr float kQuantMin = 7.888609052210118e-31f;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// one value of a tensor whose type is a run-time choice
__device__ __forceinline__ float ld_any(void const *p, int dt, int64_t i) {
  return dt == EIR_FP32 ? static_cast<float const *>(p)[i]
                        : __bfloat162float(static_cast<__nv_bfloat16 const *>(p)[i]);
}
__device__ __forceinline__ void st_any(void *p, int dt, int64_t i, float v) {
  if (dt == EIR_FP32) static_cast<float *>(p)[i] = v;
  else static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// a word of another block's shared memory (a shared::cluster address)
__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr_cluster) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr_cluster) : "memory");
  return v;
}

// packed FP32 arithmetic: two roundings of one instruction
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "mul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z, u;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 u, x, y, z;\n\tmov.b64 {%0, %1}, u;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}

// the larger, NaN if either is. Magnitudes as bits keep their order, NaNs above
// infinity, so that an integer maximum carries a NaN through
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// A row's 8-bit scaling from the bits of its largest magnitude: the factor
// 127 / m of round(v * factor), which 127 bounds, and the scale m * unit / 127 of
// the integers. A row with an infinity or NaN is all zeros, and its scale says so.
struct QuantScale {
  float inv, scale;
  bool finite;
};
__device__ __forceinline__ QuantScale quant_scale(uint32_t max_bits, float unit) {
  QuantScale q;
  const float m = __uint_as_float(max_bits);
  q.finite = max_bits < 0x7f800000u;
  const bool some = q.finite && m >= kQuantMin;
  q.inv = some ? __fdiv_rn(127.f, m) : 0.f;
  q.scale = q.finite ? (some ? __fdiv_rn(__fmul_rn(m, unit), 127.f) : 0.f) : __uint_as_float(0x7fc00000u);
  return q;
}
}  // namespace eir
