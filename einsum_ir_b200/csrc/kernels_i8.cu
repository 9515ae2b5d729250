// Contraction of 8-bit integers with a scale for each token (left row) and
// channel (right row): acc = sum_k a b in 32-bit integers (exact, so any
// order of the sum gives the same bits), then in FP32
// z = acc sa sb + bias and the activation, rounded once when stored.
#include "eir_launch.h"
#include "eir_common.cuh"
#include "op_common.cuh"
#include "op_params.h"

namespace eir {

__device__ __forceinline__ float i8_scaled(int32_t acc, float sa, float sb, float bias) {
  return fmaf((float)acc, sa * sb, bias);
}
__device__ __forceinline__ float silu(float z) { return z / (1.f + expf(-z)); }

// 64 tokens x 64 channels (gated: 32 gates and their 32 values) a CTA, K
// staged in shared memory byte by byte in blocks of 64, so that any stride
// and alignment will do; 4-way byte dot products (dp4a).
constexpr int kI8Tile = 64, kI8Block = 64, kI8Pitch = kI8Block / 4 + 1;

__global__ void __launch_bounds__(256) i8_simt_kernel(const I8Params p, const I8Ptrs a) {
  __shared__ uint32_t sl[kI8Tile * kI8Pitch], sr[kI8Tile * kI8Pitch];
  pdl_launch_dependents();
  pdl_wait();
  const bool gated = p.act == EIR_ACT_GATED_SILU;
  const int64_t n_out = gated ? p.n / 2 : p.n;
  const int per = gated ? kI8Tile / 2 : kI8Tile;  // output channels of a CTA
  const uint32_t c_tiles = (uint32_t)((n_out + per - 1) / per);
  const int64_t t0 = (int64_t)(blockIdx.x / c_tiles) * kI8Tile, c0 = (int64_t)(blockIdx.x % c_tiles) * per;
  // the tile's right row j: channel c0 + j, or for the values of a gated tile its value channel
  auto channel = [&](int j) { return j < per ? c0 + j : c0 + (j - per) + n_out; };
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  int32_t acc[4][4] = {};
  for (int64_t k0 = 0; k0 < p.k; k0 += kI8Block) {
    __syncthreads();
    for (int i = threadIdx.x; i < kI8Tile * kI8Block; i += 256) {
      const int j = i / kI8Block, b = i % kI8Block;
      const int64_t k = k0 + b, t = t0 + j, c = channel(j);
      const bool own = j < per ? c < n_out : c < p.n;
      reinterpret_cast<int8_t *>(sl + j * kI8Pitch)[b] = (k < p.k && t < p.m) ? a.l[t * p.s_l + k] : 0;
      reinterpret_cast<int8_t *>(sr + j * kI8Pitch)[b] = (k < p.k && own) ? a.r[c * p.s_r + k] : 0;
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < kI8Block / 4; ++kk) {
      uint32_t l[4], r[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        l[i] = sl[(ty + 16 * i) * kI8Pitch + kk];
        r[i] = sr[(tx + 16 * i) * kI8Pitch + kk];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a((int)l[i], (int)r[j], acc[i][j]);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t t = t0 + ty + 16 * i;
    if (t >= p.m) continue;
    const float sa = a.scale_l ? a.scale_l[t] : 1.f;
    auto z = [&](int j) {  // tile column tx + 16 j
      const int64_t c = channel(tx + 16 * j);
      return i8_scaled(acc[i][j], sa, a.scale_r ? a.scale_r[c] : 1.f, a.bias ? a.bias[c] : 0.f);
    };
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t c = c0 + tx + 16 * j;
      if (gated && j >= 2) break;
      if (c >= n_out) continue;
      float v = z(j);
      if (gated) v = silu(v) * z(j + 2 < 4 ? j + 2 : 3);
      else if (p.act == EIR_ACT_RELU) v = v > 0.f ? v : (v != v ? v : 0.f);
      st_any(a.out, p.dt_out, t * p.s_out + c, v);
    }
  }
}

cudaError_t launch_i8_simt(I8Params const &p, I8Ptrs const &a, cudaStream_t st) {
  const bool gated = p.act == EIR_ACT_GATED_SILU;
  const int64_t n_out = gated ? p.n / 2 : p.n, per = gated ? kI8Tile / 2 : kI8Tile;
  const int64_t tiles = ((n_out + per - 1) / per) * ((p.m + kI8Tile - 1) / kI8Tile);
  if (tiles > INT32_MAX) return cudaErrorInvalidConfiguration;
  const dim3 grid((unsigned)tiles);
  return launch_kernel(i8_simt_kernel, grid, dim3(256), 0, st, p, a);
}

}  // namespace eir
