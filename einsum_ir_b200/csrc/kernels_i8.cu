// Contraction of 8-bit integers on the CUDA cores, for operands that the
// tensor cores cannot take, and the copy that lays rows out for them.
#include "eir_launch.h"
#include "i8_common.cuh"

namespace eir {

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
  const float low = p.act == EIR_ACT_RELU ? 0.f : -INFINITY;
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
      else v = relu_from(v, low);
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

// Rows of k bytes into rows `ld` bytes apart (a multiple of 16): TMA needs
// 16-byte strides and a 16-byte base. A thread writes 16 bytes, read as
// aligned words shifted into place; a word that reaches outside the tensor's
// bytes is read byte by byte.
__global__ void __launch_bounds__(256) i8_pack_kernel(int64_t rows, int64_t k, int64_t stride,
                                                      int8_t const *__restrict__ src, int8_t *__restrict__ dst,
                                                      int64_t ld) {
  pdl_launch_dependents();
  pdl_wait();
  const uintptr_t begin = reinterpret_cast<uintptr_t>(src);
  const uintptr_t end = begin + (uintptr_t)((rows - 1) * stride + k);
  const int64_t per_row = ld / 16, total = rows * per_row;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per_row, b = (i - r * per_row) * 16;
    const uintptr_t at = begin + (uintptr_t)(r * stride + b), base = at & ~(uintptr_t)3;
    uint32_t w[5];
#pragma unroll
    for (int j = 0; j < 5; ++j) {
      const uintptr_t q = base + 4 * j;
      if (q >= begin && q + 4 <= end) {
        w[j] = *reinterpret_cast<uint32_t const *>(q);
      } else {
        w[j] = 0;
        for (int e = 0; e < 4; ++e)
          if (q + e >= begin && q + e < end) w[j] |= (uint32_t) * reinterpret_cast<uint8_t const *>(q + e) << (8 * e);
      }
    }
    const uint32_t sh = 8 * (uint32_t)(at & 3);
    uint4 v;
    v.x = __funnelshift_r(w[0], w[1], sh);
    v.y = __funnelshift_r(w[1], w[2], sh);
    v.z = __funnelshift_r(w[2], w[3], sh);
    v.w = __funnelshift_r(w[3], w[4], sh);
    *reinterpret_cast<uint4 *>(dst + r * ld + b) = v;
  }
}

cudaError_t launch_i8_pack(int64_t rows, int64_t k, int64_t stride, int8_t const *src, int8_t *dst, int64_t ld,
                           int num_sms, cudaStream_t st) {
  const int64_t blocks = (rows * (ld / 16) + 255) / 256, most = (int64_t)num_sms * 8;
  return launch_kernel(i8_pack_kernel, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, st, rows, k,
                       stride, src, dst, ld);
}

}  // namespace eir
