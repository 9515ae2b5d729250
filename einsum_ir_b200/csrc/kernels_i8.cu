// Contraction of 8-bit integers on the CUDA cores, for operands that the
// tensor cores cannot take, and the copy that lays rows out for them.
#include "eir_launch.h"
#include "i8_common.cuh"
#include "row_vec.cuh"

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

// Rows of k bytes of one or two operands into rows `ld` bytes apart (a multiple of 16): TMA
// needs 16-byte strides and a 16-byte base. A warp copies a row at a time: a lane reads the
// two aligned vectors that cover its 16 bytes and shifts them into place (the
// shift is the same for the row); a vector that reaches outside the tensor is
// read byte by byte.
__device__ __forceinline__ uint4 pack_vector(uintptr_t at, uintptr_t begin, uintptr_t end) {
  if (at >= begin && at + 16 <= end) return *reinterpret_cast<uint4 const *>(at);
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    w[j] = 0;
    for (int e = 0; e < 4; ++e) {
      const uintptr_t q = at + 4 * j + e;
      if (q >= begin && q < end) w[j] |= (uint32_t)*reinterpret_cast<uint8_t const *>(q) << (8 * e);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__global__ void __launch_bounds__(256) i8_pack_kernel(const I8Pack one, const I8Pack two, int64_t k, int64_t ld,
                                                      int parts) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t step = (int64_t)gridDim.x * 8;
  for (int64_t unit = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); unit < (one.rows + two.rows) * parts;
       unit += step) {
    const int64_t any = unit / parts;
    const int part = (int)(unit - any * parts);
    const bool second = any >= one.rows;
    const int64_t r = second ? any - one.rows : any, stride = second ? two.stride : one.stride;
    const uintptr_t begin = reinterpret_cast<uintptr_t>(second ? two.src : one.src);
    const uintptr_t end = begin + (uintptr_t)(((second ? two.rows : one.rows) - 1) * stride + k);
    int8_t *dst = second ? two.dst : one.dst;
    const int v0 = (int)(ld / 16 * part / parts), v1 = (int)(ld / 16 * (part + 1) / parts);  // vectors of the row
    const uintptr_t row = begin + (uintptr_t)(r * stride);
    const uint32_t off = (uint32_t)(row & 15);
    const uintptr_t base = row - off;
    int8_t *to = dst + r * ld;
    auto put = [&](int v, uint4 lo, uint4 hi) {
      const uint32_t a[4] = {lo.x, lo.y, lo.z, lo.w}, b[4] = {hi.x, hi.y, hi.z, hi.w};
      uint32_t o[4];
      shifted_words<4>(a, b, off, o);
      *reinterpret_cast<uint4 *>(to + 16 * (int64_t)v) = make_uint4(o[0], o[1], o[2], o[3]);
    };
    int v = v0 + lane;
    if (base + 16 * (uintptr_t)v0 >= begin) {
      // four vectors of a lane at a time, all inside the tensor
      for (; v + 96 < v1 && base + 16 * (uintptr_t)(v0 + (v - v0) / 128 * 128 + 128) + 16 <= end; v += 128) {
        uint4 lo[4], hi[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint4 const *q = reinterpret_cast<uint4 const *>(base + 16 * (uintptr_t)(v + 32 * i));
          lo[i] = __ldg(q);
          hi[i] = __ldg(q + 1);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) put(v + 32 * i, lo[i], hi[i]);
      }
    }
    for (; v < v1; v += 32)
      put(v, pack_vector(base + 16 * (uintptr_t)v, begin, end), pack_vector(base + 16 * (uintptr_t)v + 16, begin, end));
  }
}

cudaError_t launch_i8_pack(I8Pack const &one, I8Pack const &two, int64_t k, int64_t ld, int num_sms, cudaStream_t st) {
  // a row in parts where there are too few rows for the GPU's warps
  const int64_t rows = one.rows + two.rows;
  int parts = 1;
  while (rows * parts < (int64_t)num_sms * 32 && ld / 16 >= 64 * parts) parts *= 2;
  const int64_t blocks = (rows * parts + 7) / 8, most = (int64_t)num_sms * 8;
  return launch_kernel(i8_pack_kernel, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, st, one, two, k,
                       ld, parts);
}

}  // namespace eir
