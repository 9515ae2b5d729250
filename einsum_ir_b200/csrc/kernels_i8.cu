// The 8-bit contraction's smaller kernels: a contraction over nothing (k = 0), and the copy that
// lays rows out for the tensor cores.
#include "eir_launch.h"
#include "i8_common.cuh"
#include "row_vec.cuh"

namespace eir {

// k = 0: every sum is 0, and the epilogue alone is left; an output a thread at a time
__global__ void __launch_bounds__(256) i8_bias_kernel(const I8Params p, const I8Ptrs a) {
  pdl_launch_dependents();
  pdl_wait();
  const bool gated = p.act == EIR_ACT_GATED_SILU;
  const int64_t n_out = gated ? p.n / 2 : p.n, step = (int64_t)gridDim.x * 256;
  const float low = p.act == EIR_ACT_RELU ? 0.f : -INFINITY;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < p.m * n_out; i += step) {
    const int64_t t = i / n_out, c = i - t * n_out;
    const float sa = a.scale_l ? a.scale_l[t] : 1.f;
    auto z = [&](int64_t ch) { return i8_scaled(0, sa, a.scale_r ? a.scale_r[ch] : 1.f, a.bias ? a.bias[ch] : 0.f); };
    st_any(a.out, p.dt_out, t * p.s_out + c, gated ? silu(z(c)) * z(c + n_out) : relu_from(z(c), low));
  }
}

cudaError_t launch_i8_bias(I8Params const &p, I8Ptrs const &a, int num_sms, cudaStream_t st) {
  const int64_t n_out = p.act == EIR_ACT_GATED_SILU ? p.n / 2 : p.n;
  const int64_t blocks = (p.m * n_out + 255) / 256, most = (int64_t)num_sms * 8;
  return launch_kernel(i8_bias_kernel, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, st, p, a);
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
