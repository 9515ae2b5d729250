// Contraction of 8-bit integers for a single token on the CUDA cores.
//
// A token needs each weight byte once, so the kernel is bound by the weights'
// bytes (HBM) and, for small layers, by latency: a warp streams two channels
// (gated: two gates and their values) with aligned 16-byte loads, eight in
// flight a lane, and the token's row comes from L1. Byte dot products (dp4a)
// accumulate in 32-bit integers, which one warp reduction adds exactly. There is no
// ring, barrier or TMEM to set up, which is what it saves over the tensor-core
// kernel (4096 x 4096: 4.0 against 6.1 us a call); from two tokens on the
// byte products cost more than that.
//
// Rows off the 16-byte grid: rows 16 apart lie alike on it, whatever the
// stride, so a warp takes channels c and c + 16, reads the aligned chunks
// that cover them, and shifts the token's row instead, once for both (zeros
// before and after it cancel the neighbouring rows' bytes).
#include <algorithm>
#include "eir_launch.h"
#include "i8_common.cuh"

namespace eir {

constexpr int kRowWarps = 8;

// the row bytes k .. k + 15 of the token, zeros outside 0 .. k_end - 1
template <bool ALIGNED>
__device__ __forceinline__ uint4 i8_token_chunk(int8_t const *row, int64_t k, int64_t k_end) {
  if (ALIGNED ? k + 16 <= k_end : (k >= 16 && k + 32 <= k_end)) {  // the aligned words are inside the row
    const uintptr_t at = reinterpret_cast<uintptr_t>(row + k);
    if (ALIGNED) return __ldg(reinterpret_cast<uint4 const *>(at));
    uint4 const *base = reinterpret_cast<uint4 const *>(at & ~(uintptr_t)15);
    const uint4 lo = __ldg(base), hi = __ldg(base + 1);
    const uint32_t sh = 8 * (uint32_t)(at & 3);
    auto pick = [&](uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t e) {
      return make_uint4(__funnelshift_r(a, b, sh), __funnelshift_r(b, c, sh), __funnelshift_r(c, d, sh),
                        __funnelshift_r(d, e, sh));
    };
    switch ((at >> 2) & 3) {  // the same for every chunk
      case 0: return pick(lo.x, lo.y, lo.z, lo.w, hi.x);
      case 1: return pick(lo.y, lo.z, lo.w, hi.x, hi.y);
      case 2: return pick(lo.z, lo.w, hi.x, hi.y, hi.z);
      default: return pick(lo.w, hi.x, hi.y, hi.z, hi.w);
    }
  }
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = 0;
    for (int e = 0; e < 4; ++e) {
      const int64_t q = k + 4 * i + e;
      if (q >= 0 && q < k_end) w[i] |= (uint32_t)(uint8_t)row[q] << (8 * e);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// an aligned chunk of the weights; the bytes outside the tensor are not read
__device__ __forceinline__ uint4 i8_weight_chunk(uintptr_t at, uintptr_t begin, uintptr_t end) {
  if (at >= begin && at + 16 <= end) return __ldg(reinterpret_cast<uint4 const *>(at));
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = 0;
    for (int e = 0; e < 4; ++e) {
      const uintptr_t q = at + 4 * i + e;
      if (q >= begin && q < end) w[i] |= (uint32_t)*reinterpret_cast<uint8_t const *>(q) << (8 * e);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ int32_t dot16(uint4 a, uint4 b, int32_t c) {
  c = __dp4a((int)a.x, (int)b.x, c);
  c = __dp4a((int)a.y, (int)b.y, c);
  c = __dp4a((int)a.z, (int)b.z, c);
  return __dp4a((int)a.w, (int)b.w, c);
}

// `per`: warps that share a warp's channels (each takes every per-th piece of K)
template <bool GATED, bool ALIGNED, typename T>
__global__ void __launch_bounds__(32 * kRowWarps) i8_row_kernel(const I8Params p, const I8Ptrs a, int per) {
  constexpr int H = GATED ? 2 : 1, U = GATED ? 2 : 4;  // halves; K pieces in flight (8 weight loads a lane)
  __shared__ int32_t part[kRowWarps][2 * H];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t n_out = GATED ? p.n / 2 : p.n;
  const int64_t unit = (int64_t)blockIdx.x * (kRowWarps / per) + warp / per;
  // the warp's channels: neighbours, or 16 apart where the rows' places on the grid have to agree
  constexpr int kApart = ALIGNED ? 1 : 16;
  const int64_t c0 = unit / kApart * (2 * kApart) + unit % kApart, c1 = c0 + kApart;
  pdl_launch_dependents();
  pdl_wait();
  int32_t acc[2 * H] = {};  // [half][channel]
  if (c0 < n_out) {
    const uintptr_t begin = reinterpret_cast<uintptr_t>(a.r);
    const uintptr_t end = begin + (uintptr_t)((p.n - 1) * p.s_r + p.k);
    uintptr_t at[2 * H];  // the aligned chunks that hold the rows' first bytes
    int off[H];           // bytes of the neighbour's row before them
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const uintptr_t r0 = begin + (uintptr_t)((c0 + h * n_out) * p.s_r);
      off[h] = ALIGNED ? 0 : (int)(r0 & 15);
      at[2 * h] = r0 - off[h];
      // a missing second channel repeats the first, and is not stored
      at[2 * h + 1] = c1 < n_out ? at[2 * h] + (uintptr_t)(kApart * p.s_r) : at[2 * h];
    }
    const int64_t step = 512 * per, k_end = p.k + (ALIGNED ? 0 : 15);
    int64_t k = (warp % per) * 512 + lane * 16;
    auto token = [&](int h, int64_t q) { return i8_token_chunk<ALIGNED>(a.l, q - off[h], p.k); };
    // whole chunks inside the tensor (the first row may start before it)
    for (; at[0] >= begin && k + (U - 1) * step + 32 <= p.k; k += U * step) {
      uint4 w[2 * H * U];
#pragma unroll
      for (int i = 0; i < U; ++i)
#pragma unroll
        for (int r = 0; r < 2 * H; ++r)
          w[2 * H * i + r] = __ldg(reinterpret_cast<uint4 const *>(at[r] + (k + i * step)));
#pragma unroll
      for (int i = 0; i < U; ++i)
#pragma unroll
        for (int h = 0; h < H; ++h) {
          const uint4 x = token(h, k + i * step);
          acc[2 * h] = dot16(w[2 * H * i + 2 * h], x, acc[2 * h]);
          acc[2 * h + 1] = dot16(w[2 * H * i + 2 * h + 1], x, acc[2 * h + 1]);
        }
    }
    for (; k < k_end; k += step) {
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const uint4 x = token(h, k);
        acc[2 * h] = dot16(i8_weight_chunk(at[2 * h] + k, begin, end), x, acc[2 * h]);
        acc[2 * h + 1] = dot16(i8_weight_chunk(at[2 * h + 1] + k, begin, end), x, acc[2 * h + 1]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 2 * H; ++i) acc[i] = __reduce_add_sync(0xffffffffu, acc[i]);
  if (per > 1) {
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < 2 * H; ++i) part[warp][i] = acc[i];
    }
    __syncthreads();
    if (warp % per != 0) return;
#pragma unroll
    for (int i = 0; i < 2 * H; ++i)
      for (int j = 1; j < per; ++j) acc[i] += part[warp + j][i];
  }
  // lanes 0 and 1: the two channels
  const int64_t c = lane == 0 ? c0 : c1;
  if (lane > 1 || c >= n_out) return;
  const float sa = a.scale_l ? a.scale_l[0] : 1.f;
  float z[H];
#pragma unroll
  for (int h = 0; h < H; ++h) {
    const int64_t r = c + h * n_out;
    z[h] = i8_scaled(lane == 0 ? acc[2 * h] : acc[2 * h + 1], sa, a.scale_r ? a.scale_r[r] : 1.f,
                     a.bias ? a.bias[r] : 0.f);
  }
  const float v = GATED ? silu(z[0]) * z[H - 1] : relu_from(z[0], p.act == EIR_ACT_RELU ? 0.f : -INFINITY);
  static_cast<T *>(a.out)[c] = from_f32<T>(v);
}

template <bool GATED, bool ALIGNED>
static cudaError_t launch_row(I8Params const &p, I8Ptrs const &a, int num_sms, cudaStream_t st) {
  const int64_t n_out = GATED ? p.n / 2 : p.n, units = ALIGNED ? (n_out + 1) / 2 : (n_out + 31) / 32 * 16;
  // several warps a pair of channels until 16 warps an SM are at work
  int per = 1;
  while (per < kRowWarps && units * per < (int64_t)num_sms * 16 && p.k > 512 * per) per *= 2;
  const int64_t blocks = (units * per + kRowWarps - 1) / kRowWarps;
  auto kern = p.dt_out == EIR_BF16 ? i8_row_kernel<GATED, ALIGNED, __nv_bfloat16> : i8_row_kernel<GATED, ALIGNED, float>;
  return launch_kernel(kern, dim3((unsigned)blocks), dim3(32 * kRowWarps), 0, st, p, a, per);
}

cudaError_t launch_i8_row(I8Params const &p, I8Ptrs const &a, int num_sms, cudaStream_t st) {
  // with an aligned base and stride every chunk but a row's last lies inside the row
  const bool aligned = ((reinterpret_cast<uintptr_t>(a.l) | reinterpret_cast<uintptr_t>(a.r)) & 15) == 0 && p.s_r % 16 == 0;
  if (p.act == EIR_ACT_GATED_SILU)
    return aligned ? launch_row<true, true>(p, a, num_sms, st) : launch_row<true, false>(p, a, num_sms, st);
  return aligned ? launch_row<false, true>(p, a, num_sms, st) : launch_row<false, false>(p, a, num_sms, st);
}

}  // namespace eir
