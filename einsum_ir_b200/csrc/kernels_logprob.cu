// Log probabilities of given tokens, log-sum-exp, entropy and top alternatives
// of rows of logits, and the gradient of the first and third.
//
// With m = max x, S = sum e^(x - m), U = sum (x - m) e^(x - m):
// lse = m + log S, entropy = log S - U / S (no difference of large numbers:
// U <= 0), log p = (x - m) - log S (exact differences where the logits are
// large and near one another). Backward: dx = dlogprob (onehot - p) - dentropy p (x - lse + H).
#include "eir_launch.h"
#include "eir_common.cuh"
#include "op_common.cuh"
#include "op_params.h"

namespace eir {

constexpr int kLogThreads = 256;

// a logit's rank as an unsigned integer: the order of the floats, both zeros
// alike, NaNs highest
__device__ __forceinline__ uint32_t rank_bits(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
// rank and place in one word: larger logits first, then lower indices
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t index) {
  return ((uint64_t)rank_bits(x) << 32) | (uint32_t)~index;
}

__device__ __forceinline__ float logit_nan() { return __uint_as_float(0x7fc00000u); }

template <typename T>
__global__ void __launch_bounds__(kLogThreads) logprob_kernel(const LogprobParams p, const LogprobPtrs a) {
  __shared__ float red[3][kLogThreads / 32];
  __shared__ uint64_t best[kLogThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    T const *x = static_cast<T const *>(a.x) + row * p.s_x;
    float m = -INFINITY;
    for (int64_t c = threadIdx.x; c < p.vocab; c += kLogThreads) m = fmaxf(m, to_f32(x[c]));
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    __syncthreads();
    if (lane == 0) red[0][warp] = m;
    __syncthreads();
    for (int w = 0; w < kLogThreads / 32; ++w) m = fmaxf(m, red[0][w]);
    const float ref = m == -INFINITY ? 0.f : m;
    float S = 0.f, U = 0.f;
    for (int64_t c = threadIdx.x; c < p.vocab; c += kLogThreads) {
      const float d = to_f32(x[c]) - ref;
      const float e = expf(d);
      S += e;
      U += d == -INFINITY ? 0.f : d * e;
    }
    S = warp_sum(S);
    U = warp_sum(U);
    if (lane == 0) {
      red[1][warp] = S;
      red[2][warp] = U;
    }
    __syncthreads();
    S = U = 0.f;
    for (int w = 0; w < kLogThreads / 32; ++w) {
      S += red[1][w];
      U += red[2][w];
    }
    const bool none = S == 0.f;
    const float log_s = logf(S), lse = none ? -INFINITY : ref + log_s;
    if (threadIdx.x == 0) {
      if (a.lse) a.lse[row] = lse;
      if (a.entropy) a.entropy[row] = none ? 0.f : log_s - U / S;
      if (a.targets) {
        const int64_t t = a.targets[row];
        a.logprob[row] = t < 0 ? 0.f : (t >= p.vocab ? logit_nan() : (none ? -INFINITY : to_f32(x[t]) - ref - log_s));
      }
    }
    uint64_t last = ~0ull;  // every key is below
    for (int i = 0; i < p.top; ++i) {
      uint64_t k = 0;
      for (int64_t c = threadIdx.x; c < p.vocab; c += kLogThreads) {
        const uint64_t key = rank_key(to_f32(x[c]), (uint32_t)c);
        if (key < last || i == 0) k = key > k ? key : k;
      }
      for (int o = 16; o > 0; o >>= 1) {
        const uint64_t other = __shfl_xor_sync(0xffffffffu, k, o);
        k = other > k ? other : k;
      }
      __syncthreads();
      if (lane == 0) best[warp] = k;
      __syncthreads();
      for (int w = 0; w < kLogThreads / 32; ++w) k = best[w] > k ? best[w] : k;
      last = k;
      if (threadIdx.x == 0) {
        const uint32_t at = ~(uint32_t)k;
        if (a.top_index) a.top_index[row * p.top + i] = at;
        if (a.top_logprob) a.top_logprob[row * p.top + i] = none ? -INFINITY : to_f32(x[at]) - ref - log_s;
      }
    }
  }
}

// p = e^(x - lse) of one logit, and its gradient
__device__ __forceinline__ float logit_grad(float x, float lse, float dlp, float dent, float ent) {
  const float d = x - lse;
  const float pr = expf(d);
  float g = -dlp * pr;
  if (dent != 0.f && pr != 0.f) g -= dent * pr * (d + ent);
  return g;
}

template <typename T>
__global__ void __launch_bounds__(kLogThreads) logprob_backward_kernel(const LogprobParams p,
                                                                       const LogprobGradPtrs a) {
  pdl_launch_dependents();
  pdl_wait();
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    T const *x = static_cast<T const *>(a.x) + row * p.s_x;
    T *dx = static_cast<T *>(a.dx) + row * p.s_dx;
    const float lse = a.lse[row];
    const int64_t t = a.targets ? a.targets[row] : -1;
    float dlp = t >= 0 ? a.dlogprob[row] : 0.f;
    if (t >= p.vocab) dlp = logit_nan();
    const float dent = a.dentropy ? a.dentropy[row] : 0.f, ent = a.dentropy ? a.entropy[row] : 0.f;
    const bool none = lse == -INFINITY;
    for (int64_t c = threadIdx.x; c < p.vocab; c += kLogThreads) {
      float g = none ? 0.f : logit_grad(to_f32(x[c]), lse, dlp, dent, ent);
      if (c == t && !none) g += dlp;
      dx[c] = from_f32<T>(g);
    }
  }
}

static dim3 logprob_grid(int64_t rows, int num_sms) {
  const int64_t most = (int64_t)num_sms * 8;
  return dim3((unsigned)(rows < most ? rows : most));
}

cudaError_t launch_logprob(LogprobParams const &p, LogprobPtrs const &a, int num_sms, cudaStream_t st) {
  auto kern = p.dt == EIR_FP32 ? logprob_kernel<float> : logprob_kernel<__nv_bfloat16>;
  return launch_kernel(kern, logprob_grid(p.rows, num_sms), dim3(kLogThreads), 0, st, p, a);
}

cudaError_t launch_logprob_backward(LogprobParams const &p, LogprobGradPtrs const &a, int num_sms,
                                    cudaStream_t st) {
  auto kern = p.dt == EIR_FP32 ? logprob_backward_kernel<float> : logprob_backward_kernel<__nv_bfloat16>;
  return launch_kernel(kern, logprob_grid(p.rows, num_sms), dim3(kLogThreads), 0, st, p, a);
}

}  // namespace eir
