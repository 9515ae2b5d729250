// Parameters of the row operators and the 8-bit contraction (eir_operators.h)
// and the host-callable launchers of their kernels (internal to the library).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace eir {

constexpr int kMaxSms = 160;  // sizes the workspaces of plans made before the device is known

struct NormParams {
  int64_t rows = 0, cols = 0;
  int32_t dt = 0, dt_w = 0, dt_out = 0, dt_grad = 0;
  float eps = 0.f;
  int64_t s_x = 0, s_res = 0, s_sum = 0, s_out = 0, s_h = 0, s_dy = 0, s_dsum = 0, s_dx = 0;
};

struct NormPtrs {
  void const *x, *res, *w;
  void *sum, *out;
  float *scale, *rstd;
};

struct NormGradPtrs {
  void const *dy, *h, *w, *dsum;
  float const *rstd;
  void *dx;
  float *dw;
  float *part;  // partial weight gradients [ctas][cols]
};

struct QuantizeParams {
  int64_t rows = 0, cols = 0;
  int32_t dt = 0;
  int64_t s_x = 0, s_out = 0;
};

struct I8Params {
  int64_t m = 0, n = 0, k = 0;
  int32_t dt_out = 0, act = 0;
  int64_t s_l = 0, s_r = 0, s_out = 0;
};

// how the tensor-core kernels tile a contraction: token tiles of `tokens`
// (0: the CTA-pair kernel), K split over clusters of `split` CTAs
struct I8TcPlan {
  int64_t c_tiles = 0, t_tiles = 0;
  int tokens = 0, split = 1;
};

struct I8Ptrs {
  int8_t const *l, *r;
  float const *scale_l, *scale_r, *bias;
  void *out;
};

struct LogprobParams {
  int64_t rows = 0, vocab = 0;
  int32_t dt = 0, top = 0;
  int64_t s_x = 0, s_dx = 0;
};

struct LogprobPtrs {
  void const *x;
  int64_t const *targets;
  float *logprob, *entropy, *lse, *top_logprob;
  int64_t *top_index;
};

struct LogprobGradPtrs {
  void const *x;
  int64_t const *targets;
  float const *lse, *entropy, *dlogprob, *dentropy;
  void *dx;
};

cudaError_t launch_norm(NormParams const &p, NormPtrs const &a, uint32_t *err, int num_sms, cudaStream_t st);
// elements between the partial rows of the weight gradient: 16-byte pieces
__host__ __device__ inline int64_t norm_part_pitch(int64_t cols) { return (cols + 3) & ~(int64_t)3; }
// the most partial rows of the weight gradient that the backward kernels write; *parts: how many
int64_t norm_backward_parts(NormParams const &p, int num_sms);
cudaError_t launch_norm_backward(NormParams const &p, NormGradPtrs const &a, uint32_t *err, int num_sms,
                                 cudaStream_t st, int64_t *parts);
cudaError_t launch_norm_dweight(NormParams const &p, float const *part, int64_t n_part, float *dw,
                                cudaStream_t st);
cudaError_t launch_quantize(QuantizeParams const &p, void const *x, int8_t *q, float *scale, uint32_t *err,
                            int num_sms, cudaStream_t st);
// k = 0: scales, bias and activation alone
cudaError_t launch_i8_bias(I8Params const &p, I8Ptrs const &a, int num_sms, cudaStream_t st);
cudaError_t launch_i8_tc(I8TcPlan const &tp, CUtensorMap const &map_channels, CUtensorMap const &map_tokens,
                         I8Params const &p, I8Ptrs const &a, uint32_t *err, cudaStream_t st);
// one token (m = 1), any stride and alignment
cudaError_t launch_i8_row(I8Params const &p, I8Ptrs const &a, int num_sms, cudaStream_t st);
// token rows of one TMA box of the tiling `tp`
int i8_box_tokens(I8TcPlan const &tp);
// rows of k bytes, `stride` apart, into rows `ld` bytes apart, of one or two operands (rows = 0: absent)
struct I8Pack {
  int64_t rows, stride;
  int8_t const *src;
  int8_t *dst;
};
cudaError_t launch_i8_pack(I8Pack const &one, I8Pack const &two, int64_t k, int64_t ld, int num_sms, cudaStream_t st);
cudaError_t launch_logprob(LogprobParams const &p, LogprobPtrs const &a, uint32_t *err, int num_sms,
                           cudaStream_t st);
cudaError_t launch_logprob_backward(LogprobParams const &p, LogprobGradPtrs const &a, int num_sms,
                                    cudaStream_t st);

}  // namespace eir
