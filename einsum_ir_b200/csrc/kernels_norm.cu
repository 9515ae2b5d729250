// Root-mean-square norm with the residual's addition, its backward pass, and
// the quantisation of rows to 8-bit integers.
//
// Forward, a row of C columns: h = x + r, rstd = (sum h^2 / C + eps)^(-1/2),
// y = h rstd w. With 8-bit output v = h w, m = max|v|: y / s = v 127 / m for
// s = m rstd / 127, so the integers need no rstd and the row's two statistics
// (sum of squares, maximum) come from one pass. Backward: g = w dy,
// dx = rstd (g - h rstd^2 mean(g h)) + dsum, dw = sum over rows of dy h rstd.
// All sums in FP32. Bound by memory: each input is read once from HBM and each
// output written once; the second pass over a row hits L2.
#include "eir_launch.h"
#include "eir_common.cuh"
#include "op_common.cuh"
#include "op_params.h"

namespace eir {

constexpr int kRowThreads = 256;

// one CTA a row: a pass for the statistics, a pass for the output
template <typename T>
__global__ void __launch_bounds__(kRowThreads) norm_kernel(const NormParams p, const NormPtrs a) {
  __shared__ uint32_t red[64];
  pdl_launch_dependents();
  pdl_wait();
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    T const *x = static_cast<T const *>(a.x) + row * p.s_x;
    T const *r = a.res ? static_cast<T const *>(a.res) + row * p.s_res : nullptr;
    T *sum = a.sum ? static_cast<T *>(a.sum) + row * p.s_sum : nullptr;
    float ss = 0.f;
    uint32_t mx = 0;
    for (int64_t c = threadIdx.x; c < p.cols; c += kRowThreads) {
      float h = to_f32(x[c]);
      if (r) h += to_f32(r[c]);
      ss += h * h;
      const float w = a.w ? ld_any(a.w, p.dt_w, c) : 1.f;
      mx = max(mx, abs_bits(__fmul_rn(h, w)));
    }
    block_sum_max<kRowThreads / 32>(ss, mx, red);
    const float rstd = rsqrtf(ss / (float)p.cols + p.eps);
    const QuantScale q = quant_scale(mx, rstd);
    for (int64_t c = threadIdx.x; c < p.cols; c += kRowThreads) {
      float h = to_f32(x[c]);
      if (r) h += to_f32(r[c]);
      const float w = a.w ? ld_any(a.w, p.dt_w, c) : 1.f;
      if (sum) sum[c] = from_f32<T>(h);
      if (p.dt_out == EIR_INT8)
        static_cast<int8_t *>(a.out)[row * p.s_out + c] = (int8_t)quant_one(__fmul_rn(h, w), q);
      else
        st_any(a.out, p.dt_out, row * p.s_out + c, h * rstd * w);
    }
    if (threadIdx.x == 0) {
      if (a.rstd) a.rstd[row] = rstd;
      if (p.dt_out == EIR_INT8) a.scale[row] = q.scale;
    }
  }
}

// a CTA walks rows blockIdx.x, + gridDim.x, ...; its thread t owns the columns
// t, t + 256, ... of every row and adds their dy h rstd into its partial row
// of the weight gradient (same thread, same order: no atomics)
template <typename T>
__global__ void __launch_bounds__(kRowThreads) norm_backward_kernel(const NormParams p, const NormGradPtrs a) {
  __shared__ uint32_t red[64];
  pdl_launch_dependents();
  pdl_wait();
  float *part = a.part ? a.part + (int64_t)blockIdx.x * p.cols : nullptr;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    T const *h = static_cast<T const *>(a.h) + row * p.s_h;
    const float rstd = a.rstd[row];
    float gh = 0.f;
    uint32_t unused = 0;
    for (int64_t c = threadIdx.x; c < p.cols; c += kRowThreads) {
      const float w = a.w ? ld_any(a.w, p.dt_w, c) : 1.f;
      gh += w * ld_any(a.dy, p.dt_grad, row * p.s_dy + c) * to_f32(h[c]);
    }
    block_sum_max<kRowThreads / 32>(gh, unused, red);
    const float k = rstd * rstd * (gh / (float)p.cols);
    for (int64_t c = threadIdx.x; c < p.cols; c += kRowThreads) {
      const float w = a.w ? ld_any(a.w, p.dt_w, c) : 1.f;
      const float dy = ld_any(a.dy, p.dt_grad, row * p.s_dy + c), hv = to_f32(h[c]);
      float d = rstd * (w * dy - hv * k);
      if (a.dsum) d += ld_any(a.dsum, p.dt_grad, row * p.s_dsum + c);
      if (part) part[c] = (row == blockIdx.x ? 0.f : part[c]) + dy * (hv * rstd);
      st_any(a.dx, p.dt_grad, row * p.s_dx + c, d);
    }
  }
}

// dw[c] = sum of the partial rows, in their order
__global__ void __launch_bounds__(kRowThreads) norm_dweight_kernel(int64_t cols, float const *__restrict__ part,
                                                                   int64_t n_part, float *__restrict__ dw) {
  pdl_launch_dependents();
  pdl_wait();
  const int64_t c = (int64_t)blockIdx.x * kRowThreads + threadIdx.x;
  if (c >= cols) return;
  float s = 0.f;
  for (int64_t i = 0; i < n_part; ++i) s += part[i * cols + c];
  dw[c] = s;
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads) quantize_kernel(const QuantizeParams p, void const *xv,
                                                               int8_t *__restrict__ out, float *scale) {
  __shared__ uint32_t red[64];
  pdl_launch_dependents();
  pdl_wait();
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    T const *x = static_cast<T const *>(xv) + row * p.s_x;
    uint32_t mx = 0;
    float unused = 0.f;
    for (int64_t c = threadIdx.x; c < p.cols; c += kRowThreads) mx = max(mx, abs_bits(to_f32(x[c])));
    block_sum_max<kRowThreads / 32>(unused, mx, red);
    const QuantScale q = quant_scale(mx, 1.f);
    for (int64_t c = threadIdx.x; c < p.cols; c += kRowThreads)
      out[row * p.s_out + c] = (int8_t)quant_one(to_f32(x[c]), q);
    if (threadIdx.x == 0) scale[row] = q.scale;
  }
}

static dim3 row_grid(int64_t rows, int num_sms) {
  const int64_t most = (int64_t)num_sms * 8;
  return dim3((unsigned)(rows < most ? rows : most));
}

cudaError_t launch_norm(NormParams const &p, NormPtrs const &a, int num_sms, cudaStream_t st) {
  auto kern = p.dt == EIR_FP32 ? norm_kernel<float> : norm_kernel<__nv_bfloat16>;
  return launch_kernel(kern, row_grid(p.rows, num_sms), dim3(kRowThreads), 0, st, p, a);
}

int64_t norm_backward_ctas(NormParams const &p, int num_sms) { return row_grid(p.rows, num_sms).x; }

cudaError_t launch_norm_backward(NormParams const &p, NormGradPtrs const &a, int num_sms, cudaStream_t st) {
  auto kern = p.dt == EIR_FP32 ? norm_backward_kernel<float> : norm_backward_kernel<__nv_bfloat16>;
  return launch_kernel(kern, row_grid(p.rows, num_sms), dim3(kRowThreads), 0, st, p, a);
}

cudaError_t launch_norm_dweight(NormParams const &p, float const *part, int64_t n_part, float *dw,
                                cudaStream_t st) {
  return launch_kernel(norm_dweight_kernel, dim3((unsigned)((p.cols + kRowThreads - 1) / kRowThreads)),
                       dim3(kRowThreads), 0, st, p.cols, part, n_part, dw);
}

cudaError_t launch_quantize(QuantizeParams const &p, void const *x, int8_t *q, float *scale, int num_sms,
                            cudaStream_t st) {
  auto kern = p.dt == EIR_FP32 ? quantize_kernel<float> : quantize_kernel<__nv_bfloat16>;
  return launch_kernel(kern, row_grid(p.rows, num_sms), dim3(kRowThreads), 0, st, p, x, q, scale);
}

}  // namespace eir
