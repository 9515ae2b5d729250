// C-ABI of the row operators and the 8-bit contraction (eir_operators.h):
// argument checks, workspaces and launches.
#include <algorithm>
#include <mutex>
#include <new>
#include <string>
#include "eir_operators.h"
#include "eir_plan.h"

namespace {

using eir::ProfScope;

enum { kWhatNorm = 3, kWhatQuantize = 4, kWhatInt8 = 5, kWhatLogprob = 6 };

int fail(int code, char const *msg) { return eir::api_set_error(code, msg); }
int bad_argument(char const *msg) { return fail(EIR_INVALID_ARGUMENT, msg); }
int null_pointer(char const *msg) { return fail(EIR_NO_DATA_PTR_PROVIDED, msg); }

bool is_float(int dt) { return dt == EIR_FP32 || dt == EIR_BF16; }
char const *type_text(int dt) { return dt == EIR_FP32 ? "fp32" : dt == EIR_BF16 ? "bf16" : "int8"; }
int64_t type_bytes(int dt) { return dt == EIR_FP32 ? 4 : dt == EIR_BF16 ? 2 : 1; }

// rows x cols within the range of the kernels' 64-bit offsets and 31-bit grids
bool sizes_ok(int64_t rows, int64_t cols) {
  return rows >= 0 && rows <= INT32_MAX && cols >= 1 && cols <= INT32_MAX;
}
bool stride_in_ok(int64_t s) { return s >= 0 && s < ((int64_t)1 << 40); }
bool stride_out_ok(int64_t s, int64_t cols, int64_t rows) {
  return stride_in_ok(s) && (rows <= 1 || s >= cols);
}
bool aligned(void const *p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % (uintptr_t)bytes == 0; }

// the plan object, or null when memory is out (no exception leaves the C entry)
template <typename Fill>
int make_plan(eir_plan **out, int what, int family, Fill fill) {
  eir_plan *p = nullptr;
  try {
    p = new eir_plan();
    p->what = what;
    p->family = family;
    fill(p);
  } catch (std::exception const &) {
    delete p;
    return fail(EIR_UNDEFINED_ERROR, "out of host memory");
  }
  *out = p;
  return EIR_SUCCESS;
}

// Tiling of an 8-bit contraction on the tensor cores. Pair tiles where one-CTA
// tiles would not all fit the GPU at once (two an SM), and from 32 of them (of the GPU's 74 CTA pairs)
// on for a longer K walk, since one-CTA tiles move twice the operand bytes (512 tokens x 4096 x 2048:
// 10.1 us against 11.3; 1024 x 4096 x 1024: 8.1 against 7.2). Else one-CTA tiles of just enough
// tokens, the K walk of each split over a cluster. The split is the one with the least time by this
// account, in tenths of a K block (0.25 us): the CTA's own K blocks, and for the exchange 45, half the
// tile's tokens, and 6 to 10 a CTA (100 tokens x 4096: K = 1024 takes 5.7 us unsplit and 8.2 split by 4,
// K = 4096 12.1 and 10.4, 10.8 split by 8). All tiles' clusters have to fit the GPU at once, two CTAs
// an SM (measured limits; a second wave costs more than the split gains: 256 tokens x 4096 x 4096,
// 64 tiles, take 14.4 us unsplit, 11.8 split by 4 and 21.7 split by 8).
eir::I8TcPlan i8_tiling(eir::I8Params const &p) {
  eir::I8TcPlan t;
  const int64_t blocks = (p.k + 127) / 128;
  t.c_tiles = (p.n + 255) / 256;  // gated: 128 gates and their values a tile
  t.t_tiles = (p.m + 255) / 256;
  const int64_t single = ((p.n + 127) / 128) * ((p.m + 127) / 128);
  if (p.m > 128 && (single > 296 || (t.c_tiles * t.t_tiles >= 32 && blocks > 8))) return t;
  t.tokens = 128;
  for (int n : {96, 80, 64, 32, 16})
    if (p.m <= n) t.tokens = n;
  t.c_tiles = (p.n + 127) / 128;
  t.t_tiles = (p.m + t.tokens - 1) / t.tokens;
  struct {
    int split, tiles;
  } const fits[] = {{2, 148}, {3, 90}, {4, 66}, {8, 32}};
  int64_t least = 10 * blocks;
  for (auto const &f : fits) {
    const int64_t cost =
        10 * ((blocks + f.split - 1) / f.split) + 45 + t.tokens / 2 + f.split * (6 + t.tokens / 32);
    if (t.c_tiles * t.t_tiles > f.tiles || blocks < f.split || cost >= least) continue;
    t.split = f.split;
    least = cost;
  }
  return t;
}

// an operand's rows as the TMA loads take them: read in place where base and
// stride are multiples of 16 bytes, else copied into the workspace
struct I8Operand {
  int8_t const *ptr;
  int64_t rows, stride;
  bool copy;
};
int64_t packed_stride(int64_t k) { return (k + 15) / 16 * 16; }
I8Operand i8_operand(void const *ptr, int64_t rows, int64_t k, int64_t stride) {
  I8Operand o{static_cast<int8_t const *>(ptr), rows, stride, false};
  if (rows == 1) o.stride = packed_stride(k);  // no second row: any stride will do
  o.copy = !aligned(ptr, 16) || o.stride % 16 != 0 || o.stride < k;
  return o;
}

// K rows of 128 bytes; `halves` (a gated layer's right operand): gate rows and
// value rows as the third dim, 16 rows of each in a box
int i8_map(I8Operand const &o, int64_t k, int box_rows, bool halves, CUtensorMap *map) {
  eir::MapSpec m;
  m.rank = halves ? 3 : 2;
  m.dims[0] = (uint64_t)k;
  m.dims[1] = (uint64_t)(halves ? o.rows / 2 : o.rows);
  m.dims[2] = 2;
  m.strides_bytes[0] = (uint64_t)o.stride;
  m.strides_bytes[1] = (uint64_t)(o.rows / 2 * o.stride);
  m.box[0] = 128;
  m.box[1] = halves ? 16 : (uint32_t)box_rows;
  m.box[2] = halves ? 2 : 1;
  m.dtype = CU_TENSOR_MAP_DATA_TYPE_UINT8;
  return eir::api_encode_map(m, o.ptr, map);
}

// One token: the row kernel, but for large layers that TMA can stream in place (4096 x 4096: 4.4 us against
// 6.0; 8192 x 28672: 40.6 against 37.9). It reads operands of any alignment, so that one token copies none
bool i8_large_row(eir::I8Params const &p) { return p.n * p.k >= ((int64_t)1 << 26); }

int launched(cudaError_t e, char const *where) {
  if (e != cudaSuccess) return eir::api_cuda_fail(e, where);
  eir::api_count_launch();
  return EIR_SUCCESS;
}

}  // namespace

extern "C" {

// ---------------------------------------------------------------- norm

int eir_norm_plan_create(eir_norm_desc const *d, eir_plan **out) {
  if (d == nullptr || out == nullptr) return bad_argument("null descriptor or plan pointer");
  if (!sizes_ok(d->rows, d->cols)) return bad_argument("norm: rows must be 0 .. 2^31 - 1 and cols 1 .. 2^31 - 1");
  if (!is_float(d->dtype) || !is_float(d->dtype_weight) || !is_float(d->dtype_grad) ||
      !(is_float(d->dtype_out) || d->dtype_out == EIR_INT8))
    return fail(EIR_INVALID_DTYPE, "norm: FP32 or BF16 data (dtype_out: INT8 too)");
  if (!(d->eps >= 0.0) || d->eps > 3.0e38) return bad_argument("norm: eps must be a finite number >= 0");
  for (int64_t s : {d->stride_x, d->stride_residual, d->stride_h, d->stride_dy, d->stride_dsum})
    if (!stride_in_ok(s)) return bad_argument("norm: an input's row stride must be >= 0");
  for (int64_t s : {d->stride_sum, d->stride_out, d->stride_dx})
    if (!stride_out_ok(s, d->cols, d->rows)) return bad_argument("norm: an output's row stride must be >= cols");
  return make_plan(out, kWhatNorm, EIR_FAMILY_ROW, [&](eir_plan *p) {
    eir::NormParams &n = p->norm;
    n.rows = d->rows;
    n.cols = d->cols;
    n.dt = d->dtype;
    n.dt_w = d->dtype_weight;
    n.dt_out = d->dtype_out;
    n.dt_grad = d->dtype_grad;
    n.eps = (float)d->eps;
    n.s_x = d->stride_x;
    n.s_res = d->stride_residual;
    n.s_sum = d->stride_sum;
    n.s_out = d->stride_out;
    n.s_h = d->stride_h;
    n.s_dy = d->stride_dy;
    n.s_dsum = d->stride_dsum;
    n.s_dx = d->stride_dx;
    p->empty = d->rows == 0;
    // partial rows of the weight gradient
    p->ws_bytes = eir::norm_backward_parts(n, eir::kMaxSms) * eir::norm_part_pitch(d->cols) * 4;
    p->text = std::string("norm ") + type_text(n.dt) + " -> " + type_text(n.dt_out) + " rows=" +
              std::to_string(n.rows) + " cols=" + std::to_string(n.cols);
  });
}

int eir_norm(eir_plan *p, void const *x, void const *residual, void const *weight, void *sum, void *out,
             float *scale, float *rstd, void *stream) {
  if (p == nullptr || p->what != kWhatNorm) return bad_argument("not a norm plan");
  if (p->empty) return EIR_SUCCESS;
  eir::NormParams const &n = p->norm;
  if (x == nullptr || out == nullptr) return null_pointer("norm: null x or out");
  if (n.dt_out == EIR_INT8 && scale == nullptr) return null_pointer("norm: INT8 output needs scale");
  const int64_t e = type_bytes(n.dt);
  if (!aligned(x, e) || !aligned(residual, e) || !aligned(sum, e) || !aligned(weight, type_bytes(n.dt_w)) ||
      !aligned(out, type_bytes(n.dt_out)) || !aligned(scale, 4) || !aligned(rstd, 4))
    return bad_argument("norm: a pointer is not aligned to its element");
  int num_sms = 0;
  uint32_t *err = nullptr;
  int rc = eir::api_device(&num_sms, &err);
  if (rc != EIR_SUCCESS) return rc;
  const eir::NormPtrs a{x, residual, weight, sum, out, scale, rstd};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  ProfScope prof(p, st);
  return launched(eir::launch_norm(n, a, err, num_sms, st), "norm launch");
}

int eir_norm_backward(eir_plan *p, void const *dy, void const *h, void const *weight, float const *rstd,
                      void const *dsum, void *dx, float *dweight, void *stream) {
  if (p == nullptr || p->what != kWhatNorm) return bad_argument("not a norm plan");
  return eir_norm_backward_strided(p, dy, h, p->norm.s_h, weight, rstd, dsum, dx, dweight, stream);
}

int eir_norm_backward_strided(eir_plan *p, void const *dy, void const *h, int64_t stride_h, void const *weight,
                              float const *rstd, void const *dsum, void *dx, float *dweight, void *stream) {
  if (p == nullptr || p->what != kWhatNorm) return bad_argument("not a norm plan");
  if (!stride_in_ok(stride_h)) return bad_argument("norm backward: the row stride of h must be >= 0");
  eir::NormParams n = p->norm;
  n.s_h = stride_h;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (!aligned(dweight, 4)) return bad_argument("norm backward: a pointer is not aligned to its element");
  if (p->empty) {  // a sum over no rows
    if (dweight == nullptr) return EIR_SUCCESS;
    cudaError_t e = cudaMemsetAsync(dweight, 0, (size_t)n.cols * 4, st);
    return e == cudaSuccess ? EIR_SUCCESS : eir::api_cuda_fail(e, "cudaMemsetAsync(dweight)");
  }
  if (dy == nullptr || h == nullptr || rstd == nullptr || dx == nullptr)
    return null_pointer("norm backward: null dy, h, rstd or dx");
  const int64_t e = type_bytes(n.dt), g = type_bytes(n.dt_grad);
  if (!aligned(h, e) || !aligned(dy, g) || !aligned(dsum, g) || !aligned(dx, g) || !aligned(rstd, 4) ||
      !aligned(weight, type_bytes(n.dt_w)))
    return bad_argument("norm backward: a pointer is not aligned to its element");
  int num_sms = 0;
  uint32_t *err = nullptr;
  int rc = eir::api_device(&num_sms, &err);
  if (rc != EIR_SUCCESS) return rc;
  num_sms = std::min(num_sms, eir::kMaxSms);
  eir::NormGradPtrs a{dy, h, weight, dsum, rstd, dx, dweight, nullptr};
  int64_t parts = 0;
  std::unique_lock<std::mutex> held;
  if (dweight != nullptr) {
    void *ws = nullptr;
    held = p->op_ws.hold();
    rc = p->op_ws.take(p->ws_bytes, st, &ws);
    if (rc != EIR_SUCCESS) return rc;
    a.part = static_cast<float *>(ws);
  }
  {
    ProfScope prof(p, st);
    rc = launched(eir::launch_norm_backward(n, a, err, num_sms, st, &parts), "norm backward launch");
  }
  if (dweight == nullptr) return rc;
  if (rc == EIR_SUCCESS)
    rc = launched(eir::launch_norm_dweight(n, a.part, parts, dweight, st), "norm weight gradient launch");
  return p->op_ws.used(st, rc);
}

// ---------------------------------------------------------------- quantize

int eir_quantize_plan_create(eir_quantize_desc const *d, eir_plan **out) {
  if (d == nullptr || out == nullptr) return bad_argument("null descriptor or plan pointer");
  if (!sizes_ok(d->rows, d->cols))
    return bad_argument("quantize: rows must be 0 .. 2^31 - 1 and cols 1 .. 2^31 - 1");
  if (!is_float(d->dtype)) return fail(EIR_INVALID_DTYPE, "quantize: FP32 or BF16 data");
  if (!stride_in_ok(d->stride_x)) return bad_argument("quantize: the input's row stride must be >= 0");
  if (!stride_out_ok(d->stride_out, d->cols, d->rows))
    return bad_argument("quantize: the output's row stride must be >= cols");
  return make_plan(out, kWhatQuantize, EIR_FAMILY_ROW, [&](eir_plan *p) {
    p->quant.rows = d->rows;
    p->quant.cols = d->cols;
    p->quant.dt = d->dtype;
    p->quant.s_x = d->stride_x;
    p->quant.s_out = d->stride_out;
    p->empty = d->rows == 0;
    p->text = std::string("quantize ") + type_text(d->dtype) + " rows=" + std::to_string(d->rows) +
              " cols=" + std::to_string(d->cols);
  });
}

int eir_quantize(eir_plan *p, void const *x, void *q, float *scale, void *stream) {
  if (p == nullptr || p->what != kWhatQuantize) return bad_argument("not a quantize plan");
  if (p->empty) return EIR_SUCCESS;
  if (x == nullptr || q == nullptr || scale == nullptr) return null_pointer("quantize: null x, q or scale");
  if (!aligned(x, type_bytes(p->quant.dt)) || !aligned(scale, 4))
    return bad_argument("quantize: a pointer is not aligned to its element");
  int num_sms = 0;
  uint32_t *err = nullptr;
  int rc = eir::api_device(&num_sms, &err);
  if (rc != EIR_SUCCESS) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  ProfScope prof(p, st);
  return launched(eir::launch_quantize(p->quant, x, static_cast<int8_t *>(q), scale, err, num_sms, st),
                  "quantize launch");
}

// ---------------------------------------------------------------- 8-bit contraction

int eir_contract_int8_plan_create(eir_contract_int8_desc const *d, eir_plan **out) {
  if (d == nullptr || out == nullptr) return bad_argument("null descriptor or plan pointer");
  if (d->m < 0 || d->n < 0 || d->k < 0 || d->m > INT32_MAX || d->n > INT32_MAX)
    return bad_argument("8-bit contraction: m, n must be 0 .. 2^31 - 1");
  if (d->k > 131071) return bad_argument("8-bit contraction: k must be at most 131071 (32-bit sums)");
  if (!is_float(d->dtype_out)) return fail(EIR_INVALID_DTYPE, "8-bit contraction: dtype_out FP32 or BF16");
  if (d->activation < EIR_ACT_NONE || d->activation > EIR_ACT_GATED_SILU)
    return fail(EIR_INVALID_KTYPE, "8-bit contraction: unknown activation");
  const bool gated = d->activation == EIR_ACT_GATED_SILU;
  if (gated && d->n % 2 != 0) return bad_argument("8-bit contraction: gated SiLU needs an even n");
  if (!stride_in_ok(d->stride_left) || !stride_in_ok(d->stride_right))
    return bad_argument("8-bit contraction: an input's row stride must be >= 0");
  const int64_t n_out = gated ? d->n / 2 : d->n;
  if (!stride_out_ok(d->stride_out, n_out, d->m))
    return bad_argument("8-bit contraction: the output's row stride must be >= its columns");
  return make_plan(out, kWhatInt8, EIR_FAMILY_SIMT, [&](eir_plan *p) {
    eir::I8Params &q = p->i8;
    q.m = d->m;
    q.n = d->n;
    q.k = d->k;
    q.dt_out = d->dtype_out;
    q.act = d->activation;
    q.s_l = d->stride_left;
    q.s_r = d->stride_right;
    q.s_out = d->stride_out;
    p->empty = d->m == 0 || n_out == 0;
    const bool row = d->m == 1 && !i8_large_row(q), products = d->k > 0 && !p->empty;
    if (products && !row) {
      p->family = EIR_FAMILY_TC;
      p->i8_tc = i8_tiling(q);
      // copies of operands that TMA cannot read in place
      if (d->m > 1) p->ws_bytes = (d->m + d->n) * packed_stride(d->k);
    }
    p->text = std::string("int8 ") + (!products ? "simt" : row ? "row" : p->i8_tc.tokens == 0 ? "pair" : "split");
    if (p->family == EIR_FAMILY_TC)
      p->text += " tokens=" + std::to_string(p->i8_tc.tokens) + " split=" + std::to_string(p->i8_tc.split);
    p->text += " m=" + std::to_string(d->m) + " n=" + std::to_string(d->n) + " k=" + std::to_string(d->k);
    if (d->m == 1 && p->family == EIR_FAMILY_TC) p->text += " (row where operands are off the 16-byte grid)";
  });
}

int eir_contract_int8(eir_plan *p, void const *left, void const *right, float const *scale_left,
                      float const *scale_right, float const *bias, void *out, void *stream) {
  if (p == nullptr || p->what != kWhatInt8) return bad_argument("not an 8-bit contraction plan");
  if (p->empty) return EIR_SUCCESS;
  if (out == nullptr || (p->i8.k > 0 && (left == nullptr || right == nullptr)))
    return null_pointer("8-bit contraction: null operand pointer");
  if (!aligned(scale_left, 4) || !aligned(scale_right, 4) || !aligned(bias, 4) ||
      !aligned(out, type_bytes(p->i8.dt_out)))
    return bad_argument("8-bit contraction: a pointer is not aligned to its element");
  const eir::I8Ptrs a{static_cast<int8_t const *>(left), static_cast<int8_t const *>(right),
                      scale_left, scale_right, bias, out};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int num_sms = 0;
  uint32_t *err = nullptr;
  int rc = eir::api_device(&num_sms, &err);
  if (rc != EIR_SUCCESS) return rc;
  if (p->i8.k == 0) {
    ProfScope prof(p, st);
    return launched(eir::launch_i8_bias(p->i8, a, num_sms, st), "8-bit contraction launch");
  }
  I8Operand ops[2] = {i8_operand(left, p->i8.m, p->i8.k, p->i8.s_l), i8_operand(right, p->i8.n, p->i8.k, p->i8.s_r)};
  if (p->i8.m == 1 && (ops[0].copy || ops[1].copy || !i8_large_row(p->i8))) {
    ProfScope prof(p, st);
    return launched(eir::launch_i8_row(p->i8, a, num_sms, st), "8-bit contraction launch");
  }
  const int64_t ld = packed_stride(p->i8.k);
  const bool copies = ops[0].copy || ops[1].copy;
  eir::I8Pack packs[2] = {};
  std::unique_lock<std::mutex> held;
  if (copies) {
    void *ws = nullptr;
    held = p->op_ws.hold();
    rc = p->op_ws.take(p->ws_bytes, st, &ws);
    if (rc != EIR_SUCCESS) return rc;
    for (int i = 0; i < 2; ++i) {
      I8Operand &o = ops[i];
      if (!o.copy) continue;
      int8_t *to = static_cast<int8_t *>(ws) + (i == 0 ? 0 : p->i8.m * ld);
      packs[i] = eir::I8Pack{o.rows, i == 0 ? p->i8.s_l : p->i8.s_r, o.ptr, to};
      o.ptr = to;
      o.stride = ld;
    }
  }
  CUtensorMap map_t, map_c;
  rc = i8_map(ops[0], p->i8.k, eir::i8_box_tokens(p->i8_tc), false, &map_t);
  if (rc != EIR_SUCCESS) return rc;
  rc = i8_map(ops[1], p->i8.k, 128, p->i8.act == EIR_ACT_GATED_SILU, &map_c);
  if (rc != EIR_SUCCESS) return rc;
  if (copies) rc = launched(eir::launch_i8_pack(packs[0], packs[1], p->i8.k, ld, num_sms, st), "8-bit operand copy");
  if (rc == EIR_SUCCESS) {
    ProfScope prof(p, st);
    rc = launched(eir::launch_i8_tc(p->i8_tc, map_c, map_t, p->i8, a, err, st), "8-bit contraction launch");
  }
  return copies ? p->op_ws.used(st, rc) : rc;
}

// ---------------------------------------------------------------- log probabilities

int eir_logprob_plan_create(eir_logprob_desc const *d, eir_plan **out) {
  if (d == nullptr || out == nullptr) return bad_argument("null descriptor or plan pointer");
  if (!sizes_ok(d->rows, d->vocab))
    return bad_argument("logprob: rows must be 0 .. 2^31 - 1 and vocab 1 .. 2^31 - 1");
  if (!is_float(d->dtype)) return fail(EIR_INVALID_DTYPE, "logprob: FP32 or BF16 logits");
  if (d->top < 0 || d->top > 32 || d->top > d->vocab)
    return bad_argument("logprob: top must be 0 .. min(32, vocab)");
  if (!stride_in_ok(d->stride_logits)) return bad_argument("logprob: the logits' row stride must be >= 0");
  if (!stride_out_ok(d->stride_dlogits, d->vocab, d->rows))
    return bad_argument("logprob: the gradient's row stride must be >= vocab");
  return make_plan(out, kWhatLogprob, EIR_FAMILY_ROW, [&](eir_plan *p) {
    eir::LogprobParams &l = p->logprob;
    l.rows = d->rows;
    l.vocab = d->vocab;
    l.dt = d->dtype;
    l.top = d->top;
    l.s_x = d->stride_logits;
    l.s_dx = d->stride_dlogits;
    p->empty = d->rows == 0;
    p->text = std::string("logprob ") + type_text(l.dt) + " rows=" + std::to_string(l.rows) +
              " vocab=" + std::to_string(l.vocab) + " top=" + std::to_string(l.top);
  });
}

int eir_logprob(eir_plan *p, void const *logits, int64_t const *targets, float *logprob, float *entropy,
                float *lse, float *top_logprob, int64_t *top_index, void *stream) {
  if (p == nullptr || p->what != kWhatLogprob) return bad_argument("not a log-probability plan");
  if (p->empty) return EIR_SUCCESS;
  if (logits == nullptr) return null_pointer("logprob: null logits");
  if ((targets == nullptr) != (logprob == nullptr))
    return null_pointer("logprob: targets and logprob go together");
  if (!aligned(logits, type_bytes(p->logprob.dt)) || !aligned(targets, 8) || !aligned(top_index, 8) ||
      !aligned(logprob, 4) || !aligned(entropy, 4) || !aligned(lse, 4) || !aligned(top_logprob, 4))
    return bad_argument("logprob: a pointer is not aligned to its element");
  int num_sms = 0;
  uint32_t *err = nullptr;
  int rc = eir::api_device(&num_sms, &err);
  if (rc != EIR_SUCCESS) return rc;
  eir::LogprobParams q = p->logprob;
  if (top_logprob == nullptr && top_index == nullptr) q.top = 0;
  const eir::LogprobPtrs a{logits, targets, logprob, entropy, lse, top_logprob, top_index};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  ProfScope prof(p, st);
  return launched(eir::launch_logprob(q, a, err, num_sms, st), "logprob launch");
}

int eir_logprob_backward(eir_plan *p, void const *logits, int64_t const *targets, float const *lse,
                         float const *entropy, float const *dlogprob, float const *dentropy, void *dlogits,
                         void *stream) {
  if (p == nullptr || p->what != kWhatLogprob) return bad_argument("not a log-probability plan");
  if (p->empty) return EIR_SUCCESS;
  if (logits == nullptr || lse == nullptr || dlogits == nullptr)
    return null_pointer("logprob backward: null logits, lse or dlogits");
  if ((targets == nullptr) != (dlogprob == nullptr))
    return null_pointer("logprob backward: targets and dlogprob go together");
  if (dentropy != nullptr && entropy == nullptr)
    return null_pointer("logprob backward: dentropy needs entropy");
  const int64_t e = type_bytes(p->logprob.dt);
  if (!aligned(logits, e) || !aligned(dlogits, e) || !aligned(targets, 8) || !aligned(lse, 4) ||
      !aligned(entropy, 4) || !aligned(dlogprob, 4) || !aligned(dentropy, 4))
    return bad_argument("logprob backward: a pointer is not aligned to its element");
  int num_sms = 0;
  uint32_t *err = nullptr;
  int rc = eir::api_device(&num_sms, &err);
  if (rc != EIR_SUCCESS) return rc;
  const eir::LogprobGradPtrs a{logits, targets, lse, entropy, dlogprob, dentropy, dlogits};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  ProfScope prof(p, st);
  return launched(eir::launch_logprob_backward(p->logprob, a, num_sms, st), "logprob backward launch");
}

}  // extern "C"
