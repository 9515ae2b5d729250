"""The row operators and the 8-bit contraction (include/eir_operators.h).

``NormPlan`` (root-mean-square norm with the residual's addition, float or
8-bit output, and its backward pass), ``QuantizePlan`` (rows to 8-bit integers
with a scale a row), ``Int8ContractPlan`` (8-bit contraction with a scale for
each token and channel) and ``LogprobPlan`` (log probabilities of given tokens,
entropy, top alternatives, and their backward pass). As in ``cabi``, sizes,
types and strides are the plan's; a call takes device pointers or tensors,
writes into the caller's outputs and is asynchronous on ``stream``. Row strides
are in elements and default to packed rows.
"""
from __future__ import annotations

import ctypes
from ctypes import c_void_p

from . import cabi
from .cabi import BF16, FP32, INT8, check

ACT_NONE, ACT_RELU, ACT_GATED_SILU = 0, 1, 2
INVALID_ARGUMENT = 52  # a status code (eir_cuda.h)

__all__ = ["ACT_NONE", "ACT_RELU", "ACT_GATED_SILU", "FP32", "BF16", "INT8", "NormPlan", "QuantizePlan",
           "Int8ContractPlan", "LogprobPlan"]


def _ptr(x):
    """device address of a tensor, an address, or None"""
    if x is None or isinstance(x, int):
        return x
    return x.data_ptr()


# The forward calls below write the usual case out (tensors, or None where that
# is allowed) and leave plain addresses to an exception: a decoding step makes
# them every few microseconds (norm: 1.5 us in Python and ctypes instead of 1.9).


def _packed(stride, cols):
    return cols if stride is None else stride


class _OpPlan(cabi.Plan):
    def __init__(self, create, desc):
        h = c_void_p()
        check(create(ctypes.byref(desc), ctypes.byref(h)))
        super().__init__(h)


class NormPlan(_OpPlan):
    """h = x + residual; y = h * rstd * weight with rstd = (mean(h^2) + eps)^(-1/2)
    over rows of ``cols`` elements. ``dtype``: x, residual, sum and h;
    ``dtype_out``: y, FP32, BF16 or INT8 (default: dtype); ``dtype_grad``: dy, dsum and
    dx (default: dtype). ``stride_h``: of the backward pass's h (default: see backward)."""

    def __init__(self, rows, cols, dtype, dtype_weight=None, dtype_out=None, dtype_grad=None, eps=1e-6,
                 stride_x=None, stride_residual=None, stride_sum=None, stride_out=None, stride_h=None,
                 stride_dy=None, stride_dsum=None, stride_dx=None):
        pick = lambda t: dtype if t is None else t
        sx = _packed(stride_x, cols)
        super().__init__(cabi.lib().eir_norm_plan_create, cabi.EirNormDesc(
            rows, cols, dtype, pick(dtype_weight), pick(dtype_out), pick(dtype_grad), eps, sx,
            _packed(stride_residual, cols), _packed(stride_sum, cols), _packed(stride_out, cols),
            sx if stride_h is None else stride_h, _packed(stride_dy, cols), _packed(stride_dsum, cols),
            _packed(stride_dx, cols)))
        self._norm = cabi.lib().eir_norm
        self._backward = cabi.lib().eir_norm_backward_strided
        self._rows, self._cols, self._esize = rows, cols, 4 if dtype == FP32 else 2
        self._stride_x, self._stride_sum = sx, _packed(stride_sum, cols)
        # h's row stride; None: asked of h itself
        self._stride_h = stride_h if stride_h is not None else sx if sx == self._stride_sum or rows < 2 else None

    def norm(self, x, out, weight=None, residual=None, sum=None, scale=None, rstd=None, stream: int = 0) -> None:
        """out = y, or with INT8 output its integers (``scale``: FP32 [rows]);
        sum = h and rstd (FP32 [rows]) are what the backward pass reads."""
        try:
            rc = self._norm(self._h, x.data_ptr(), None if residual is None else residual.data_ptr(), None if
                            weight is None else weight.data_ptr(), None if sum is None else sum.data_ptr(),
                            out.data_ptr(), None if scale is None else scale.data_ptr(), None if rstd is None
                            else rstd.data_ptr(), stream)
        except AttributeError:
            rc = self._norm(self._h, _ptr(x), _ptr(residual), _ptr(weight), _ptr(sum), _ptr(out), _ptr(scale),
                            _ptr(rstd), stream)
        if rc:
            check(rc)

    def backward(self, dy, h, rstd, dx, weight=None, dsum=None, dweight=None, stream: int = 0) -> None:
        """dx: the gradient of x and of residual from dy and dsum (the
        gradient that reaches h past the norm); dweight: FP32 [cols]. ``h``
        is the forward call's sum, or its x where it had no residual. Its rows
        are the plan's ``stride_h`` apart; where that was not given, a tensor
        [..., cols] says itself whether they lie like x's or the sum's, and an
        address stands for rows ``stride_x`` apart."""
        stride_h = self._stride_h if self._stride_h is not None else self._row_stride_h(h)
        check(self._backward(self._h, _ptr(dy), _ptr(h), stride_h, _ptr(weight), _ptr(rstd), _ptr(dsum), _ptr(dx),
                             _ptr(dweight), stream))

    def _row_stride_h(self, h):
        x, sum = self._stride_x, self._stride_sum
        if not hasattr(h, "element_size"):
            return x
        if h.dim() > 1 and h.shape[-1] == self._cols and h.numel() == self._rows * self._cols:
            try:
                stride = h.view(self._rows, self._cols).stride(0)
            except RuntimeError:  # rows that are not one distance apart
                stride = -1
            if stride in (x, sum):
                return stride
            raise cabi.EirError(INVALID_ARGUMENT, f"norm backward: the rows of h are not stride_x ({x}) or stride_sum "
                                f"({sum}) apart: give stride_h")
        # a buffer of another shape: x's rows, unless it ends before theirs
        room = h.numel() * h.element_size() // self._esize - self._cols
        return sum if sum * (self._rows - 1) <= room < x * (self._rows - 1) else x


class QuantizePlan(_OpPlan):
    """Rows to 8-bit integers: q = round(x * 127 / max|x|), scale = max|x| / 127."""

    def __init__(self, rows, cols, dtype, stride_x=None, stride_out=None):
        super().__init__(cabi.lib().eir_quantize_plan_create, cabi.EirQuantizeDesc(
            rows, cols, dtype, 0, _packed(stride_x, cols), _packed(stride_out, cols)))
        self._quantize = cabi.lib().eir_quantize

    def quantize(self, x, q, scale, stream: int = 0) -> None:
        """q int8 [rows, cols], scale FP32 [rows]"""
        try:
            rc = self._quantize(self._h, x.data_ptr(), q.data_ptr(), scale.data_ptr(), stream)
        except AttributeError:
            rc = self._quantize(self._h, _ptr(x), _ptr(q), _ptr(scale), stream)
        if rc:
            check(rc)


class Int8ContractPlan(_OpPlan):
    """out[t, c] = act(sum_k left[t, k] right[c, k] * scale_left[t] * scale_right[c] + bias[c])
    for int8 ``left`` [m, k] (tokens) and ``right`` [n, k] (channels). ACT_GATED_SILU: out
    [m, n / 2] = silu(first half of the channels) * second half."""

    def __init__(self, m, n, k, dtype_out=BF16, activation=ACT_NONE, stride_left=None, stride_right=None,
                 stride_out=None):
        n_out = n // 2 if activation == ACT_GATED_SILU else n
        super().__init__(cabi.lib().eir_contract_int8_plan_create, cabi.EirContractInt8Desc(
            m, n, k, dtype_out, activation, _packed(stride_left, k), _packed(stride_right, k),
            _packed(stride_out, n_out)))
        self._contract = cabi.lib().eir_contract_int8

    def contract(self, left, right, scale_left, scale_right, out, bias=None, stream: int = 0) -> None:
        """scale_left FP32 [m], scale_right FP32 [n] (None: ones), bias FP32 [n] or None"""
        try:
            rc = self._contract(self._h, left.data_ptr(), right.data_ptr(), None if scale_left is None else
                                scale_left.data_ptr(), None if scale_right is None else scale_right.data_ptr(),
                                None if bias is None else bias.data_ptr(), out.data_ptr(), stream)
        except AttributeError:
            rc = self._contract(self._h, _ptr(left), _ptr(right), _ptr(scale_left), _ptr(scale_right),
                                _ptr(bias), _ptr(out), stream)
        if rc:
            check(rc)


class LogprobPlan(_OpPlan):
    """Log probabilities of given tokens over rows of ``vocab`` logits, with
    log-sum-exp, entropy and the ``top`` most likely tokens (ties: lowest index)."""

    def __init__(self, rows, vocab, dtype, top=0, stride_logits=None, stride_dlogits=None):
        super().__init__(cabi.lib().eir_logprob_plan_create, cabi.EirLogprobDesc(
            rows, vocab, dtype, top, _packed(stride_logits, vocab), _packed(stride_dlogits, vocab)))
        self._logprob = cabi.lib().eir_logprob
        self._backward = cabi.lib().eir_logprob_backward

    def logprob(self, logits, targets=None, logprob=None, entropy=None, lse=None, top_logprob=None,
                top_index=None, stream: int = 0) -> None:
        """targets int64 [rows] (negative: ignored); logprob, entropy, lse FP32
        [rows]; top_logprob FP32 and top_index int64 [rows, top]"""
        try:
            rc = self._logprob(self._h, logits.data_ptr(), None if targets is None else targets.data_ptr(), None
                               if logprob is None else logprob.data_ptr(), None if entropy is None else
                               entropy.data_ptr(), None if lse is None else lse.data_ptr(), None if top_logprob
                               is None else top_logprob.data_ptr(), None if top_index is None else
                               top_index.data_ptr(), stream)
        except AttributeError:
            rc = self._logprob(self._h, _ptr(logits), _ptr(targets), _ptr(logprob), _ptr(entropy), _ptr(lse),
                               _ptr(top_logprob), _ptr(top_index), stream)
        if rc:
            check(rc)

    def backward(self, logits, targets, lse, dlogprob, dlogits, entropy=None, dentropy=None,
                 stream: int = 0) -> None:
        """dlogits from the gradients of logprob and entropy"""
        check(self._backward(self._h, _ptr(logits), _ptr(targets), _ptr(lse), _ptr(entropy), _ptr(dlogprob),
                             _ptr(dentropy), _ptr(dlogits), stream))
