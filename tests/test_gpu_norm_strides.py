"""The norm's forward and backward pass chained on plans whose x and sum lie differently."""
from __future__ import annotations

import pytest
import torch

from einsum_ir_b200 import cabi, operators as op
from tests._operators import norm64, norm_backward64
from tests.test_gpu_operators import BF16, CODE, F32, U, close, gen, round_tol, rows_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("pad_x,pad_sum", [(8, 0), (3, 0), (0, 8), (8, 3)])
@pytest.mark.parametrize("rows,cols", [(2, 96), (700, 136), (33, 1000), (900, 2311), (5, 20001)])
def test_forward_and_backward_on_one_plan(cuda, rows, cols, pad_x, pad_sum, dtype):
    """with a residual h is the sum, without one it is x"""
    g = gen(rows + cols + pad_x)
    x, res = rows_of(g, rows, cols, dtype, pad_x), rows_of(g, rows, cols, dtype, pad_x)
    s = rows_of(g, rows, cols, dtype, pad_sum)
    dy, w = rows_of(g, rows, cols, dtype), rows_of(g, 1, cols, dtype)[0]
    plan = op.NormPlan(rows, cols, CODE[dtype], eps=1e-5, stride_x=cols + pad_x, stride_residual=cols + pad_x,
                       stride_sum=cols + pad_sum)
    for residual in (res, None):
        y, rstd = torch.empty((rows, cols), device="cuda", dtype=dtype), torch.empty(rows, device="cuda")
        dx, dw = torch.empty_like(y), torch.empty(cols, device="cuda")
        plan.norm(x, y, weight=w, residual=residual, sum=None if residual is None else s, rstd=rstd)
        h = x if residual is None else s
        plan.backward(dy, h, rstd, dx, weight=w, dweight=dw)
        want_rstd = norm64(x, residual, w, 1e-5)["rstd"]
        close(rstd, want_rstd, want_rstd * (cols / 32 + 16) * U)
        want, want_w = norm_backward64(dy, h, w, rstd, None)
        r, gd, hd = rstd.double()[:, None], (dy.double() * w.double()).abs(), h.double().abs()
        parts = r * (gd + hd * r.square() * (gd * hd).mean(1, keepdim=True))
        close(dx, want, parts * ((cols / 32 + 16) * U) + round_tol(want, dtype))
        close(dw, want_w, (dy.double() * hd * r).abs().sum(0) * ((rows + 16) * U))
    cabi.check_device_errors()
