"""CPU tests of the row operators and the 8-bit contraction: what their plans
and calls refuse, and their gradients' formulas against differences."""
from __future__ import annotations

import pytest
import torch

from einsum_ir_b200 import cabi, operators as op
from tests._operators import logprob_backward64, logprob64, norm64, norm_backward64

BAD_ARGUMENT, NO_POINTER, BAD_DTYPE, BAD_KTYPE = 52, 4, 9, 10


def _refused(code, make):
    with pytest.raises(cabi.EirError) as e:
        make()
    assert e.value.code == code, e.value


@pytest.mark.parametrize("code,args", [
    (BAD_ARGUMENT, dict(rows=-1)), (BAD_ARGUMENT, dict(cols=0)), (BAD_ARGUMENT, dict(rows=1 << 31)),
    (BAD_ARGUMENT, dict(eps=-1.0)), (BAD_ARGUMENT, dict(eps=float("nan"))), (BAD_ARGUMENT, dict(eps=float("inf"))),
    (BAD_ARGUMENT, dict(stride_x=-8)), (BAD_ARGUMENT, dict(stride_dsum=-1)), (BAD_ARGUMENT, dict(stride_out=63)),
    (BAD_ARGUMENT, dict(stride_dx=0)), (BAD_ARGUMENT, dict(stride_sum=1)), (BAD_DTYPE, dict(dtype=cabi.FP64)),
    (BAD_DTYPE, dict(dtype_weight=cabi.INT8)), (BAD_DTYPE, dict(dtype_grad=cabi.INT8)), (BAD_DTYPE, dict(dtype_out=7)),
])
def test_norm_plan_refusals(code, args):
    _refused(code, lambda: op.NormPlan(**{**dict(rows=4, cols=64, dtype=cabi.FP32), **args}))


@pytest.mark.parametrize("code,args", [
    (BAD_ARGUMENT, dict(rows=-1)), (BAD_ARGUMENT, dict(cols=0)), (BAD_DTYPE, dict(dtype=cabi.INT8)),
    (BAD_ARGUMENT, dict(stride_x=-1)), (BAD_ARGUMENT, dict(stride_out=63)),
])
def test_quantize_plan_refusals(code, args):
    _refused(code, lambda: op.QuantizePlan(**{**dict(rows=4, cols=64, dtype=cabi.FP32), **args}))


@pytest.mark.parametrize("code,args", [
    (BAD_ARGUMENT, dict(m=-1)), (BAD_ARGUMENT, dict(n=1 << 31)), (BAD_ARGUMENT, dict(k=131072)),
    (BAD_ARGUMENT, dict(k=-1)), (BAD_DTYPE, dict(dtype_out=cabi.FP64)), (BAD_KTYPE, dict(activation=3)),
    (BAD_KTYPE, dict(activation=-1)), (BAD_ARGUMENT, dict(n=63, activation=op.ACT_GATED_SILU)),
    (BAD_ARGUMENT, dict(stride_left=-1)), (BAD_ARGUMENT, dict(stride_out=63)),
    (BAD_ARGUMENT, dict(activation=op.ACT_GATED_SILU, stride_out=31)),
])
def test_contract_int8_plan_refusals(code, args):
    _refused(code, lambda: op.Int8ContractPlan(**{**dict(m=4, n=64, k=64), **args}))


@pytest.mark.parametrize("code,args", [
    (BAD_ARGUMENT, dict(rows=-1)), (BAD_ARGUMENT, dict(vocab=0)), (BAD_ARGUMENT, dict(top=33)),
    (BAD_ARGUMENT, dict(top=-1)), (BAD_ARGUMENT, dict(vocab=4, top=5)), (BAD_DTYPE, dict(dtype=cabi.FP64)),
    (BAD_ARGUMENT, dict(stride_logits=-1)), (BAD_ARGUMENT, dict(stride_dlogits=1)),
])
def test_logprob_plan_refusals(code, args):
    _refused(code, lambda: op.LogprobPlan(**{**dict(rows=4, vocab=64, dtype=cabi.FP32), **args}))


def test_call_refusals():
    """null and misaligned pointers and plans of another kind are refused before anything is launched"""
    a = 1 << 20  # an address that no refused call reads
    norm8 = op.NormPlan(4, 64, cabi.FP32, dtype_out=cabi.INT8)
    _refused(NO_POINTER, lambda: norm8.norm(None, a, scale=a))
    _refused(NO_POINTER, lambda: norm8.norm(a, None, scale=a))
    _refused(NO_POINTER, lambda: norm8.norm(a, a))
    _refused(BAD_ARGUMENT, lambda: norm8.norm(a + 2, a, scale=a))
    _refused(BAD_ARGUMENT, lambda: norm8.norm(a, a, scale=a + 1))
    _refused(NO_POINTER, lambda: norm8.backward(a, a, None, a))
    _refused(NO_POINTER, lambda: norm8.backward(a, a, a, None))
    _refused(BAD_ARGUMENT, lambda: norm8.backward(a, a + 1, a, a))
    quant = op.QuantizePlan(4, 64, cabi.BF16)
    _refused(NO_POINTER, lambda: quant.quantize(a, None, a))
    _refused(NO_POINTER, lambda: quant.quantize(a, a, None))
    _refused(BAD_ARGUMENT, lambda: quant.quantize(a + 1, a, a))
    con = op.Int8ContractPlan(4, 64, 64)
    _refused(NO_POINTER, lambda: con.contract(None, a, a, a, a))
    _refused(NO_POINTER, lambda: con.contract(a, a, a, a, None))
    _refused(BAD_ARGUMENT, lambda: con.contract(a, a, a, a, a + 1))
    _refused(BAD_ARGUMENT, lambda: con.contract(a, a, a + 2, a, a))
    lp = op.LogprobPlan(4, 64, cabi.BF16, top=2)
    _refused(NO_POINTER, lambda: lp.logprob(None, a, a))
    _refused(NO_POINTER, lambda: lp.logprob(a, a, None))
    _refused(NO_POINTER, lambda: lp.logprob(a, None, a))
    _refused(BAD_ARGUMENT, lambda: lp.logprob(a, a + 4, a))
    _refused(NO_POINTER, lambda: lp.backward(a, a, None, a, a))
    _refused(NO_POINTER, lambda: lp.backward(a, a, a, None, a))
    _refused(NO_POINTER, lambda: lp.backward(a, a, a, a, a, dentropy=a))
    for rc in (cabi.lib().eir_quantize(norm8.handle, a, a, a, 0), cabi.lib().eir_norm(None, a, a, a, a, a, a, a, 0),
               cabi.lib().eir_contract(lp.handle, a, a, a, a, 0), cabi.lib().eir_permute(con.handle, a, a, 0)):
        assert rc == BAD_ARGUMENT
    for create in ("eir_norm_plan_create", "eir_quantize_plan_create", "eir_contract_int8_plan_create",
                   "eir_logprob_plan_create"):
        assert getattr(cabi.lib(), create)(None, None) == BAD_ARGUMENT


def test_empty_calls_do_nothing():
    op.NormPlan(0, 64, cabi.FP32).norm(None, None)
    op.QuantizePlan(0, 64, cabi.FP32).quantize(None, None, None)
    op.Int8ContractPlan(0, 64, 64).contract(None, None, None, None, None)
    op.Int8ContractPlan(4, 0, 64).contract(None, None, None, None, None)
    op.LogprobPlan(0, 64, cabi.FP32).logprob(None)
    op.LogprobPlan(0, 64, cabi.FP32).backward(None, None, None, None, None)


def _differences(f, x, step=1e-5):
    """central differences of the scalar f at x (64 bits: error about step^2 + 1e-16 / step)"""
    g = torch.zeros_like(x)
    for i in range(x.numel()):
        y = x.clone().view(-1)
        y[i] += step
        up = f(y.view_as(x))
        y[i] -= 2 * step
        g.view(-1)[i] = (up - f(y.view_as(x))) / (2 * step)
    return g


def test_norm_gradient_formula_against_differences():
    g = torch.Generator().manual_seed(1)
    h, dy, w = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((3, 7), (3, 7), (7,)))
    dsum = torch.randn((3, 7), generator=g, dtype=torch.float64)
    loss = lambda h, w: ((norm64(h, None, w, 1e-3)["y"] * dy).sum() + (h * dsum).sum())
    rstd = norm64(h, None, w, 1e-3)["rstd"]
    dx, dw = norm_backward64(dy, h, w, rstd, dsum)
    assert (dx - _differences(lambda v: loss(v, w), h)).abs().max() < 1e-8
    assert (dw - _differences(lambda v: loss(h, v), w)).abs().max() < 1e-8


def test_logprob_gradient_formula_against_differences():
    g = torch.Generator().manual_seed(2)
    x = torch.randn((4, 9), generator=g, dtype=torch.float64) * 2
    x[1, 3] = -float("inf")
    t = torch.tensor([2, 0, -100, 8])
    dlp, dent = (torch.randn(4, generator=g, dtype=torch.float64) for _ in range(2))

    def loss(x):
        o = logprob64(x, t, 0)
        return (o["logprob"] * dlp + o["entropy"] * dent).sum()

    o = logprob64(x, t, 0)
    dx = logprob_backward64(x, t, o["lse"], o["entropy"], dlp, dent)
    fine = torch.isfinite(x)
    diff = _differences(loss, torch.where(fine, x, -1e9))
    assert (dx - diff)[fine].abs().max() < 1e-8 and dx[~fine].abs().max() == 0
