"""Row operators and the 8-bit contraction on the GPU against 64-bit definitions.

Tolerances, fixed from the arithmetic: u = 2^-24 is the FP32 rounding, 2^-8 the
BF16 one. A row's sum of C terms is off by at most (C / 32 + 16) u of the sum of
their magnitudes (no kernel adds fewer than 32 partial sums, and their tree is
at most 16 deep). The integers of the quantising operators are defined by FP32
operations that round the same way everywhere, so they are equal.
"""
from __future__ import annotations

import pytest
import torch

from einsum_ir_b200 import cabi, operators as op
from tests._operators import contract64, logprob64, logprob_backward64, norm64, norm_backward64, quantized32

pytestmark = pytest.mark.gpu

U, UB = 2.0 ** -24, 2.0 ** -8
CODE = {torch.float32: cabi.FP32, torch.bfloat16: cabi.BF16, torch.int8: cabi.INT8}
F32, BF16 = torch.float32, torch.bfloat16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rows_of(g, rows, cols, dtype, pad=0, offset=0, scale=1.0):
    """[rows, cols] inside a wider buffer, `offset` elements off its start"""
    buf = torch.randn(rows * (cols + pad) + offset + 1, generator=g, device="cuda") * scale
    return buf.to(dtype)[offset:offset + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]


def outside_of(buf, rows, cols, stride, offset):
    """mask of the elements of a flat buffer outside the [rows, cols] view"""
    mask = torch.ones_like(buf, dtype=torch.bool)
    mask[offset:offset + rows * stride].view(rows, stride)[:, :cols] = False
    return mask


def close(got, want, tol):
    """|got - want| <= tol where want is finite, and the same infinities and NaNs elsewhere"""
    got, want = got.double(), want.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    rest = ~fine & ~torch.isnan(want)
    assert torch.equal(got[rest], want[rest])
    tol = tol.expand_as(want) if isinstance(tol, torch.Tensor) else torch.full_like(want, tol)
    off = ((got - want).abs() - tol)[fine]
    assert off.numel() == 0 or off.max() <= 0, off.max()


def round_tol(want, dtype):
    return want.abs() * (UB if dtype == BF16 else U)


SHAPES = [(1, 1), (1, 4096), (3, 7), (5, 64), (33, 1000), (2, 2311), (7, 4096), (300, 512), (4, 16384), (3, 16400),
          (2, 40001), (2500, 136)]
LAYOUTS = [(0, 0), (8, 0), (3, 1)]  # (columns beside the row, elements before the first)


# ---------------------------------------------------------------- norm

@pytest.mark.parametrize("out", ["same", "f32", "int8"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("pad,offset", LAYOUTS)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_norm(cuda, rows, cols, pad, offset, dtype, out):
    g = gen(rows * 31 + cols)
    x = rows_of(g, rows, cols, dtype, pad, offset)
    res = rows_of(g, rows, cols, dtype, pad, offset, 3.0)
    w = rows_of(g, 1, cols, dtype, 0, offset)[0] if cols % 2 else rows_of(g, 1, cols, F32)[0]
    dt_out = {"same": dtype, "f32": F32, "int8": torch.int8}[out]
    ld = cols + pad
    plan = op.NormPlan(rows, cols, CODE[dtype], dtype_weight=CODE[w.dtype], dtype_out=CODE[dt_out], eps=1e-5,
                       stride_x=x.stride(0), stride_residual=res.stride(0), stride_sum=ld, stride_out=ld)
    y = torch.full((rows * ld + offset,), 77, device="cuda", dtype=dt_out)
    s = torch.full((rows * ld + offset,), 77.0, device="cuda", dtype=dtype)
    scale, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    plan.norm(x, y[offset:], weight=w, residual=res, sum=s[offset:], scale=scale, rstd=rstd)
    view = lambda b: b[offset:].view(rows, ld)[:, :cols]
    want = norm64(x, res, w, 1e-5)
    depth = (cols / 32 + 16) * U
    assert torch.equal(view(s), (x.float() + res.float()).to(dtype))
    close(rstd, want["rstd"], want["rstd"] * depth)
    if out == "int8":
        q, m, _ = quantized32((x.float() + res.float()) * w.float())
        assert torch.equal(view(y), q)
        close(scale, m.double() * want["rstd"] / 127, m.double() * want["rstd"] / 127 * (depth + 4 * U))
    else:
        close(view(y), want["y"], want["y"].abs() * (depth + 4 * U) + round_tol(want["y"], dt_out) +
              (x.double().abs() + res.double().abs()) * U * (want["rstd"][:, None] * w.double().abs()))
    for b in (y, s):  # nothing beside the rows is written
        assert (b[outside_of(b, rows, cols, ld, offset)] == 77).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_norm_without_options_and_broadcast_rows(cuda, dtype):
    """no residual, weight or statistics; a row stride of 0 repeats one row"""
    x = rows_of(gen(1), 1, 640, dtype)
    y = torch.empty((9, 640), device="cuda", dtype=dtype)
    op.NormPlan(9, 640, CODE[dtype], eps=0.0, stride_x=0).norm(x, y)
    want = norm64(x, None, None, 0.0)["y"].expand(9, -1)
    close(y, want, want.abs() * 40 * U + round_tol(want, dtype))


@pytest.mark.parametrize("cols", [64, 999, 4096, 20000])
def test_norm_in_place_sum(cuda, cols):
    """the sum over the residual, and over x"""
    g = gen(cols)
    for which in range(2):
        x, res = rows_of(g, 40, cols, BF16), rows_of(g, 40, cols, BF16)
        plan = op.NormPlan(40, cols, cabi.BF16, dtype_out=cabi.INT8)
        h = x.float() + res.float()
        q, scale = torch.empty((40, cols), device="cuda", dtype=torch.int8), torch.empty(40, device="cuda")
        plan.norm(x, q, residual=res, sum=res if which else x, scale=scale)
        assert torch.equal(res if which else x, h.to(BF16))
        assert torch.equal(q, quantized32(h)[0])


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,cols", [(3, 8200), (300, 8193), (2, 57345), (5, 65537), (150, 70000)])
def test_norm_wide_rows(cuda, rows, cols, dtype, offset):
    """rows held in shared memory and rows read twice, in place and not, and their backward pass"""
    g = gen(rows + cols)
    w = rows_of(g, 1, cols, BF16)[0]
    for which in range(3):
        x, res = rows_of(g, rows, cols, dtype, 0, offset), rows_of(g, rows, cols, dtype, 0, offset)
        want = norm64(x, res, w, 1e-5)
        h = x.float() + res.float()
        s = (torch.empty_like(x), x, res)[which]
        q, scale, rstd = (torch.empty((rows, cols), device="cuda", dtype=torch.int8), torch.empty(rows, device="cuda"),
                          torch.empty(rows, device="cuda"))
        op.NormPlan(rows, cols, CODE[dtype], dtype_weight=cabi.BF16, dtype_out=cabi.INT8, eps=1e-5).norm(
            x, q, weight=w, residual=res, sum=s, scale=scale, rstd=rstd)
        assert torch.equal(s, h.to(dtype))
        assert torch.equal(q, quantized32(h * w.float())[0])
        close(rstd, want["rstd"], want["rstd"] * (cols / 32 + 16) * U)
        dy = rows_of(g, rows, cols, dtype, 0, offset)
        dx, dw = torch.empty_like(dy), torch.empty(cols, device="cuda")
        back = dy.clone() if which else dy
        op.NormPlan(rows, cols, CODE[dtype], dtype_weight=cabi.BF16).backward(
            back, s, rstd, back if which else dx, weight=w, dsum=dy, dweight=dw)
        got = back if which else dx
        want_x, want_w = norm_backward64(dy, s, w, rstd, dy)
        r, gd, hd = rstd.double()[:, None], (dy.double() * w.double()).abs(), s.double().abs()
        parts = r * (gd + hd * r.square() * (gd * hd).mean(1, keepdim=True)) + dy.double().abs()
        close(got, want_x, parts * ((cols / 32 + 16) * U) + round_tol(want_x, dtype))
        close(dw, want_w, (dy.double() * hd * r).abs().sum(0) * ((rows + 16) * U))


@pytest.mark.parametrize("cols", [48, 4096, 20001])
def test_norm_special_rows(cuda, cols):
    """zeros, tiny values, infinities and NaN, each in a row of its own"""
    x = rows_of(gen(3), 8, cols, F32)
    x[1] = 0
    x[2] = 1e-32
    x[3, cols // 2] = float("inf")
    x[4, cols - 1] = float("nan")
    x[5, 0] = -float("inf")
    x[6] = 0
    x[6, 7] = -5
    q, scale = torch.empty((8, cols), device="cuda", dtype=torch.int8), torch.empty(8, device="cuda")
    y = torch.empty((8, cols), device="cuda")
    op.NormPlan(8, cols, cabi.FP32, dtype_out=cabi.INT8, eps=1e-6).norm(x, q, scale=scale)
    op.NormPlan(8, cols, cabi.FP32, eps=1e-6).norm(x, y)
    assert torch.equal(q, quantized32(x)[0]) and (q[1:6] == 0).all() and q[6, 7] == -127
    assert scale[1] == 0 and scale[2] == 0 and torch.isnan(scale[3:6]).all() and torch.isfinite(scale[[0, 6, 7]]).all()
    assert torch.isfinite(y[[0, 1, 2, 6, 7]]).all() and torch.isnan(y[4]).all() and torch.isnan(y[3, cols // 2])


@pytest.mark.parametrize("grad", [F32, BF16])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("pad,offset", LAYOUTS)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_norm_backward(cuda, rows, cols, pad, offset, dtype, grad):
    g = gen(rows + cols)
    h = rows_of(g, rows, cols, dtype, pad, offset, 2.0)
    dy, dsum = rows_of(g, rows, cols, grad, pad, offset), rows_of(g, rows, cols, grad, pad, offset)
    w = rows_of(g, 1, cols, dtype)[0]
    rstd = norm64(h, None, None, 1e-5)["rstd"].float()
    ld = cols + pad
    plan = op.NormPlan(rows, cols, CODE[dtype], dtype_grad=CODE[grad], stride_h=h.stride(0), stride_dy=dy.stride(0),
                       stride_dsum=dsum.stride(0), stride_dx=ld)
    dx = torch.full((rows * ld + offset,), 77.0, device="cuda", dtype=grad)
    dw = torch.empty(cols, device="cuda")
    view = dx[offset:].view(rows, ld)[:, :cols]
    for with_sum in (True, False):
        plan.backward(dy, h, rstd, dx[offset:], weight=w, dsum=dsum if with_sum else None, dweight=dw)
        want, want_w = norm_backward64(dy, h, w, rstd, dsum if with_sum else None)
        r, gd, hd = rstd.double()[:, None], (dy.double() * w.double()).abs(), h.double().abs()
        parts = r * (gd + hd * r.square() * (gd * hd).mean(1, keepdim=True)) + (dsum.double().abs() if with_sum else 0)
        close(view, want, parts * ((cols / 32 + 16) * U) + round_tol(want, grad))
        close(dw, want_w, (dy.double() * hd * r).abs().sum(0) * ((rows + 16) * U))
        assert (dx[outside_of(dx, rows, cols, ld, offset)] == 77).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("pad,offset", LAYOUTS)
@pytest.mark.parametrize("cols", [300, 1003, 2048, 4095, 5000])
def test_norm_backward_many_rows(cuda, cols, pad, offset, dtype):
    test_norm_backward(cuda, 4900, cols, pad, offset, dtype, dtype)


def test_norm_backward_in_place_no_options_and_repeats(cuda):
    g = gen(9)
    h, dy = rows_of(g, 1500, 777, BF16), rows_of(g, 1500, 777, BF16)
    rstd = norm64(h, None, None, 1e-5)["rstd"].float()
    plan = op.NormPlan(1500, 777, cabi.BF16)
    a, b, dw, dw2 = torch.empty_like(dy), torch.empty_like(dy), torch.empty(777, device="cuda"), torch.empty(777, device="cuda")
    plan.backward(dy, h, rstd, a)
    plan.backward(dy, h, rstd, b, dweight=dw)
    plan.backward(dy, h, rstd, b, dweight=dw2)
    assert torch.equal(dw, dw2) and torch.equal(a, b)  # a fixed order of the sum
    c = dy.clone()
    plan.backward(c, h, rstd, c, dsum=None)
    assert torch.equal(a, c)
    z = torch.full((64,), 5.0, device="cuda")
    op.NormPlan(0, 64, cabi.BF16).backward(None, None, None, None, dweight=z)
    assert (z == 0).all()


def test_norm_backward_gradients_chain_to_autograd(cuda):
    """the forward's sum and rstd through the backward pass give the gradients of the whole expression"""
    g = gen(4)
    x, res = (rows_of(g, 17, 300, F32).double().requires_grad_() for _ in range(2))
    w = torch.randn(300, generator=g, device="cuda", dtype=torch.float64).requires_grad_()
    dy, dh = rows_of(g, 17, 300, F32), rows_of(g, 17, 300, F32)
    h = x + res
    y = h / (h.square().mean(1, keepdim=True) + 1e-5).sqrt() * w
    torch.autograd.backward([y, h], [dy.double(), dh.double()])
    plan = op.NormPlan(17, 300, cabi.FP32, eps=1e-5)
    out, s, rstd = torch.empty((17, 300), device="cuda"), torch.empty((17, 300), device="cuda"), torch.empty(17, device="cuda")
    w32 = w.detach().float()
    plan.norm(x.detach().float(), out, weight=w32, residual=res.detach().float(), sum=s, rstd=rstd)
    dx, dw = torch.empty_like(out), torch.empty(300, device="cuda")
    plan.backward(dy, s, rstd, dx, weight=w32, dsum=dh, dweight=dw)
    # every operand is off by a few u of terms of order ten at most
    close(dx, x.grad, 10 * 100 * U)
    close(dw, w.grad, 17 * 10 * 100 * U)
    assert torch.equal(x.grad, res.grad)


# ---------------------------------------------------------------- quantize

@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("pad,offset", LAYOUTS)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize(cuda, rows, cols, pad, offset, dtype):
    x = rows_of(gen(cols), rows, cols, dtype, pad, offset)
    ld = cols + pad
    q = torch.full((rows * ld + offset,), 99, device="cuda", dtype=torch.int8)
    scale = torch.empty(rows, device="cuda")
    op.QuantizePlan(rows, cols, CODE[dtype], stride_x=x.stride(0), stride_out=ld).quantize(x, q[offset:], scale)
    want, m, _ = quantized32(x)
    got = q[offset:].view(rows, ld)[:, :cols]
    assert torch.equal(got, want) and torch.equal(scale, (m.double() / 127).float())
    assert (q[outside_of(q, rows, cols, ld, offset)] == 99).all()
    # half an integer step, and the rounding of the factor and the product (|q| <= 127)
    close(got.double() * scale.double()[:, None], x, (m.double() / 127 * (0.5 + 127 * 3 * U))[:, None])


@pytest.mark.parametrize("cols", [40, 4096, 30001])
def test_quantize_special_rows(cuda, cols):
    x = rows_of(gen(2), 6, cols, BF16)
    x[0] = 0
    x[1, 5] = float("nan")
    x[2, cols - 1] = -float("inf")
    x[3] = 3e38
    x[4] = 1e-31
    q, scale = torch.empty((6, cols), device="cuda", dtype=torch.int8), torch.empty(6, device="cuda")
    op.QuantizePlan(6, cols, cabi.BF16).quantize(x, q, scale)
    assert torch.equal(q, quantized32(x)[0])
    assert scale[0] == 0 and scale[4] == 0 and torch.isnan(scale[1:3]).all() and (q[3] == 127).all()


# ---------------------------------------------------------------- 8-bit contraction

def codes(g, rows, k, stride=None, offset=0):
    ld = k if stride is None else stride
    b = torch.randint(-128, 128, (rows * ld + offset + 1,), generator=g, device="cuda").to(torch.int8)
    return b[offset:offset + rows * ld].view(rows, ld)[:, :k]


def contract_case(m, n, k, act, out, bias=True, scales=True, ld=None, offset=0, seed=0, stream=None):
    g = gen(m * 7 + n * 3 + k + seed)
    a, b = codes(g, m, k, ld, offset), codes(g, n, k, ld, offset)
    rand = lambda c: torch.rand(c, generator=g, device="cuda")
    # products of order one, so that the gated activation bends
    sa, sb = ((rand(m) + 0.5) * 2 ** -7, (rand(n) + 0.5) * 2 ** -6 / max(1, k) ** 0.5) if scales else (None, None)
    bv = (rand(n) - 0.5 if scales else torch.randint(-9, 9, (n,), generator=g, device="cuda").float()) if bias else None
    n_out = n // 2 if act == op.ACT_GATED_SILU else n
    pad = 5
    y = torch.full((m, n_out + pad), 77.0, device="cuda", dtype=out)
    plan = op.Int8ContractPlan(m, n, k, dtype_out=CODE[out], activation=act, stride_left=a.stride(0),
                               stride_right=b.stride(0), stride_out=n_out + pad)
    if stream is not None:
        stream.wait_stream(torch.cuda.current_stream())
    plan.contract(a, b, sa, sb, y, bias=bv, stream=stream.cuda_stream if stream is not None else 0)
    torch.cuda.synchronize()
    cabi.check_device_errors()
    want = contract64(a, b, sa, sb, bv, act)
    z = contract64(a, b, sa, sb, None, 0).abs() + (bv.double().abs() if bias else 0)
    if act == op.ACT_GATED_SILU:
        # z is off by 5 u |z|; silu's slope is below 1.1 and silu(z) <= |z|; exp, sum and quotient add 8 u
        zg, zv = z.chunk(2, 1)
        tol = 5 * U * (1.1 * zg * zv + zg * zv) + (zg * zv) * (8 + zg) * U
    else:
        tol = 5 * U * z
    close(y[:, :n_out], want, tol + round_tol(want, out))
    assert (y[:, n_out:] == 77).all()
    return plan


ACTS = [op.ACT_NONE, op.ACT_RELU, op.ACT_GATED_SILU]


@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,n,k", [(1, 2, 1), (1, 4096, 4096), (1, 1000, 333), (2, 66, 64), (5, 130, 100), (16, 256, 512),
                                   (17, 514, 1024), (33, 2050, 2048), (64, 128, 16), (77, 1022, 496), (128, 512, 4096),
                                   (129, 258, 160), (300, 1000, 640), (513, 770, 1040), (1000, 384, 8192), (2049, 2306, 128)])
def test_contract_int8(cuda, m, n, k, act, out):
    contract_case(m, n, k, act, out)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m", [15, 31, 32, 63, 65, 79, 80, 81, 96, 97, 127])
@pytest.mark.parametrize("n,k", [(200, 256), (262, 2100), (40000, 130)])
def test_contract_int8_token_tiles(cuda, n, k, m, act):
    contract_case(m, n, k, act, BF16)


@pytest.mark.parametrize("m", [1, 3, 40, 300])
@pytest.mark.parametrize("ld,offset", [(544, 0), (513, 0), (512, 1), (528, 16), (520, 8)])
def test_contract_int8_strides_and_alignment(cuda, m, ld, offset):
    contract_case(m, 390, 512, op.ACT_RELU, F32, ld=ld, offset=offset)
    contract_case(m, 390, 512, op.ACT_GATED_SILU, BF16, ld=ld, offset=offset)


@pytest.mark.parametrize("m,n,k", [(1, 64, 131071), (3, 300, 131056), (140, 300, 131071), (260, 260, 131056)])
def test_contract_int8_extremes(cuda, m, n, k):
    """the largest sums: every product 16384, exact in 32 bits and rounded once to FP32"""
    a = torch.full((m, k), -128, device="cuda", dtype=torch.int8)
    b = torch.full((n, k), -128, device="cuda", dtype=torch.int8)
    b[1::2] = 127
    y = torch.empty((m, n), device="cuda")
    op.Int8ContractPlan(m, n, k, dtype_out=cabi.FP32).contract(a, b, None, None, y)
    assert (y[:, 0::2] == float(torch.tensor(k * 16384, dtype=torch.float32))).all()
    assert (y[:, 1::2] == float(torch.tensor(-k * 16256, dtype=torch.float32))).all()


@pytest.mark.parametrize("m,n,k", [(1, 100, 96), (50, 100, 96), (400, 300, 96)])
def test_contract_int8_options(cuda, m, n, k):
    contract_case(m, n, k, op.ACT_NONE, F32, bias=False, scales=False)
    contract_case(m, n, k, op.ACT_NONE, F32, bias=True, scales=False)
    contract_case(m, n, k, op.ACT_RELU, BF16, bias=False)
    contract_case(m, n, k, op.ACT_GATED_SILU, F32, bias=False)


@pytest.mark.parametrize("m", [2, 200])
def test_contract_int8_empty_sum_broadcast_and_nan(cuda, m):
    """k = 0 leaves the bias; a row stride of 0 repeats a token; a token's NaN scale stays in its row"""
    bias = torch.randn(64, device="cuda")
    y = torch.empty((m, 64), device="cuda")
    op.Int8ContractPlan(m, 64, 0, dtype_out=cabi.FP32, activation=op.ACT_RELU).contract(None, None, None, None, y, bias=bias)
    assert torch.equal(y, torch.relu(bias).expand(m, -1))
    g = gen(m)
    a, b = codes(g, 1, 160), codes(g, 64, 160)
    sa = torch.ones(m, device="cuda")
    sa[1] = float("nan")
    op.Int8ContractPlan(m, 64, 160, dtype_out=cabi.FP32, activation=op.ACT_RELU, stride_left=0).contract(a, b, sa, None, y)
    want = torch.relu(contract64(a, b, None, None, None, 0)).float().expand(m, -1)
    assert torch.isnan(y[1]).all() and torch.equal(y[0], want[0]) and torch.equal(y[2:], want[2:])


@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,n", [(1, 2), (33, 130), (3001, 2050)])
def test_contract_int8_no_sum(cuda, m, n, act, out):
    """k = 0: scales, bias and activation alone"""
    contract_case(m, n, 0, act, out)


def test_contract_int8_other_stream_and_reuse(cuda):
    s = torch.cuda.Stream()
    for m in (1, 24, 300):
        plan = contract_case(m, 600, 1536, op.ACT_RELU, BF16, stream=s)
        assert plan.describe().startswith("int8")
        contract_case(m, 600, 1530, op.ACT_RELU, BF16, stream=s)


# ---------------------------------------------------------------- log probabilities

def logits_of(g, rows, vocab, dtype, pad=0, offset=0):
    x = rows_of(g, rows, vocab, dtype, pad, offset, 3.0)
    if vocab > 8:
        x[:, torch.randint(vocab, (max(1, vocab // 50),), generator=g, device="cuda")] = -float("inf")
    return x


def check_logprob(x, t, top, outs):
    want = logprob64(x, t, top)
    v = x.shape[1]
    # lse: the sum of positive terms and the logarithm; x - lse: one more rounding of each
    fin = torch.where(torch.isfinite(want["lse"]), want["lse"].abs(), 0.0)
    xm = torch.where(torch.isfinite(x), x.double().abs(), 0.0).amax(1)
    tol = (v / 32 + 48 + 4 * xm) * U + 4 * (fin + xm) * U
    close(outs["lse"], want["lse"], tol)
    if t is not None:
        close(outs["logprob"], want["logprob"], 2 * tol)
    # U / S: terms p |x - m| of one sign, each off like p
    close(outs["entropy"], want["entropy"], tol * (4 + 2 * xm))
    if top:
        assert torch.equal(outs["top_index"], want["top_index"])
        close(outs["top_logprob"], want["top_logprob"], (2 * tol)[:, None])


def run_logprob(x, t, top, stream=0):
    rows, v = x.shape
    e = lambda *s, d=F32: torch.full(s, 55, device="cuda", dtype=d)
    o = {"lse": e(rows), "entropy": e(rows), "logprob": e(rows) if t is not None else None}
    o |= {"top_logprob": e(rows, top), "top_index": e(rows, top, d=torch.int64)} if top else {}
    op.LogprobPlan(rows, v, CODE[x.dtype], top=top, stride_logits=x.stride(0)).logprob(
        x, t, o["logprob"], entropy=o["entropy"], lse=o["lse"], top_logprob=o.get("top_logprob"),
        top_index=o.get("top_index"), stream=stream)
    return o


VOCABS = [(1, 1), (3, 2), (2, 33), (5, 1000), (7, 4097), (1, 32768), (3, 131072), (700, 517), (2, 200003), (900, 2048)]


@pytest.mark.parametrize("top", [0, 1, 5, 32])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("pad,offset", LAYOUTS)
@pytest.mark.parametrize("rows,vocab", VOCABS)
def test_logprob(cuda, rows, vocab, pad, offset, dtype, top):
    top = min(top, vocab)
    g = gen(rows + vocab + top)
    x = logits_of(g, rows, vocab, dtype, pad, offset)
    t = torch.randint(vocab, (rows,), generator=g, device="cuda")
    t[3::4] = -100
    check_logprob(x, t, top, run_logprob(x, t, top))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [40, 2048, 50021])
def test_logprob_ties(cuda, dtype, vocab):
    """equal logits, both zeros, sorted both ways: the lowest indices come first"""
    x = torch.zeros((6, vocab), device="cuda", dtype=dtype)
    x[0, 1::2] = -0.0
    x[1] = 1.5
    x[2] = torch.arange(vocab, device="cuda").float()
    x[3] = -torch.arange(vocab, device="cuda").float()
    x[4] = (torch.arange(vocab, device="cuda") % 7).float()
    x[5, vocab - 3:] = 2
    for top in (1, 8, 32):
        o = run_logprob(x, None, top)
        assert torch.equal(o["top_index"], logprob64(x, None, top)["top_index"])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [50, 3000, 70000])
def test_logprob_special_rows(cuda, dtype, vocab):
    """nothing allowed, one token allowed, the type's lowest value as a mask, NaN, +infinity, targets off the row"""
    x = logits_of(gen(vocab), 9, vocab, dtype)
    x[0] = -float("inf")
    x[1] = -float("inf")
    x[1, vocab - 2] = 4.0
    x[2] = torch.finfo(dtype).min
    x[2, 3] = 1.0
    x[3] = torch.finfo(dtype).min
    x[4, vocab // 2] = float("nan")
    x[5, 7] = float("inf")
    t = torch.tensor([1, vocab - 2, 3, 0, 2, 2, vocab, -1, (1 << 40)], device="cuda")
    o = run_logprob(x, t, 4)
    assert torch.isnan(o["lse"][4:6]).all() and torch.isnan(o["entropy"][4:6]).all() and torch.isnan(o["logprob"][4:6]).all()
    assert o["top_index"][4, 0] == vocab // 2 and o["top_index"][5, 0] == 7
    assert torch.isnan(o["logprob"][6]) and o["logprob"][7] == 0 and torch.isnan(o["logprob"][8])
    assert o["lse"][0] == -float("inf") and o["logprob"][0] == -float("inf") and o["entropy"][0] == 0
    assert o["lse"][1] == 4 and o["logprob"][1] == 0 and o["entropy"][1] == 0 and o["top_index"][1, 0] == vocab - 2
    assert o["lse"][2] == 1 and o["logprob"][2] == 0 and o["entropy"][2] == 0
    assert torch.equal(o["top_index"][0], torch.arange(4, device="cuda"))
    for row in (0, 1, 2):
        want = logprob64(x[row:row + 1], t[row:row + 1], 4)
        assert torch.equal(o["top_index"][row], want["top_index"][0])
        close(o["top_logprob"][row], want["top_logprob"][0], 64 * U * torch.nan_to_num(want["top_logprob"][0]).abs() + 64 * U)
    # equal logits at the lowest value: a uniform row, within the roundings of log V
    assert abs(o["entropy"][3].item() - float(torch.log(torch.tensor(float(vocab))))) < (vocab / 32 + 64) * 12 * U


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("pad,offset", LAYOUTS)
@pytest.mark.parametrize("rows,vocab", VOCABS)
def test_logprob_backward(cuda, rows, vocab, pad, offset, dtype):
    g = gen(rows + 2 * vocab)
    x = logits_of(g, rows, vocab, dtype, pad, offset)
    t = torch.randint(vocab, (rows,), generator=g, device="cuda")
    t[3::4] = -7
    o = logprob64(x, t, 0)
    lse, ent = o["lse"].float(), o["entropy"].float()
    dlp, dent = (torch.randn(rows, generator=g, device="cuda") for _ in range(2))
    ld = vocab + pad
    plan = op.LogprobPlan(rows, vocab, CODE[dtype], stride_logits=x.stride(0), stride_dlogits=ld)
    dx = torch.full((rows * ld + offset,), 77.0, device="cuda", dtype=dtype)
    view = dx[offset:].view(rows, ld)[:, :vocab]
    d = torch.where(o["p"] > 0, x.double() - lse.double()[:, None], 0.0).abs()
    for use_t, use_e in ((True, True), (True, False), (False, True)):
        plan.backward(x, t if use_t else None, lse, dlp if use_t else None, dx[offset:], entropy=ent if use_e else None,
                      dentropy=dent if use_e else None)
        want = logprob_backward64(x, t if use_t else None, lse, ent, dlp, dent if use_e else None)
        # p is off by the rounding of x - lse and of its exponential
        size = (dlp.double().abs()[:, None] * (o["p"] + (d == d)) if use_t else 0) + \
            (dent.double().abs()[:, None] * o["p"] * (d + ent.double()[:, None] + 1) if use_e else 0)
        close(view, want, size * (16 + 4 * d) * U + round_tol(want, dtype))
        assert (dx[outside_of(dx, rows, vocab, ld, offset)] == 77).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [2, 400])
@pytest.mark.parametrize("step", [1, 4, 8, 128, 512, 1024, 2048, 4096, 8192])
def test_logprob_alternatives_at_a_distance(cuda, step, rows, dtype):
    """the most likely tokens `step` apart, so that threads, warps and chunks hold several of them"""
    g = gen(step)
    x = logits_of(g, rows, 70000, dtype)
    for r in range(rows):
        at = (r * 37 + step * torch.arange(8, device="cuda")) % 70000
        x[r, at] = 40 - torch.randperm(8, generator=g, device="cuda").to(dtype) // 2  # (pairs are ties)
    t = torch.randint(70000, (rows,), generator=g, device="cuda")
    check_logprob(x, t, 8, run_logprob(x, t, 8))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab", [(2, 6528), (74, 4736), (568, 3136), (96, 6117), (30, 10007), (9, 24001), (1, 1500)])
def test_logprob_backward_every_target(cuda, rows, vocab, dtype):
    """targets spread over the whole row: the one-hot term lands in its column whatever thread holds it"""
    g = gen(rows)
    x = rows_of(g, rows, vocab, dtype)
    t = torch.linspace(0, vocab - 1, rows, device="cuda").round().long()
    lse = torch.logsumexp(x.double(), 1).float()
    dlp = torch.full((rows,), 2.0, device="cuda")
    dx = torch.empty_like(x)
    op.LogprobPlan(rows, vocab, CODE[dtype]).backward(x, t, lse, dlp, dx)
    want = logprob_backward64(x, t, lse, None, dlp, None)
    close(dx, want, 64 * U + round_tol(want, dtype))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_logprob_backward_special_rows_and_in_place(cuda, dtype):
    vocab = 1203
    x = logits_of(gen(6), 6, vocab, dtype)
    x[0] = -float("inf")
    x[1, 5] = -float("inf")
    t = torch.tensor([3, 5, vocab, -1, 0, 7], device="cuda")
    o = run_logprob(x, t, 0)
    dlp, dent = torch.ones(6, device="cuda"), torch.ones(6, device="cuda")
    plan = op.LogprobPlan(6, vocab, CODE[dtype])
    dx = torch.empty_like(x)
    plan.backward(x, t, o["lse"], dlp, dx, entropy=o["entropy"], dentropy=dent)
    assert (dx[0] == 0).all()
    assert abs(dx[1, 5].item() - 1) < 1e-6 and torch.isfinite(dx[1]).all()  # a ruled-out target still pulls
    assert torch.isnan(dx[2]).all()
    y = x.clone()
    plan.backward(y, t, o["lse"], dlp, y, entropy=o["entropy"], dentropy=dent)
    assert torch.equal(torch.nan_to_num(y, 9.0), torch.nan_to_num(dx, 9.0))


def test_row_operators_on_another_stream(cuda):
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        x = rows_of(gen(8), 200, 3000, BF16)
        t = torch.zeros(200, device="cuda", dtype=torch.int64)
        o = run_logprob(x, t, 3, stream=s.cuda_stream)
        q, scale = torch.empty((200, 3000), device="cuda", dtype=torch.int8), torch.empty(200, device="cuda")
        op.QuantizePlan(200, 3000, cabi.BF16).quantize(x, q, scale, stream=s.cuda_stream)
    s.synchronize()
    check_logprob(x, t, 3, o)
    assert torch.equal(q, quantized32(x)[0])


@pytest.mark.parametrize("case", range(6))
def test_repeats_are_equal(cuda, case):
    """the same call many times, the GPU full of blocks: bit for bit the same, and right"""
    g = gen(case)
    if case < 3:
        rows, vocab, dtype = [(2144, 9920, BF16), (3000, 5000, F32), (1200, 30011, BF16)][case]
        x = rows_of(g, rows, vocab, dtype, scale=3.0)
        first = run_logprob(x, None, 8)
        check_logprob(x, None, 8, first)
        again = lambda: run_logprob(x, None, 8)
    elif case < 5:
        rows, cols, dtype = [(3000, 4096, BF16), (2500, 2311, F32)][case - 3]
        h, dy = rows_of(g, rows, cols, dtype, 1), rows_of(g, rows, cols, dtype, 8)
        rstd = norm64(h, None, None, 1e-5)["rstd"].float()
        plan = op.NormPlan(rows, cols, CODE[dtype], dtype_out=cabi.INT8, stride_x=cols + 1, stride_dy=cols + 8)

        def again():
            o = {"dx": torch.empty((rows, cols), device="cuda", dtype=dtype), "dw": torch.empty(cols, device="cuda"),
                 "q": torch.empty((rows, cols), device="cuda", dtype=torch.int8), "scale": torch.empty(rows, device="cuda")}
            plan.norm(h, o["q"], scale=o["scale"])
            plan.backward(dy, h, rstd, o["dx"], dweight=o["dw"])
            return o
        first = again()
        assert torch.equal(first["q"], quantized32(h)[0])
    else:
        a, b = codes(g, 300, 2000), codes(g, 1500, 2000)
        plan = op.Int8ContractPlan(300, 1500, 2000, dtype_out=cabi.FP32)

        def again():
            y = torch.empty((300, 1500), device="cuda")
            plan.contract(a, b, None, None, y)
            return {"y": y}
        first = again()
        assert torch.equal(first["y"].double(), contract64(a, b, None, None, None, 0).float().double())
    for _ in range(60):
        for k, v in again().items():
            assert v is None or torch.equal(v, first[k]), k


def test_workspaces_over_streams(cuda):
    """calls of one plan on two streams share its workspace in turn"""
    g = gen(11)
    rows, cols, m, n, k = 700, 1500, 300, 520, 1023
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    norm, product = op.NormPlan(rows, cols, cabi.FP32), op.Int8ContractPlan(m, n, k, dtype_out=cabi.FP32)
    rstd = torch.rand(rows, generator=g, device="cuda") + 0.5
    h = torch.randn(rows, cols, generator=g, device="cuda")
    dy = [torch.randn(rows, cols, generator=g, device="cuda") for _ in range(2)]
    b = codes(g, n, k)
    a = [codes(g, m, k) for _ in range(2)]
    dw = [torch.empty(cols, device="cuda") for _ in range(20)]
    y = [torch.empty(m, n, device="cuda") for _ in range(20)]
    dx = torch.empty(2, rows, cols, device="cuda")
    torch.cuda.synchronize()
    for i in range(20):
        s = streams[i % 2].cuda_stream
        norm.backward(dy[i % 2], h, rstd, dx[i % 2], dweight=dw[i], stream=s)
        product.contract(a[i % 2], b, None, None, y[i], stream=s)
    torch.cuda.synchronize()
    cabi.check_device_errors()
    for i in range(2):
        exact = contract64(a[i], b, None, None, None, 0).float()
        want = (dy[i].double() * h.double() * rstd.double()[:, None]).sum(0)
        assert all(torch.equal(v, exact) for v in y[i::2]) and all(torch.equal(v, dw[i]) for v in dw[i::2])
        # a product's two roundings and the order of `rows` sums
        close(dw[i], want, (rows + 3) * U * (dy[i].double() * h.double() * rstd.double()[:, None]).abs().sum(0))


def test_workspaces_in_a_capture(cuda):
    """a first call that needs memory is refused in a capture; one after it is captured and replayed"""
    contract_case(2, 16, 32, op.ACT_NONE, F32)  # the device's own state exists
    g = gen(12)
    a, b = codes(g, 300, 1023), codes(g, 520, 1023)
    y = torch.empty(300, 520, device="cuda")
    plan = op.Int8ContractPlan(300, 520, 1023, dtype_out=cabi.FP32)
    exact = contract64(a, b, None, None, None, 0).float()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        y.zero_()
        with pytest.raises(cabi.EirError):
            plan.contract(a, b, None, None, y, stream=stream.cuda_stream)
    plan.contract(a, b, None, None, y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        plan.contract(a, b, None, None, y, stream=stream.cuda_stream)
    y.zero_()
    graph.replay()
    torch.cuda.synchronize()
    cabi.check_device_errors()
    assert torch.equal(y, exact)
    del graph
