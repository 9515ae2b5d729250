"""Log probabilities of rows with large finite logits: whole rows at a constant, a finite
constant as the mask, single large logits. Against the 64-bit definition of the row less
its maximum (which leaves probabilities as they are; 64 bits would lose log V beside 1e30).

Tolerances, fixed from the arithmetic (u = 2^-24): the sum of `vocab` positive terms and
its logarithm (V / 32 + 48) u and 4 u log V; a term's exponent is off by at most 4 u of
itself, and terms more than 104 below the maximum are 0 in FP32; a difference of two
logits rounds once, log-sum-exp in four steps.
"""
from __future__ import annotations

import math

import pytest
import torch

from tests._operators import logprob64
from tests.test_gpu_operators import BF16, F32, U, close, gen, run_logprob

pytestmark = pytest.mark.gpu

LARGE = [65504.0, 2.0 ** 20, 1e7, 2.0 ** 23, 2.0 ** 24 + 2, 1e9, 3e9, 1e10, 1e12, 1e15, 1e20, 1e30, 1e36, 1e37, 3e38]


def check_shifted(x, t, top, o):
    v = x.shape[1]
    m = x.double().amax(1, keepdim=True)
    shifted = torch.where(torch.isneginf(x), -torch.inf, x.double() - m)
    want = logprob64(shifted, t, 0)
    spread = torch.where(shifted < -104, 0.0, -shifted).amax(1)
    tol = (v / 32 + 48 + 4 * spread + 4 * math.log(v)) * U
    lse = m[:, 0] + want["lse"]
    close(o["lse"], lse, tol + 4 * U * lse.abs())
    close(o["logprob"], want["logprob"], tol + 4 * U * torch.nan_to_num(want["logprob"], neginf=0.0).abs())
    close(o["entropy"], want["entropy"], tol * (4 + 2 * spread))
    if top:
        at = logprob64(x, None, top)["top_index"]  # the order of the logits themselves
        top_logprob = (shifted - want["lse"][:, None]).gather(1, at)
        assert torch.equal(o["top_index"], at)
        close(o["top_logprob"], top_logprob, tol[:, None] + 4 * U * torch.nan_to_num(top_logprob, neginf=0.0).abs())


# one block and few threads a row, one block, clusters
SHAPES = [(700, 40), (4, 3000), (2, 33333), (2, 140000)]


@pytest.mark.parametrize("top", [0, 5])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab", SHAPES)
def test_rows_at_a_constant(cuda, rows, vocab, dtype, top):
    """nothing but one large value, of either sign, with and without ruled-out logits"""
    t = torch.arange(rows, device="cuda") % vocab
    for c in LARGE:
        for sign in (-1, 1):
            x = torch.full((rows, vocab), sign * c, device="cuda").to(dtype)
            x[1::2, 2::3] = -float("inf")
            check_shifted(x, t, top, run_logprob(x, t, top))


@pytest.mark.parametrize("top", [0, 5])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab", SHAPES)
def test_finite_masks(cuda, rows, vocab, dtype, top):
    """ordinary logits beside masked ones: the first half of the row, scattered ones, all but one"""
    g = gen(rows + vocab)
    values = (torch.randn((rows, vocab), generator=g, device="cuda") * 3).to(dtype)
    t = torch.randint(vocab, (rows,), generator=g, device="cuda")
    for c in LARGE:
        x = values.clone()
        x[0::3, : vocab // 2] = -c
        x[1::3, ::2] = -c
        x[2::3, torch.arange(vocab, device="cuda") != vocab - 2] = -c
        check_shifted(x, t, top, run_logprob(x, t, top))


@pytest.mark.parametrize("top", [0, 5])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab", SHAPES)
def test_single_large_logits(cuda, rows, vocab, dtype, top):
    """one logit, and two a little apart, far above the others"""
    g = gen(rows + vocab + 1)
    values = (torch.randn((rows, vocab), generator=g, device="cuda") * 3).to(dtype)
    t = torch.randint(vocab, (rows,), generator=g, device="cuda")
    for c in LARGE:
        x = values.clone()
        x[:, vocab // 3] = c
        x[1::2, vocab - 1] = torch.tensor(c, device="cuda", dtype=dtype) * 0.9921875
        t[0] = vocab // 3
        check_shifted(x, t, top, run_logprob(x, t, top))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [300, 140000])
def test_mixed_masks(cuda, vocab, dtype):
    """several masks in one row, each below the next, and the lowest value beside -infinity"""
    x = torch.full((3, vocab), -1e30, device="cuda").to(dtype)
    x[:, ::5] = torch.finfo(dtype).min
    x[:, 1::5] = -1e9
    x[:, 2::5] = -float("inf")
    x[1, 7] = -3.0
    x[2, ::5] = -1e37
    x[2, 1::5] = -float("inf")
    x[2, 3::5] = torch.finfo(dtype).min
    x[2, 4::5] = torch.finfo(dtype).min
    t = torch.tensor([1, 0, 5], device="cuda")
    check_shifted(x, t, 4, run_logprob(x, t, 4))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [300, 140000])
def test_nan_and_infinity_beside_large_logits(cuda, vocab, dtype):
    """a NaN or +infinity in a row of large values makes its results NaN, and leads the alternatives"""
    x = torch.full((4, vocab), -1e30, device="cuda").to(dtype)
    x[0, vocab // 2] = float("nan")
    x[1, 7] = float("inf")
    x[2] = 1e30
    x[2, vocab - 1] = float("nan")
    x[3, 3] = 5e5
    t = torch.full((4,), 3, device="cuda")
    o = run_logprob(x, t, 3)
    for name in ("lse", "entropy", "logprob", "top_logprob"):
        assert torch.isnan(o[name][:3]).all(), name
    assert o["top_index"][:3, 0].tolist() == [vocab // 2, 7, vocab - 1]
    check_shifted(x[3:], t[3:], 3, {k: v[3:] for k, v in o.items()})
