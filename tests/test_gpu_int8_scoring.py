"""The 8-bit scoring example end to end: against FP32, and its gradient against differences of its loss."""
from __future__ import annotations

import pytest
import torch

from einsum_ir_b200 import int8_scoring

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,width,hidden,layers,vocab", [(1, 256, 512, 1, 1000), (37, 256, 500, 2, 5003),
                                                              (300, 512, 1024, 2, 8192)])
def test_scores_against_fp32(cuda, tokens, width, hidden, layers, vocab):
    m = int8_scoring.Model(tokens, width, hidden, layers, vocab, top=4)
    g = torch.Generator(device="cuda").manual_seed(3)
    h = torch.randn((tokens, width), generator=g, device="cuda").to(torch.bfloat16)
    targets = torch.randint(vocab, (tokens,), generator=g, device="cuda")
    want, got = m.score_float(h, targets), m.score(h, targets)
    # an 8-bit product is off by about one in 127 sqrt(3) of its rms a factor (8 products a layer's worth
    # of factors here): a logit of rms 1 by a few hundredths, its log probability by twice that at most on average
    assert (got - want).abs().mean() < 0.1
    assert torch.isfinite(m.entropy).all() and (m.top_logprob[:, :1] >= m.top_logprob).all()


def test_training_lowers_the_loss_and_follows_the_formula(cuda):
    out = int8_scoring.main("--tokens 200 --width 256 --hidden 512 --layers 1 --vocab 3001 --steps 4".split())
    assert out["losses"] == sorted(out["losses"], reverse=True) and out["losses"][-1] < out["losses"][0]
    m = out["model"]
    targets = torch.randint(3001, (200,), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    h = torch.randn((200, 256), generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").to(torch.bfloat16)
    m.score(h, targets)
    # the gradient through the float form of what the integers stand for
    x = m.stream_out.double()
    w = m.final.double().requires_grad_()
    logits = (x * m.rstd.double()[:, None] * w) @ m.head_bf16.double().T
    torch.log_softmax(logits, 1).gather(1, targets[:, None]).mean().backward()
    got = m.gradient(targets, torch.full((200,), 1 / 200, device="cuda"))
    # 8-bit activations and BF16 logits and gradients: a few parts in a hundred
    assert (got.double() - w.grad).norm() < 0.05 * w.grad.norm()
