"""Scoring tokens with feed-forward layers in 8-bit integers, and training a norm
weight through the score: the row operators, the 8-bit contraction and the
framework's BF16 contraction together.

    python -m einsum_ir_b200.int8_scoring [--tokens T] [--width C] [--hidden F]
        [--layers L] [--vocab V] [--top K] [--steps S]

A layer is h += down(silu(gate(norm(h))) * up(norm(h))): the norm adds the last
layer's output to the residual stream and writes 8-bit rows, one contraction
computes gate, up and their product, its rows are quantised, and a second
contraction leads back to the width. After the last layer the norm's 8-bit rows meet the
vocabulary, and the log probabilities of the targets are read off the logits. The
weights are random; quantised once, one scale a channel.

A training step takes the gradient of the mean log probability: the logits'
gradient, back through the head by an ordinary BF16 contraction with the
dequantised weight (the head is frozen), and through the final norm to its weight.
"""
from __future__ import annotations

import argparse

import torch

from . import binary, cabi
from . import operators as op


def quantized(weight):
    """rows of a float matrix as 8-bit integers and their scales"""
    rows, cols = weight.shape
    code = {torch.float32: cabi.FP32, torch.bfloat16: cabi.BF16}[weight.dtype]
    q = torch.empty((rows, cols), device=weight.device, dtype=torch.int8)
    scale = torch.empty(rows, device=weight.device)
    op.QuantizePlan(rows, cols, code, stride_x=weight.stride(0)).quantize(weight, q, scale)
    return q, scale


class Model:
    """The weights, quantised, and the plans and buffers for a batch of `tokens` rows."""

    def __init__(self, tokens, width, hidden, layers, vocab, top=0, device="cuda", seed=0):
        g = torch.Generator(device=device).manual_seed(seed)
        rand = lambda *s: torch.randn(s, generator=g, device=device)
        bf16 = torch.bfloat16
        self.tokens, self.width, self.vocab = tokens, width, vocab
        self.weights = []  # as floats, for comparison
        self.layers = []
        for _ in range(layers):
            gate_up, down = rand(2 * hidden, width) * width ** -0.5, rand(width, hidden) * hidden ** -0.5
            norm = (1 + 0.1 * rand(width)).to(bf16)
            self.weights.append((norm, gate_up, down))
            self.layers.append((norm, *quantized(gate_up), *quantized(down)))
        head = rand(vocab, width) * width ** -0.5
        self.head_float = head
        self.head, self.head_scale = quantized(head)
        # the head that the gradient goes through: the quantised one, as floats
        self.head_bf16 = (self.head.float() * self.head_scale[:, None]).to(bf16)
        self.final = torch.ones(width, device=device)  # trained

        e = lambda *s, d=torch.float32: torch.empty(s, device=device, dtype=d)
        self.norm_plan = op.NormPlan(tokens, width, cabi.BF16, dtype_out=cabi.INT8)
        self.last_plan = op.NormPlan(tokens, width, cabi.BF16, dtype_weight=cabi.FP32, dtype_out=cabi.INT8,
                                     dtype_grad=cabi.FP32)
        self.gate_plan = op.Int8ContractPlan(tokens, 2 * hidden, width, activation=op.ACT_GATED_SILU)
        self.quant_plan = op.QuantizePlan(tokens, hidden, cabi.BF16)
        self.down_plan = op.Int8ContractPlan(tokens, width, hidden)
        self.head_plan = op.Int8ContractPlan(tokens, vocab, width)
        self.score_plan = op.LogprobPlan(tokens, vocab, cabi.BF16, top=top)
        il, ir, io, names = binary.parse_binary("tv,vc->tc")
        size = dict(zip(names, range(len(names))))
        sizes = {size["t"]: tokens, size["v"]: vocab, size["c"]: width}
        self.back_plan = cabi.ContractPlan(binary.contraction_dims(il, ir, io, sizes), cabi.BF16, cabi.BF16, cabi.FP32)
        self.q_width, self.q_hidden = e(tokens, width, d=torch.int8), e(tokens, hidden, d=torch.int8)
        self.scale, self.rstd = e(tokens), e(tokens)
        self.stream_out, self.act, self.out = e(tokens, width, d=bf16), e(tokens, hidden, d=bf16), e(tokens, width, d=bf16)
        self.logits = e(tokens, vocab, d=bf16)
        self.logprob, self.entropy, self.lse = e(tokens), e(tokens), e(tokens)
        self.top_logprob, self.top_index = (e(tokens, top), e(tokens, top, d=torch.int64)) if top else (None, None)
        self.dy, self.dx, self.dweight = e(tokens, width), e(tokens, width), e(width)

    def score(self, h, targets, stream=0):
        """log probabilities of `targets` after the residual stream `h` (BF16 [tokens, width])"""
        add = None
        for norm, gate_up, gate_scale, down, down_scale in self.layers:
            self.norm_plan.norm(h, self.q_width, weight=norm, residual=add, sum=self.stream_out, scale=self.scale,
                                stream=stream)
            self.gate_plan.contract(self.q_width, gate_up, self.scale, gate_scale, self.act, stream=stream)
            self.quant_plan.quantize(self.act, self.q_hidden, self.scale, stream=stream)
            self.down_plan.contract(self.q_hidden, down, self.scale, down_scale, self.out, stream=stream)
            h, add = self.stream_out, self.out
        # from the second layer on the sum replaces the residual stream in place
        self.last_plan.norm(h, self.q_width, weight=self.final, residual=add, sum=self.stream_out, scale=self.scale,
                            rstd=self.rstd, stream=stream)
        self.head_plan.contract(self.q_width, self.head, self.scale, self.head_scale, self.logits, stream=stream)
        self.score_plan.logprob(self.logits, targets, self.logprob, entropy=self.entropy, lse=self.lse,
                                top_logprob=self.top_logprob, top_index=self.top_index, stream=stream)
        return self.logprob

    def gradient(self, targets, dlogprob, stream=0):
        """gradient of the final norm's weight after score(): the logits' gradient takes the logits' place"""
        self.score_plan.backward(self.logits, targets, self.lse, dlogprob, self.logits, stream=stream)
        self.back_plan.contract(self.logits, self.head_bf16, self.dy, stream=stream)
        self.last_plan.backward(self.dy, self.stream_out, self.rstd, self.dx, weight=self.final, dweight=self.dweight,
                                stream=stream)
        return self.dweight

    def score_float(self, h, targets):
        """the same in FP32 with the float weights (for comparison)"""
        def rms(x, w):
            return x * torch.rsqrt(x.square().mean(1, keepdim=True) + 1e-6) * w.float()
        h = h.float()
        for norm, gate_up, down in self.weights:
            gate, up = (rms(h, norm) @ gate_up.T).chunk(2, 1)
            h = h + (torch.nn.functional.silu(gate) * up) @ down.T
        logp = torch.log_softmax(rms(h, self.final) @ self.head_float.T, 1)
        return logp.gather(1, targets.clamp_min(0)[:, None])[:, 0].masked_fill(targets < 0, 0.0)


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--tokens", type=int, default=512)
    p.add_argument("--width", type=int, default=1024)
    p.add_argument("--hidden", type=int, default=4096)
    p.add_argument("--layers", type=int, default=2)
    p.add_argument("--vocab", type=int, default=32768)
    p.add_argument("--top", type=int, default=5)
    p.add_argument("--steps", type=int, default=5)
    a = p.parse_args(argv)
    m = Model(a.tokens, a.width, a.hidden, a.layers, a.vocab, a.top)
    g = torch.Generator(device="cuda").manual_seed(1)
    h = torch.randn((a.tokens, a.width), generator=g, device="cuda").to(torch.bfloat16)
    targets = torch.randint(a.vocab, (a.tokens,), generator=g, device="cuda")
    want = m.score_float(h, targets)
    got = m.score(h, targets).clone()
    err = (got - want).abs().mean().item()
    print(f"log probability: mean {got.mean().item():.4f}, in FP32 {want.mean().item():.4f}, mean difference {err:.4f}")
    if a.top:
        print(f"entropy: mean {m.entropy.mean().item():.4f}; alternatives of token 0: {m.top_index[0].tolist()}")
    losses = []
    dlogprob = torch.full((a.tokens,), -1.0 / a.tokens, device="cuda")  # loss: minus the mean log probability
    for step in range(a.steps):
        losses.append(-m.score(h, targets).mean().item())
        m.final -= 200.0 * m.gradient(targets, dlogprob)
        print(f"step {step}: loss {losses[-1]:.5f}")
    cabi.check_device_errors()
    return {"difference": err, "losses": losses, "model": m}


if __name__ == "__main__":
    main()
