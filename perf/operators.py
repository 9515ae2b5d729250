"""Measured cases of the row operators and the 8-bit contraction.

Six operators: the root-mean-square norm with the residual's addition (float or
8-bit output) and its backward pass, the quantisation of rows to 8 bits, the
contraction of 8-bit integers with a scale for each token and channel, and the
log probabilities of given tokens with entropy and top alternatives and their
backward pass. ``run`` computes them with elementary torch operations in 32
bits, or, where ``own`` is set, with the framework's kernels on the same inputs.
"""
from __future__ import annotations

import math

import torch

own = False

# ---------------------------------------------------------------- cases


def listed():
    return [
        # one decoded token before a layer's first contraction: launch latency
        {"name": "norm int8 one token", "op": "norm", "rows": 1, "cols": 4096, "dtype": "bf16", "out": "int8",
         "residual": True, "pad": 0},
        # a prefill batch of the MLP configuration (8192 rows of width 4096) before an 8-bit contraction
        {"name": "norm int8 prefill", "op": "norm", "rows": 8192, "cols": 4096, "dtype": "bf16", "out": "int8",
         "residual": True, "pad": 0},
        # the backward pass of the same layer in a training step
        {"name": "norm backward bf16", "op": "norm_backward", "rows": 8192, "cols": 4096, "dtype": "bf16",
         "residual": True, "pad": 0},
        # a ragged FP32 model: odd width, rows that start off any vector boundary
        {"name": "norm backward odd f32", "op": "norm_backward", "rows": 1237, "cols": 2311, "dtype": "f32",
         "residual": False, "pad": 0},
        # a few decoded tokens between the two contractions of a feed-forward block
        {"name": "quantize few rows", "op": "quantize", "rows": 5, "cols": 16384, "dtype": "bf16", "pad": 0},
        # the hidden activations of a prefill batch, a slice of a wider buffer, ragged
        {"name": "quantize ragged", "op": "quantize", "rows": 4099, "cols": 10920, "dtype": "bf16", "pad": 24},
        # one decoded token through a 4096 x 4096 layer with bias: the weights' bytes
        {"name": "contract one token", "op": "contract", "m": 1, "n": 4096, "k": 4096, "act": "relu", "bias": True,
         "out": "bf16"},
        # the MLP configuration's layer in 8 bits: batch 8192, width 4096, bias and ReLU
        {"name": "contract mlp layer", "op": "contract", "m": 8192, "n": 4096, "k": 4096, "act": "relu", "bias": True,
         "out": "bf16"},
        # a small serving batch through a gated first layer of odd hidden width
        {"name": "contract gated batch", "op": "contract", "m": 77, "n": 10922, "k": 4096, "act": "gated_silu",
         "bias": False, "out": "bf16"},
        # a few sampled tokens over a large vocabulary, alternatives for the user
        {"name": "logprob few tokens", "op": "logprob", "rows": 3, "vocab": 131072, "dtype": "f32", "top": 8},
        # scoring a long prompt: every token's log probability, entropy and alternatives
        {"name": "logprob prompt", "op": "logprob", "rows": 4096, "vocab": 32768, "dtype": "bf16", "top": 5},
        # the loss's gradient with an entropy term over an odd vocabulary
        {"name": "logprob backward odd", "op": "logprob_backward", "rows": 2048, "vocab": 50021, "dtype": "bf16",
         "entropy": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _rows_cols(rng, lo_cols, hi_cols, most):
    cols = _log_int(rng, lo_cols, hi_cols)
    if rng.random() < 0.6:  # most widths are multiples of a vector
        cols = max(16, cols // 16 * 16)
    return _log_int(rng, 1, max(1, min(16384, most // cols))), cols


def draw(rng):
    op = rng.choice(["norm", "norm_backward", "quantize", "contract", "contract", "logprob", "logprob_backward"])
    if op in ("norm", "norm_backward", "quantize"):
        rows, cols = _rows_cols(rng, 64, 20000, 1 << 26)
        c = {"op": op, "rows": rows, "cols": cols, "dtype": rng.choice(["bf16", "bf16", "f32"]),
             "pad": rng.choice([0, 0, 8, 3])}
        if op == "norm":
            c["out"] = rng.choice(["int8", "int8", "same"])
        if op != "quantize":
            c["residual"] = rng.random() < 0.7
        return c
    if op == "contract":
        k, n = _log_int(rng, 128, 16384), _log_int(rng, 64, 32768)
        if rng.random() < 0.7:
            k = max(128, k // 64 * 64)
        if rng.random() < 0.6:
            n = max(64, n // 64 * 64)
        m = _log_int(rng, 1, max(1, min(16384, (8192 * 4096 * 4096) // (n * k))))
        act = rng.choice(["none", "relu", "gated_silu"])
        n -= n % 2 if act == "gated_silu" else 0
        return {"op": op, "m": m, "n": n, "k": k, "act": act, "bias": rng.random() < 0.5,
                "out": rng.choice(["bf16", "bf16", "f32"])}
    vocab = _log_int(rng, 1000, 200000)
    if rng.random() < 0.6:
        vocab = vocab // 64 * 64
    rows = _log_int(rng, 1, max(1, min(8192, (1 << 27) // vocab)))
    c = {"op": op, "rows": rows, "vocab": vocab, "dtype": rng.choice(["bf16", "f32"])}
    if op == "logprob":
        c["top"] = rng.choice([0, 1, 5, 8, 20])
    else:
        c["entropy"] = rng.random() < 0.5
    return c


# ---------------------------------------------------------------- inputs

_TORCH = {"bf16": torch.bfloat16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f32": 4, "int8": 1}


class _State:
    pass


def _rand(g, shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _rows(g, rows, cols, dtype, pad, scale=1.0):
    """rows of a buffer that is `pad` elements wider"""
    return _rand(g, (rows, cols + pad), dtype, scale)[:, :cols]


def _codes(g, rows, k):
    """8-bit rows with their scales, from normal values"""
    x = torch.randn((rows, k), generator=g, device="cuda")
    m = x.abs().amax(1, keepdim=True)
    return torch.round(x * (127.0 / m)).to(torch.int8), (m[:, 0] / 127.0).contiguous()


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = _State()
    s.case = case
    op = case["op"]
    if op in ("norm", "norm_backward", "quantize"):
        dt, rows, cols, pad = _TORCH[case["dtype"]], case["rows"], case["cols"], case["pad"]
        s.x = _rows(g, rows, cols, dt, pad)
        # activations have a few large channels
        s.x[:, :: max(1, cols // 7)] *= 8
        if op == "quantize":
            return s
        s.w = (1 + 0.2 * torch.randn(cols, generator=g, device="cuda")).to(dt)
        s.eps = 1e-6
        if op == "norm":
            s.r = _rows(g, rows, cols, dt, pad, 3.0) if case["residual"] else None
        else:
            s.rstd = torch.rsqrt(s.x.float().square().mean(1) + s.eps)
            s.dy = _rows(g, rows, cols, dt, pad, 0.01)
            s.dsum = _rows(g, rows, cols, dt, pad, 0.01) if case["residual"] else None
    elif op == "contract":
        m, n, k = case["m"], case["n"], case["k"]
        s.a, s.sa = _codes(g, m, k)
        s.b, s.sb = _codes(g, n, k)
        s.sb = s.sb * (2.0 / math.sqrt(k))  # activations of order one
        s.bias = _rand(g, (n,), scale=0.5) if case["bias"] else None
    else:
        rows, vocab, dt = case["rows"], case["vocab"], _TORCH[case["dtype"]]
        s.x = _rand(g, (rows, vocab), dt, 3.0)
        # a likely token in every row, and one entry in about a hundred ruled out
        likely = torch.randint(vocab, (rows, 1), generator=g, device="cuda")
        s.x.scatter_add_(1, likely, torch.full((rows, 1), 12.0, device="cuda", dtype=dt))
        out = torch.randint(vocab, (max(1, vocab // 100),), generator=g, device="cuda")
        s.x[:, out] = float("-inf")
        s.t = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.5, likely[:, 0],
                          torch.randint(vocab, (rows,), generator=g, device="cuda"))
        s.t[5::16] = -100  # padding
        if op == "logprob_backward":
            x = s.x.float()
            s.lse = torch.logsumexp(x, 1)
            p = torch.exp(x - s.lse[:, None])
            s.ent = s.lse - torch.where(p > 0, p * x, 0.0).sum(1)
            s.dlp = _rand(g, (rows,), scale=0.5)
            s.dent = _rand(g, (rows,), scale=0.1) if case["entropy"] else None
    return s


def _plan(s):
    """the framework's plan and the output buffers that a user's program keeps"""
    from einsum_ir_b200 import cabi, operators
    case, op = s.case, s.case["op"]
    code = {"bf16": cabi.BF16, "f32": cabi.FP32, "int8": cabi.INT8}
    f32 = dict(device="cuda", dtype=torch.float32)
    if op in ("norm", "norm_backward"):
        dt, rows, cols, ld = case["dtype"], case["rows"], case["cols"], s.x.stride(0)
        kind = case.get("out", "same")
        s.plan = operators.NormPlan(rows, cols, code[dt], dtype_weight=code[dt],
                                    dtype_out=code[dt if kind == "same" else kind], dtype_grad=code[dt], eps=s.eps,
                                    stride_x=ld, stride_residual=ld, stride_dy=ld, stride_dsum=ld)
        s.rows_out = torch.empty((rows, cols), device="cuda", dtype=_TORCH[dt])
        if op == "norm":
            s.sum = torch.empty_like(s.rows_out) if case["residual"] else None
            s.out_rstd = torch.empty(rows, **f32)
            s.y = torch.empty((rows, cols), device="cuda", dtype=torch.int8) if kind == "int8" else s.rows_out
            s.scale = torch.empty(rows, **f32) if kind == "int8" else None
        else:
            s.dw = torch.empty(cols, **f32)
    elif op == "quantize":
        s.plan = operators.QuantizePlan(case["rows"], case["cols"], code[case["dtype"]], stride_x=s.x.stride(0))
        s.y = torch.empty((case["rows"], case["cols"]), device="cuda", dtype=torch.int8)
        s.scale = torch.empty(case["rows"], **f32)
    elif op == "contract":
        acts = {"none": operators.ACT_NONE, "relu": operators.ACT_RELU, "gated_silu": operators.ACT_GATED_SILU}
        s.plan = operators.Int8ContractPlan(case["m"], case["n"], case["k"], dtype_out=code[case["out"]],
                                            activation=acts[case["act"]])
        n_out = case["n"] // 2 if case["act"] == "gated_silu" else case["n"]
        s.y = torch.empty((case["m"], n_out), device="cuda", dtype=_TORCH[case["out"]])
    else:
        rows, top = case["rows"], case.get("top", 0)
        s.plan = operators.LogprobPlan(rows, case["vocab"], code[case["dtype"]], top=top)
        if op == "logprob":
            s.lp, s.out_ent, s.out_lse = (torch.empty(rows, **f32) for _ in range(3))
            s.top_lp = torch.empty((rows, top), **f32) if top else None
            s.top_index = torch.empty((rows, top), device="cuda", dtype=torch.int64) if top else None
        else:
            s.dx = torch.empty_like(s.x)


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        _plan(s)
    return s


# ---------------------------------------------------------------- one pass


def _quantized(v):
    """rows of v in 8 bits: q = round(v 127 / max|v|), and the row maxima"""
    m = v.abs().amax(1, keepdim=True)
    inv = torch.where(m > 0, torch.full_like(m, 127.0) / m, 0.0)
    return torch.round(v * inv).to(torch.int8), m[:, 0]


def _plain(s):
    case, op = s.case, s.case["op"]
    if op == "norm":
        dt = s.x.dtype
        h = s.x.float() if s.r is None else s.x.float() + s.r.float()
        rstd = 1.0 / torch.sqrt((h * h).mean(1) + s.eps)
        out = {"rstd": rstd}
        if s.r is not None:
            out["sum"] = h.to(dt)
        if case["out"] == "int8":
            # the integers that a contraction multiplies; the norm's factor cancels in them
            out["q"], m = _quantized(h * s.w.float())
            out["scale"] = m * rstd / 127.0
        else:
            out["y"] = (h * rstd[:, None] * s.w.float()).to(dt)
        return out
    if op == "norm_backward":
        h, dy = s.x.float(), s.dy.float()
        g = dy * s.w.float()
        rstd = s.rstd[:, None]
        dx = rstd * (g - h * (rstd * rstd * (g * h).mean(1, keepdim=True)))
        if s.dsum is not None:
            dx = dx + s.dsum.float()
        return {"dx": dx.to(s.x.dtype), "dweight": (dy * h * rstd).sum(0)}
    if op == "quantize":
        q, m = _quantized(s.x.float())
        return {"q": q, "scale": m / 127.0}
    if op == "contract":
        y = (s.a.float() @ s.b.float().T) * s.sa[:, None] * s.sb
        if s.bias is not None:
            y = y + s.bias
        if case["act"] == "relu":
            y = torch.clamp_min(y, 0.0)
        elif case["act"] == "gated_silu":
            gate, up = y[:, : case["n"] // 2], y[:, case["n"] // 2:]
            y = gate / (1.0 + torch.exp(-gate)) * up
        return {"y": y.to(_TORCH[case["out"]])}
    x = s.x.float()
    hit = s.t.clamp_min(0)[:, None]
    kept = s.t >= 0
    if op == "logprob":
        m = x.amax(1, keepdim=True)
        lse = m[:, 0] + torch.log(torch.exp(x - m).sum(1))
        logp = x - lse[:, None]
        p = torch.exp(logp)
        out = {"logprob": torch.where(kept, logp.gather(1, hit)[:, 0], 0.0),
               "entropy": -torch.where(p > 0, p * logp, 0.0).sum(1), "lse": lse}
        if case["top"]:
            # one whole number for value and place: ties go to the lowest index
            b = (x + 0.0).view(torch.int32)
            key = (b ^ ((b >> 31) & 0x7fffffff)).to(torch.int64) << 32
            key = key + (0x7fffffff - torch.arange(x.shape[1], device=x.device))
            at = 0x7fffffff - (torch.topk(key, case["top"], dim=1).values & 0xffffffff)
            out["top_index"], out["top_logprob"] = at, logp.gather(1, at)
        return out
    logp = x - s.lse[:, None]
    p = torch.exp(logp)
    dlp = torch.where(kept, s.dlp, 0.0)[:, None]
    dx = -dlp * p
    dx.scatter_add_(1, hit, dlp)
    if s.dent is not None:
        dx = dx - s.dent[:, None] * torch.where(p > 0, p * (logp + s.ent[:, None]), 0.0)
    return {"dlogits": dx.to(s.x.dtype)}


def run(s):
    if not own:
        return _plain(s)
    op = s.case["op"]
    if op == "norm":
        s.plan.norm(s.x, s.y, weight=s.w, residual=s.r, sum=s.sum, scale=s.scale, rstd=s.out_rstd)
        out = {"rstd": s.out_rstd}
        if s.sum is not None:
            out["sum"] = s.sum
        if s.scale is not None:
            out["q"], out["scale"] = s.y, s.scale
        else:
            out["y"] = s.y
        return out
    if op == "norm_backward":
        s.plan.backward(s.dy, s.x, s.rstd, s.rows_out, weight=s.w, dsum=s.dsum, dweight=s.dw)
        return {"dx": s.rows_out, "dweight": s.dw}
    if op == "quantize":
        s.plan.quantize(s.x, s.y, s.scale)
        return {"q": s.y, "scale": s.scale}
    if op == "contract":
        s.plan.contract(s.a, s.b, s.sa, s.sb, s.y, bias=s.bias)
        return {"y": s.y}
    if op == "logprob":
        s.plan.logprob(s.x, s.t, s.lp, entropy=s.out_ent, lse=s.out_lse, top_logprob=s.top_lp, top_index=s.top_index)
        out = {"logprob": s.lp, "entropy": s.out_ent, "lse": s.out_lse}
        if s.top_lp is not None:
            out["top_index"], out["top_logprob"] = s.top_index, s.top_lp
        return out
    s.plan.backward(s.x, s.t, s.lse, s.dlp, s.dx, entropy=s.ent if s.dent is not None else None, dentropy=s.dent)
    return {"dlogits": s.dx}


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    op = case["op"]
    if op in ("norm", "norm_backward", "quantize"):
        rows, cols, e = case["rows"], case["cols"], _BYTES[case["dtype"]]
        n = rows * cols
        if op == "quantize":
            return {"bytes": n * (e + 1) + 4 * rows, "flops": 3 * n}
        if op == "norm":
            by = n * e * (3 if case["residual"] else 1) + cols * e + 4 * rows
            by += n + 4 * rows if case["out"] == "int8" else n * e
            return {"bytes": by, "flops": 5 * n}
        return {"bytes": n * e * (4 if case["residual"] else 3) + cols * (e + 4) + 4 * rows, "flops": 10 * n}
    if op == "contract":
        m, n, k = case["m"], case["n"], case["k"]
        n_out = n // 2 if case["act"] == "gated_silu" else n
        by = m * k + n * k + 4 * (m + n) + (4 * n if case["bias"] else 0) + m * n_out * _BYTES[case["out"]]
        return {"bytes": by, "flops": 2 * m * n * k}
    rows, vocab, e = case["rows"], case["vocab"], _BYTES[case["dtype"]]
    if op == "logprob":
        return {"bytes": rows * (vocab * e + 8 + 12 + 12 * case["top"]), "flops": 6 * rows * vocab}
    return {"bytes": rows * (2 * vocab * e + 8 + 16), "flops": 8 * rows * vocab}


# ---------------------------------------------------------------- the definitions in 64 bits


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op in ("norm", "norm_backward"):
        h, w = s.x.double(), s.w.double()
        if op == "norm":
            if s.r is not None:
                h = h + s.r.double()
            rms = torch.linalg.vector_norm(h, dim=1).square().div(case["cols"]).add(s.eps).sqrt()
            out = {"rstd": rms.reciprocal()}
            if s.r is not None:
                out["sum"] = h
            y = w * (h / rms[:, None])
            if case["out"] == "int8":
                out["q"], out["scale"] = None, y.abs().amax(1) / 127  # a value between two integers is rounded in 32 bits
            else:
                out["y"] = y
            return out
        dy, unit = s.dy.double(), h * s.rstd.double()[:, None]
        g = w * dy
        dx = (g - unit * torch.einsum("rc,rc->r", g, unit)[:, None] / case["cols"]) * s.rstd.double()[:, None]
        if s.dsum is not None:
            dx += s.dsum.double()
        return {"dx": dx, "dweight": torch.einsum("rc,rc->c", dy, unit)}
    if op == "quantize":
        return {"q": None, "scale": torch.linalg.vector_norm(s.x.double(), ord=float("inf"), dim=1) / 127}
    if op == "contract":
        a, b = s.a.double() * s.sa.double()[:, None], s.b.double() * s.sb.double()[:, None]
        y = torch.einsum("mk,nk->mn", a, b)
        if s.bias is not None:
            y += s.bias.double()
        if case["act"] == "relu":
            y = torch.where(y > 0, y, 0.0)
        elif case["act"] == "gated_silu":
            gate, up = y.chunk(2, dim=1)
            y = gate * torch.sigmoid(gate) * up
        return {"y": y}
    x = s.x.double()
    if op == "logprob":
        logp = torch.log_softmax(x, 1)
        lp = logp[torch.arange(len(x), device=x.device), s.t.clamp_min(0)].masked_fill(s.t < 0, 0.0)
        out = {"logprob": lp, "entropy": -torch.xlogy(logp.exp(), logp.exp()).sum(1), "lse": torch.logsumexp(x, 1)}
        if case["top"]:
            out["top_index"], out["top_logprob"] = None, logp.topk(case["top"], dim=1).values
        return out
    p = torch.exp(x - s.lse.double()[:, None])
    dlp = s.dlp.double().masked_fill(s.t < 0, 0.0)
    dx = p * -dlp[:, None]
    rows = torch.arange(len(x), device=x.device)
    dx[rows, s.t.clamp_min(0)] += dlp
    if s.dent is not None:
        surprise = torch.where(p > 0, x - (s.lse - s.ent).double()[:, None], 0.0)
        dx -= s.dent.double()[:, None] * p * surprise
    return {"dlogits": dx}
