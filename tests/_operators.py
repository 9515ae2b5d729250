"""Plain 64-bit definitions of the row operators and the 8-bit contraction."""
from __future__ import annotations

import torch


def norm64(x, residual, weight, eps):
    """h, rstd and y of rows in 64 bits"""
    h = x.double() if residual is None else x.double() + residual.double()
    rstd = (h.square().mean(1) + eps) ** -0.5
    y = h * rstd[:, None]
    return {"h": h, "rstd": rstd, "y": y if weight is None else y * weight.double()}


def norm_backward64(dy, h, weight, rstd, dsum):
    dy, h, r = dy.double(), h.double(), rstd.double()[:, None]
    g = dy if weight is None else dy * weight.double()
    dx = r * (g - h * r.square() * (g * h).mean(1, keepdim=True))
    return dx if dsum is None else dx + dsum.double(), (dy * h * r).sum(0)


def quantized32(v):
    """the integers of rows v (FP32), and the row maxima: the operators' rule, operation by operation"""
    v = v.float()
    m = v.abs().amax(1, keepdim=True)
    fine = torch.isfinite(v).all(1, keepdim=True)
    inv = torch.where(fine & (m >= 2.0 ** -100), torch.full_like(m, 127.0) / m, 0.0)
    q = torch.where(fine, torch.round(torch.where(fine, v, 0.0) * inv), 0.0).to(torch.int8)
    return q, m[:, 0], fine[:, 0]


def contract64(left, right, scale_left, scale_right, bias, act):
    """act: 0 none, 1 ReLU, 2 gated SiLU. The sums are exact (below 2^53)."""
    z = left.double() @ right.double().T
    if scale_left is not None:
        z = z * scale_left.double()[:, None]
    if scale_right is not None:
        z = z * scale_right.double()
    if bias is not None:
        z = z + bias.double()
    if act == 1:
        return torch.relu(z)
    if act == 2:
        gate, value = z.chunk(2, 1)
        return gate * torch.sigmoid(gate) * value
    return z


def logprob64(x, targets, top):
    x = x.double()
    none = torch.isneginf(x).all(1)
    lse = torch.where(none, -torch.inf, torch.logsumexp(x, 1))
    logp = torch.where(none[:, None], -torch.inf, x - lse[:, None])
    p = torch.exp(logp)
    out = {"lse": lse, "p": p, "entropy": -torch.where(p == 0, 0.0, p * logp).sum(1)}
    if targets is not None:
        v = x.shape[1]
        lp = logp.gather(1, targets.clamp(0, v - 1)[:, None])[:, 0]
        out["logprob"] = torch.where(targets < 0, 0.0, torch.where(targets >= v, torch.nan, lp))
    if top:
        nan_high = torch.where(torch.isnan(x), torch.inf, x)
        out["top_index"] = torch.sort(nan_high, dim=1, descending=True, stable=True).indices[:, :top]
        out["top_logprob"] = logp.gather(1, out["top_index"])
    return out


def logprob_backward64(x, targets, lse, entropy, dlogprob, dentropy):
    x, lse = x.double(), lse.double()
    none = torch.isneginf(lse)
    d = torch.where(none[:, None], -torch.inf, x - lse[:, None])
    p = torch.exp(d)
    dx = torch.zeros_like(x)
    if targets is not None:
        v = x.shape[1]
        dlp = torch.where(targets < 0, 0.0, torch.where(targets >= v, torch.nan, dlogprob.double()))
        dx = -dlp[:, None] * p
        dx.scatter_add_(1, targets.clamp(0, v - 1)[:, None], torch.where(none, 0.0, dlp)[:, None])
    if dentropy is not None:
        dx = dx - dentropy.double()[:, None] * torch.where(p == 0, 0.0, p * (d + entropy.double()[:, None]))
    return torch.where(none[:, None], 0.0, dx)
