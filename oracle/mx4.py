"""64-bit statements of the 4-bit expert operators and of the block norm (any device, plain torch).

MXFP4 as the OCP microscaling formats define it: E2M1 values, a shared E8M0
scale for 32 of them, the scale's exponent floor(log2 max) less E2M1's largest
exponent, round to nearest even, saturating.
"""
from __future__ import annotations

import torch

E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """fp64 values of codes [..., K / 2] and scale bytes [..., K / 32]."""
    table = torch.tensor(E2M1 + [-v for v in E2M1], dtype=torch.float64, device=codes.device)
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    s = torch.exp2(scales.double() - 127)
    s = torch.where(scales == 255, torch.full_like(s, float("nan")), s)
    return table[c] * s.repeat_interleave(32, -1)


def quantize(x: torch.Tensor):
    """(codes, scales) of x [..., K]; nearest by search over the eight magnitudes, ties to the even code."""
    v = x.double().unflatten(-1, (-1, 32))
    amax = v.abs().amax(-1)
    bad = ~torch.isfinite(v).all(-1)
    ok = torch.where(bad | (amax == 0), torch.ones_like(amax), amax)
    s = (torch.frexp(ok).exponent - 3).clamp(-127, 127)
    a = v.abs() * torch.exp2(-s.double()).unsqueeze(-1)
    a = torch.where(bad.unsqueeze(-1), torch.zeros_like(a), a)
    grid = torch.tensor(E2M1, dtype=torch.float64, device=x.device)
    d = (a.unsqueeze(-1) - grid).abs()
    best = d.amin(-1, keepdim=True)
    near = d == best                                    # two of them at a tie: one has an even code
    even = torch.arange(8, device=x.device) % 2 == 0
    code = torch.where(near.sum(-1) == 1, near.int().argmax(-1), (near & even).int().argmax(-1))
    code = code + 8 * torch.signbit(v)
    code = torch.where(bad.unsqueeze(-1), torch.zeros_like(code), code).to(torch.uint8).flatten(-2)
    s = torch.where(amax == 0, torch.full_like(s, -127), s) + 127
    s = torch.where(bad, torch.full_like(s, 255), s).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), s


def block_norm(y, residual, weight, post_weight=None, gate=None, scale=1.0, eps=1e-6):
    """(normed, new residual) in fp64."""
    z = y.double()
    if post_weight is not None:
        z = z / torch.sqrt(z.pow(2).mean(-1, keepdim=True) + eps) * post_weight.double()
    if gate is not None:
        z = z * gate.double()
    r = residual.double() + scale * z
    return r / torch.sqrt(r.pow(2).mean(-1, keepdim=True) + eps) * weight.double(), r


def route(x, router, top_k, renormalize=True):
    """(weights, ids) [T, k]: softmax of x router^T in fp64, ties to the lower id."""
    logits = x.double() @ router.double().T
    order = torch.sort(logits, dim=-1, descending=True, stable=True)
    p = torch.softmax(logits, -1).gather(1, order.indices[:, :top_k])
    return (p / p.sum(-1, keepdim=True) if renormalize else p), order.indices[:, :top_k]


def moe(x, w13, w2, weights, ids, expert_map=None):
    """(out, size, slack) in fp64 of an MoE layer with dequantised w13 [S, 2I, H] and w2 [S, H, I].  `size`: the sum
    of the magnitudes that meet in an output, sum p |a| |w2|; `slack`: what an error of one part of the magnitudes
    that meet in g and u makes of the output."""
    out, size, slack = (torch.zeros(x.shape, dtype=torch.float64, device=x.device) for _ in range(3))
    xd = x.double()
    for t in range(x.shape[0]):
        for w, e in zip(weights[t].tolist(), ids[t].tolist()):
            s = e if expert_map is None else (int(expert_map[e]) if 0 <= e < len(expert_map) else -1)
            if not 0 <= s < w13.shape[0]:
                continue
            h, m = w13[s] @ xd[t], w13[s].abs() @ xd[t].abs()
            n = h.shape[0] // 2
            g, u = h[:n], h[n:]
            a = g * torch.sigmoid(g) * u
            out[t] += w * (w2[s] @ a)
            size[t] += abs(w) * (w2[s].abs() @ a.abs())
            slack[t] += abs(w) * (w2[s].abs() @ (1.1 * m[:n] * u.abs() + (g * torch.sigmoid(g)).abs() * m[n:]
                                                 + 1.1 * m[:n] * m[n:] * 2.0 ** -12))
    return out, size, slack
