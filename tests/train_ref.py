"""The training operators in 64 bits (attention over frames, rotary head norm, LayerNorm) with bounds of what the
kernels may be off, used by their tests.

Bounds. A rounding to a type is off by at most half a step, ``finfo.eps / 2`` relative (U: bf16, 2^-8). fp32 sums of n
products are off by at most n * 2^-24 of the sum of their magnitudes, in any order.
"""
import math

import torch

from oracle import attention as OA

U = torch.finfo(torch.bfloat16).eps / 2
E32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def frame_attention(q, k, v, dout, patterns, frames, mask=None, scale=0.125):
    """fp64 results of frame_attn_fwd / frame_attn_bwd and bounds of the kernels' distance from them. q, k, v, dout
    [B, N, H, 64] (CPU or GPU, any type), mask bool [B, N] or None. {name: (value, bound)}."""
    B, N, H, D = q.shape
    geom = OA.Geometry(frames, N // frames, 0)
    names = ("out", "dq", "dk", "dv")
    val = {n: torch.zeros(B, N, H, D, dtype=torch.float64) for n in names}
    tol = {n: torch.zeros(B, N, H, D, dtype=torch.float64) for n in names}
    lse = torch.full((B, H, N), -math.inf, dtype=torch.float64)
    lse_tol = torch.zeros(B, H, N, dtype=torch.float64)
    rows = torch.arange(N)
    for b in range(B):
        there = torch.ones(N, dtype=torch.bool) if mask is None else mask[b].cpu().bool()
        for h in range(H):
            if patterns[h] == OA.SKIP:
                continue
            ok = OA.allowed_mask(patterns[h], rows, geom) & there[:, None] & there[None, :]
            some = ok.any(1)
            Q, K, V, G = (torch.where(there[:, None], t[b, :, h].detach().cpu().double(), 0.0) for t in (q, k, v, dout))
            s = (Q @ K.T) * scale
            a = (Q.abs() @ K.abs().T) * scale
            s = s.masked_fill(~ok, -math.inf)
            lse[b, h][some] = torch.logsumexp(s[some], -1)
            p = torch.where(some[:, None], torch.softmax(torch.where(some[:, None], s, 0.0), -1), 0.0) * ok
            # a score: 64 products, the scale (twice: its rounding and the product) and the subtraction of a reference
            ds_abs = (72 * E32) * a + 4 * E32 * s.masked_fill(~ok, 0).abs()
            # a probability: its score, its reference (lse or the row's maximum, of the scores' magnitude), exp2 (1 ulp)
            rel = 2 * ds_abs.max(1, keepdim=True).values + 8 * E32 * (1 + lse[b, h].masked_fill(~some, 0).abs()[:, None])
            o = p @ V
            pv = p @ V.abs()
            val["out"][b, :, h] = o
            # P rounded to bf16, the sums of N products and of N probabilities, the result rounded
            tol["out"][b, :, h] = (U + rel + 2 * N * E32) * pv + U * o.abs()
            lse_tol[b, h] = rel[:, 0] + N * E32
            gv = G @ V.T
            gva = G.abs() @ V.abs().T
            d = (G * o).sum(-1, keepdim=True)
            dsm = p * (gv - d) * ok
            # D = dO . (out + rest): P of the forward pass is rounded (U), out + rest to 2^-16
            d_tol = (U + rel + 2 * N * E32) * (p * gva).sum(-1, keepdim=True) + (2.0 ** -16 + 70 * E32) * (
                G.abs() * o.abs()).sum(-1, keepdim=True)
            ds_tol = (U + 2 * rel) * dsm.abs() + p * (d_tol * (1 + U) + 70 * E32 * gva)
            val["dq"][b, :, h] = dsm @ K * scale
            tol["dq"][b, :, h] = (ds_tol @ K.abs() + N * E32 * (dsm.abs() @ K.abs())) * scale + U * val["dq"][b, :, h].abs()
            val["dk"][b, :, h] = dsm.T @ Q * scale
            tol["dk"][b, :, h] = (ds_tol.T @ Q.abs() + N * E32 * (dsm.abs().T @ Q.abs())) * scale + U * val["dk"][b, :, h].abs()
            val["dv"][b, :, h] = p.T @ G
            tol["dv"][b, :, h] = ((U + 2 * rel + N * E32) * p).T @ G.abs() + U * val["dv"][b, :, h].abs()
    res = {n: (val[n], tol[n] + 1e-30) for n in names}
    res["lse"] = (lse, lse_tol + 1e-30)
    return res


def rotate(x, pos, cos, sin, layout, rotary_dim, sign=1.0):
    """x [B, N, G, H, D]; one section at a time by 2x2 rotations."""
    y = x.clone()
    axes = pos.shape[-1]
    S = rotary_dim // axes
    for a in range(axes):
        at = pos[..., a].long().clamp(0, cos.shape[0] - 1)
        c = cos.to(x.dtype)[at][:, :, None, None]
        s = sign * sin.to(x.dtype)[at][:, :, None, None]
        j = torch.arange(S // 2, device=x.device)
        i0 = a * S + (j if layout == "half" else 2 * j)
        i1 = i0 + (S // 2 if layout == "half" else 1)
        u, v = x[..., i0], x[..., i1]
        y[..., i0] = u * c - v * s
        y[..., i1] = v * c + u * s
    return y


def layer_norm(x, weight, bias, eps):
    m = x.mean(-1, keepdim=True)
    r = 1.0 / torch.sqrt(((x - m) ** 2).mean(-1, keepdim=True) + eps)
    xh = (x - m) * r
    y = xh
    if weight is not None:
        y = y * weight
    if bias is not None:
        y = y + bias
    return y, m.squeeze(-1), r.squeeze(-1), xh


def layer_norm_bwd(dy, xh, rstd, weight):
    g = dy if weight is None else dy * weight
    return rstd[..., None] * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
