"""The operators of a block around its attention in 64 bits (linear layers with their epilogue, gated residual and norm,
dropout) with bounds of what the kernels may be off, used by their tests.

Bounds. A rounding to a type is off by at most half a step, ``finfo.eps / 2`` relative. fp32 sums of n products are off by at
most n * 2^-24 of the sum of their magnitudes, in any order.
"""
import math

import numpy as np
import torch

import train_ref as R

E32 = R.E32


def half_step(dtype):
    return R.half_step(dtype)


def philox(counter, key):
    """Philox4x32 with ten rounds (Salmon et al., 2011): counter uint64 arrays of 32-bit words [4], key ints [2]."""
    c = [np.asarray(w, dtype=np.uint64) for w in counter]
    k = [int(w) for w in key]
    low = np.uint64(0xFFFFFFFF)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def keep_bits(state, rows, cols, first_row=0):
    """Sixteen random bits of every element, int64 [rows, cols]."""
    seed, stream = (int(v) for v in state)
    groups = -(-cols // 8)
    row = np.arange(first_row, first_row + rows, dtype=np.uint64)[:, None]
    zero = np.zeros((rows, groups), dtype=np.uint64)
    words = philox([zero + np.arange(groups, dtype=np.uint64), zero + (row & np.uint64(0xFFFFFFFF)),
                    zero + (row >> np.uint64(32)), zero + np.uint64(stream & 0xFFFFFFFF)],
                   [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF])
    bits = np.stack([w >> np.uint64(16 * h) & np.uint64(0xFFFF) for w in words for h in (0, 1)], axis=-1)
    return torch.from_numpy(bits.reshape(rows, groups * 8)[:, :cols].astype(np.int64))


def keep_factor(p, state, rows, cols):
    """keep / (1 - p), fp64 [rows, cols] or 1."""
    limit = round(p * 65536)
    if limit == 0:
        return torch.ones(1, 1, dtype=torch.float64)
    scale = 65536 / (65536 - limit) if limit < 65536 else 0.0
    return (keep_bits(state, rows, cols) >= limit).double() * scale


def activation(kind, z):
    """act(z), act'(z) and the bounds of both kernels' errors in fp32 (32 roundings of values up to 1.5 |z| or 1.5, and the
    1e-7 of the approximation; the derivative adds as many)."""
    if kind is None:
        return z, torch.ones_like(z), torch.zeros_like(z), torch.zeros_like(z)
    if kind == "gelu":
        cdf = 0.5 * torch.special.erfc(-z * math.sqrt(0.5))
        a, d = z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    else:
        c = math.sqrt(2 / math.pi)
        s = torch.sigmoid(2 * c * (z + 0.044715 * z ** 3))
        a, d = z * s, s + z * s * (1 - s) * 2 * c * (1 + 3 * 0.044715 * z * z)
    return a, d, (1e-7 + 32 * E32) * z.abs(), torch.full_like(z, 1e-7 + 96 * E32)


def rounded(value, tol, dtype):
    """The bound after the one rounding to dtype (fp16: also half of its smallest step)."""
    return tol * (1 + 2 * half_step(dtype)) + half_step(dtype) * value.abs() + (2.0 ** -25 if dtype == torch.float16 else 1e-37)


def linear(x, w, bias, kind, gate, residual, factor):
    """{name: (value, bound before its rounding)} of kept and y; every input fp64 (or None), factor of keep_factor."""
    K = x.shape[1]
    b = torch.zeros(w.shape[0], dtype=torch.float64, device=x.device) if bias is None else bias
    z = x @ w.T + b
    z_tol = (K + 4) * E32 * (x.abs() @ w.abs().T + b.abs())
    a, _, a_tol, _ = activation(kind, z)
    a_tol = a_tol + 1.13 * z_tol  # (|act'| is at most 1.129)
    g = 1.0 if gate is None else gate
    d = a * factor * g
    y = d if residual is None else residual + d
    y_tol = a_tol * (factor * (g if gate is None else g.abs())) + 4 * E32 * d.abs() + E32 * y.abs()
    return {"kept": (z, z_tol), "y": (y, y_tol)}


def linear_bwd(dy, x, w, kept, kind, gate, factor, dtype):
    """The same of dx, dweight, dbias and dgate from kept as it is stored; dz is rounded to dtype for the products."""
    rows, N = dy.shape
    a, slope, a_tol, s_tol = activation(kind, torch.zeros_like(dy) if kept is None else kept)
    g = torch.ones(N, dtype=torch.float64, device=dy.device) if gate is None else gate
    dd = dy * g * factor
    dz = dd * slope
    dz_tol = dd.abs() * s_tol + 6 * E32 * dz.abs()
    low_tol = rounded(dz, dz_tol, dtype)
    big = dz.abs() + low_tol

    def product(u, ut, v, n):
        return u @ v, ut @ v.abs() + (n + 2) * E32 * ((u.abs() + ut) @ v.abs())
    res = {"dx": product(dz, low_tol, w, N), "dweight": product(dz.T, low_tol.T, x, rows)}
    res["dbias"] = dz.sum(0), dz_tol.sum(0) + (rows + 2) * E32 * big.sum(0)
    if kept is not None:
        t = dy * factor * a
        res["dgate"] = t.sum(0), ((dy * factor).abs() * a_tol).sum(0) + (rows + 6) * E32 * t.abs().sum(0)
    return res


def residual_norm(x, branch, gate, weight, bias, eps, factor, dtype):
    """h before its rounding with its bound. (The norm reads h as it is stored: norm_of.)"""
    g = 1.0 if gate is None else gate
    d = branch * factor * g
    h = x + d
    return h, 3 * E32 * d.abs() + E32 * h.abs()
