"""Differentiable forms of the training kernels (``ops.frame_attn_*``, ``ops.head_rotary_*``, ``ops.layer_norm_*``) for
fine-tuning a patched model: the static head patterns with their gradients, the q / k prologue and the block norms.

Each function computes its gradients with the backward kernels; nothing is differentiated twice (a second
derivative raises). Without an input that needs a gradient they run the forward kernels alone. A call captured into
a graph follows torch's rules for captured autograd (warm up on a side stream, no live eager graph of the same
parameters).
"""
from __future__ import annotations

from typing import Sequence

import torch
from torch.autograd.function import once_differentiable

from . import ops
from .layout import HEAD_DIM


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, out_dtype):
        y, mean, rstd = ops.layer_norm_fwd(x, weight, bias, eps, out_dtype)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        dx, dw, db = ops.layer_norm_bwd(dy, x, mean, rstd, weight, need_params=ctx.needs_input_grad[1:3])
        return dx, dw, db if db is None else db.to(ctx.bias_dtype), None, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """LayerNorm over the last dimension (``ops.layer_norm_fwd``) with the gradients of x, weight and bias."""
    return _LayerNorm.apply(x, weight, bias, eps, out_dtype)


class _HeadRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, pos, cos, sin, layout, rotary_dim, norm, eps):
        tables = None if cos is None else (cos, sin)
        y = ops.head_rotary_fwd(x, pos, tables, layout, rotary_dim, norm, weight, bias, eps)
        # (without the norm x is not read again: its memory is the caller's)
        ctx.save_for_backward(x if norm else None, weight, pos, cos, sin)
        ctx.args = (layout, rotary_dim, norm, eps, None if bias is None else bias.dtype)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, pos, cos, sin = ctx.saved_tensors
        layout, rotary_dim, norm, eps, bias_dtype = ctx.args
        dx, dw, db = ops.head_rotary_bwd(dy, x if norm else dy, pos, None if cos is None else (cos, sin), layout,
                                         rotary_dim, norm, weight, eps, need_params=ctx.needs_input_grad[1:3])
        return (dx, dw, db if db is None else db.to(bias_dtype), *(None,) * 7)


def head_rotary(x: torch.Tensor, pos: torch.Tensor | None = None, tables=None, layout: str = "half",
                rotary_dim: int | None = None, norm: bool = False, weight: torch.Tensor | None = None,
                bias: torch.Tensor | None = None, eps: float = 1e-5) -> torch.Tensor:
    """LayerNorm over the head dimension and rotary positions (``ops.head_rotary_fwd``) with the gradients of x, weight
    and bias. The tables are constants."""
    cos, sin = (None, None) if tables is None else tables
    return _HeadRotary.apply(x, weight, bias, pos, cos, sin, layout, rotary_dim, norm, eps)


class _FrameAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, patterns, frames, token_mask, scale):
        if not any(ctx.needs_input_grad):
            return ops.frame_attn_fwd(q, k, v, patterns, frames, token_mask, scale)[0]
        out, lse, rest = ops.frame_attn_fwd(q, k, v, patterns, frames, token_mask, scale, rest=True)
        ctx.save_for_backward(q, k, v, out, lse, rest, token_mask)
        ctx.args = (patterns, frames, scale)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, rest, token_mask = ctx.saved_tensors
        patterns, frames, scale = ctx.args
        grads = ops.frame_attn_bwd(dout, q, k, v, out, lse, patterns, frames, token_mask, scale, rest)
        return (*grads, None, None, None, None)


def frame_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, patterns: Sequence[int], frames: int = 1,
                    token_mask: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    """Attention over the tokens of frames (``ops.frame_attn_fwd``) with the gradients of q, k and v."""
    return _FrameAttention.apply(q, k, v, tuple(int(p) for p in patterns), frames, token_mask, scale)


class _QkvAttention(torch.autograd.Function):
    """Prologue and attention on one qkv buffer; the gradients are written into one buffer like it."""

    @staticmethod
    def forward(ctx, qkv, weight, bias, patterns, frames, pos, cos, sin, norm, eps, token_mask, scale):
        B, N, _ = qkv.shape
        x = qkv.view(B, N, 3, len(patterns), HEAD_DIM)
        tables = None if cos is None else (cos, sin)
        qk = x[:, :, :2]
        if norm or tables is not None:
            qk = ops.head_rotary_fwd(qk, pos, tables, norm=norm, weight=weight, bias=bias, eps=eps)
        grad = any(ctx.needs_input_grad)
        res = ops.frame_attn_fwd(qk[:, :, 0], qk[:, :, 1], x[:, :, 2], patterns, frames, token_mask, scale, rest=grad)
        if grad:
            ctx.save_for_backward(qkv, qk, *res, weight, pos, cos, sin, token_mask)
            ctx.args = (patterns, frames, norm, eps, scale, None if bias is None else bias.dtype)
        return res[0].view(B, N, -1)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        qkv, qk, out, lse, rest, weight, pos, cos, sin, token_mask = ctx.saved_tensors
        patterns, frames, norm, eps, scale, bias_dtype = ctx.args
        x = qkv.view(*qkv.shape[:2], 3, len(patterns), HEAD_DIM)
        dqkv = torch.empty_like(qkv, memory_format=torch.contiguous_format)
        dx = dqkv.view(x.shape)
        prologue = norm or cos is not None
        dqk = torch.empty_like(qk, memory_format=torch.contiguous_format) if prologue else dx[:, :, :2]
        ops.frame_attn_bwd(dout.reshape(out.shape), qk[:, :, 0], qk[:, :, 1], x[:, :, 2], out, lse, patterns, frames,
                           token_mask, scale, rest, grads=(dqk[:, :, 0], dqk[:, :, 1], dx[:, :, 2]))
        dw = db = None
        if prologue:
            rows = x[:, :, :2]
            if norm and token_mask is not None:  # (the norm's sums take every row: zeros where a token is not there)
                rows = torch.where((token_mask != 0)[:, :, None, None, None], rows, 0.0)
            _, dw, db = ops.head_rotary_bwd(dqk, rows, pos, None if cos is None else (cos, sin), norm=norm,
                                            weight=weight, eps=eps, need_params=ctx.needs_input_grad[1:3],
                                            out=dx[:, :, :2])
        return (dqkv, dw, db if db is None else db.to(bias_dtype), *(None,) * 9)


def qkv_attention(qkv: torch.Tensor, patterns: Sequence[int], frames: int = 1, pos: torch.Tensor | None = None,
                  tables=None, norm: bool = False, weight: torch.Tensor | None = None,
                  bias: torch.Tensor | None = None, eps: float = 1e-5, token_mask: torch.Tensor | None = None,
                  scale: float | None = None) -> torch.Tensor:
    """A layer's attention between its two projections: qkv bf16 [clips, tokens, 3 * heads * 64] (the qkv Linear's
    output) -> bf16 [clips, tokens, heads * 64]. Norm of q and k over the head dimension (``norm``, ``weight`` / ``bias``
    [2, 64]: q's, k's), rotary positions (``tables``, ``pos`` [clips, tokens, axes], half layout), then
    ``frame_attention``. The gradients of qkv are written in place into one buffer. What the rows of tokens that
    ``token_mask`` removes hold reaches no result and no gradient; their own gradients are zeros."""
    _, _, width = qkv.shape
    if width != 3 * len(patterns) * HEAD_DIM or qkv.dtype != torch.bfloat16:
        raise ValueError(f"qkv must be bfloat16 [clips, tokens, {3 * len(patterns) * HEAD_DIM}], got {qkv.dtype} "
                         f"{tuple(qkv.shape)}")
    cos, sin = (None, None) if tables is None else tables
    return _QkvAttention.apply(qkv.contiguous(), weight, bias, tuple(int(p) for p in patterns), frames, pos, cos, sin,
                               norm, eps, token_mask, scale)


def computed_as(module: torch.nn.Module, kind: type) -> bool:
    """Whether calling ``module`` is ``kind``'s forward and nothing else, so that a kernel can stand for the call: no
    forward of a subclass or of the instance, no hooks."""
    own = module.__dict__
    return (isinstance(module, kind) and type(module).forward is kind.forward and "forward" not in own
            and not (own["_forward_hooks"] or own["_forward_pre_hooks"] or own["_backward_hooks"]
                     or own["_backward_pre_hooks"]))


def _head_norms(attn):
    """(norm, eps, weight, bias) of ``q_norm`` and ``k_norm``, which are one kind: LayerNorm over a head's elements with the
    same eps and the same parameters, or Identity. Others are refused: they would be trained as something else."""
    q, k = attn.q_norm, attn.k_norm
    norm = isinstance(q, torch.nn.LayerNorm)
    kind = torch.nn.LayerNorm if norm else torch.nn.Identity
    for name, m in (("q_norm", q), ("k_norm", k)):
        if not isinstance(m, (torch.nn.LayerNorm, torch.nn.Identity)):
            raise NotImplementedError(f"{name} {type(m).__name__} is not LayerNorm / Identity")
        if not isinstance(m, kind):
            raise NotImplementedError(f"q_norm {type(q).__name__} and k_norm {type(k).__name__} differ")
        if not computed_as(m, kind):
            raise NotImplementedError(f"{name} {type(m).__name__} has a forward of its own or hooks")
    if not norm:
        return False, 1e-5, None, None
    if k.eps != q.eps:
        raise NotImplementedError("q_norm and k_norm of different eps")
    pairs = ((q.weight, k.weight), (q.bias, k.bias))
    if any((a is None) != (b is None) for a, b in pairs):
        raise NotImplementedError("q_norm and k_norm differ in their parameters")
    for m in (q, k):
        if tuple(m.normalized_shape) != (HEAD_DIM,):
            raise NotImplementedError(f"q_norm / k_norm over {tuple(m.normalized_shape)} and not over a head's {HEAD_DIM}")
    return True, q.eps, *(None if a is None else torch.stack([a, b]) for a, b in pairs)


def module_attention(attn, qkv: torch.Tensor, pos: torch.Tensor | None, patterns: Sequence[int], frames: int = 1,
                     positions: int | None = None, token_mask: torch.Tensor | None = None) -> torch.Tensor:
    """``qkv_attention`` with the norms, rotary positions and scale of an ``Attention``-shaped module (``q_norm``,
    ``k_norm``, ``rope`` by its ``base_frequency``, ``scale``): qkv [clips, tokens, 3 * heads * 64], pos int [clips,
    tokens, 2]. ``positions``: length of the rotary tables (default: the largest position + 1, which costs one
    device-to-host read); positions behind it are taken to its end. Raises NotImplementedError for what the kernels do not
    compute: norms of other kinds (or two different ones), and dropout of the probabilities (``attn_drop``) in training."""
    drop = getattr(attn, "attn_drop", 0.0)
    if getattr(attn, "training", False) and getattr(drop, "p", drop):
        raise NotImplementedError(f"attn_drop {getattr(drop, 'p', drop)}: no dropout of the probabilities in training")
    norm, eps, weight, bias = _head_norms(attn)
    tables = None
    if attn.rope is not None and pos is not None:
        n = int(pos.max().item()) + 1 if positions is None else positions
        tables = ops.rope_tables(n, float(attn.rope.base_frequency), qkv.device)
        if pos.dtype not in (torch.int32, torch.int64):
            pos = pos.long()
    else:
        pos = None
    return qkv_attention(qkv, patterns, frames, pos, tables, norm, weight, bias, eps, token_mask,
                         getattr(attn, "scale", None))
