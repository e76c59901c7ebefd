"""Operators around the sequence mixers of a token model: group norm with an activation over
channel-last tensors, and the embedding lookup with scaling.  Both are differentiable; the
``*_fused`` / ``*_vjp`` functions are the operators behind them.  The reference uses PyTorch's own
modules for these (``layers/para_slstm_block.py:144-152``, ``models/``)."""

from __future__ import annotations

import torch
from torch import Tensor

from . import _lib as L
from .ops import _check_cuda, _dtype_code

ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2}


# ------------------------------------------------------------------------------------ group norm

def _norm_check(x: Tensor, num_groups: int, weight: Tensor | None, bias: Tensor | None, activation):
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {tuple(ACTIVATIONS)}, got {activation!r}")
    if x.dim() < 2:
        raise ValueError(f"x must be (N, ..., C), got {tuple(x.shape)}")
    C = x.shape[-1]
    if num_groups < 1 or C < 1 or C % num_groups:
        raise ValueError(f"num_groups={num_groups} must divide the channels ({C})")
    if x.numel() == 0:
        raise ValueError(f"x is empty: {tuple(x.shape)}")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if tuple(p.shape) != (C,):
            raise ValueError(f"{name} must be ({C},), got {tuple(p.shape)}")
        if p.dtype not in (torch.float32, x.dtype):
            raise TypeError(f"{name} must be float32 or {x.dtype}, got {p.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"weight and bias must have one dtype, got {weight.dtype} and {bias.dtype}")
    _dtype_code(x)
    _check_cuda(x, weight, bias)


def group_norm_fused(x: Tensor, num_groups: int, weight: Tensor | None = None, bias: Tensor | None = None,
                     eps: float = 1e-5, activation: str | None = None, *, want_stats: bool = True):
    """``(y, stats)``: ``y`` like ``x``, ``stats (N, num_groups, 2)`` fp32 = mean and ``1/sqrt(var+eps)``."""
    _norm_check(x, num_groups, weight, bias, activation)
    return L.native().norm_fwd(x, num_groups, weight, bias, eps, ACTIVATIONS[activation], want_stats)


def group_norm_vjp(x: Tensor, grad_y: Tensor, stats: Tensor, num_groups: int, weight: Tensor | None = None,
                   bias: Tensor | None = None, activation: str | None = None, *, want_params: bool = True):
    """``(g_x, g_weight, g_bias)``; parameter gradients in the parameters' dtype, summed in fp32."""
    _norm_check(x, num_groups, weight, bias, activation)
    if tuple(grad_y.shape) != tuple(x.shape):
        raise ValueError(f"grad_y must be {tuple(x.shape)}, got {tuple(grad_y.shape)}")
    if tuple(stats.shape) != (x.shape[0], num_groups, 2) or stats.dtype != torch.float32:
        raise ValueError(f"stats must be float32 {(x.shape[0], num_groups, 2)}, got {stats.dtype} {tuple(stats.shape)}")
    _check_cuda(x, grad_y, stats)
    return L.native().norm_bwd(x, grad_y, stats, num_groups, weight, bias, ACTIVATIONS[activation], want_params)


def group_norm(x: Tensor, num_groups: int, weight: Tensor | None = None, bias: Tensor | None = None,
               eps: float = 1e-5, activation: str | None = None) -> Tensor:
    """Group norm with an activation over channel-last ``x (N, ..., C)``: the statistics of each of
    ``num_groups`` runs of ``C / num_groups`` channels over all positions of a sample, then
    ``activation(xhat * weight + bias)`` with activation ``None``, ``"silu"`` or ``"gelu"`` (exact).

    ``x`` float32 or bfloat16; ``weight`` and ``bias`` ``(C,)`` in float32 or ``x.dtype``.  For the norm
    over each head's channels of every token pass ``x`` as ``(B * T, C)``.  Differentiable in ``x``,
    ``weight`` and ``bias``."""
    num_groups = int(num_groups)
    _norm_check(x, num_groups, weight, bias, activation)
    return L.native().norm(x, weight, bias, num_groups, eps, ACTIVATIONS[activation])


# ------------------------------------------------------------------------------------- embedding

def _embed_check(ids: Tensor, weight: Tensor) -> None:
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"ids must be int32 or int64, got {ids.dtype}")
    if weight.dim() != 2 or weight.numel() == 0:
        raise ValueError(f"weight must be (vocab, channels), got {tuple(weight.shape)}")
    _dtype_code(weight)
    _check_cuda(ids, weight)


def embedding_fused(ids: Tensor, weight: Tensor, scale: float = 1.0) -> Tensor:
    """``scale * weight[ids]`` in ``weight.dtype``; ids outside the table give rows of zeros."""
    _embed_check(ids, weight)
    return L.native().embed_fwd(ids, weight, scale)


def embedding_vjp(ids: Tensor, grad_out: Tensor, vocab: int, scale: float = 1.0) -> Tensor:
    """Dense gradient ``(vocab, channels)`` in ``grad_out.dtype``, each row's terms added in fp32 in the
    order of their positions (repeats bit for bit)."""
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"ids must be int32 or int64, got {ids.dtype}")
    if tuple(grad_out.shape[:-1]) != tuple(ids.shape) or grad_out.dim() != ids.dim() + 1 or grad_out.shape[-1] < 1:
        raise ValueError(f"grad_out must be {tuple(ids.shape)} + (channels,), got {tuple(grad_out.shape)}")
    if vocab < 1:
        raise ValueError(f"vocab must be >= 1, got {vocab}")
    _dtype_code(grad_out)
    _check_cuda(ids, grad_out)
    return L.native().embed_bwd(ids, grad_out, vocab, scale)


def embedding(ids: Tensor, weight: Tensor, scale: float = 1.0) -> Tensor:
    """Embedding lookup with scaling: ``scale * weight[ids]``, shape ``ids.shape + (C,)``, in
    ``weight.dtype`` (float32 or bfloat16; ids int32 or int64 on the same device).  Ids outside the table
    (padding) give rows of zeros and no gradient.  Differentiable in ``weight`` (dense gradient, a
    deterministic sum by sorted tokens)."""
    _embed_check(ids, weight)
    return L.native().embed(ids, weight, scale)
