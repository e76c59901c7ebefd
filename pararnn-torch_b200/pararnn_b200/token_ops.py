"""Operators around the sequence mixers of a token model: group norm with an activation over
channel-last tensors, and the embedding lookup with scaling.  Both are differentiable; the
``*_fused`` / ``*_vjp`` functions are the operators behind them.  The reference uses PyTorch's own
modules for these (``layers/para_slstm_block.py:144-152``, ``models/``)."""

from __future__ import annotations

import torch
from torch import Tensor

from . import _lib as L
from .ops import _check_cuda, _device_guard, _dtype_code, _once, _raise, _raw_stream

ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2}


def _aligned(t: Tensor) -> Tensor:
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _p(t: Tensor | None):
    return None if t is None else t.data_ptr()


def _scratch(nbytes: int, dev) -> Tensor | None:
    return torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None


# ------------------------------------------------------------------------------------ group norm

def _norm_shape(x: Tensor, num_groups: int, weight: Tensor | None, bias: Tensor | None, activation):
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {tuple(ACTIVATIONS)}, got {activation!r}")
    if x.dim() < 2:
        raise ValueError(f"x must be (N, ..., C), got {tuple(x.shape)}")
    C = x.shape[-1]
    if num_groups < 1 or C < 1 or C % num_groups:
        raise ValueError(f"num_groups={num_groups} must divide the channels ({C})")
    if x.numel() == 0:
        raise ValueError(f"x is empty: {tuple(x.shape)}")
    w_code = L.PRB_F32
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if tuple(p.shape) != (C,):
            raise ValueError(f"{name} must be ({C},), got {tuple(p.shape)}")
        if p.dtype not in (torch.float32, x.dtype):
            raise TypeError(f"{name} must be float32 or {x.dtype}, got {p.dtype}")
        w_code = _dtype_code(p)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"weight and bias must have one dtype, got {weight.dtype} and {bias.dtype}")
    N = x.shape[0]
    return N, x.numel() // (N * C), C, w_code


def _plain(p: Tensor | None) -> Tensor | None:
    return None if p is None else p.contiguous()


def group_norm_fused(x: Tensor, num_groups: int, weight: Tensor | None = None, bias: Tensor | None = None,
                     eps: float = 1e-5, activation: str | None = None, *, want_stats: bool = True):
    """``(y, stats)``: ``y`` like ``x``, ``stats (N, num_groups, 2)`` fp32 = mean and ``1/sqrt(var+eps)``."""
    N, P, C, w_code = _norm_shape(x, num_groups, weight, bias, activation)
    code = _dtype_code(x)
    dev = _check_cuda(x, weight, bias)
    xc, w, b = _aligned(x), _plain(weight), _plain(bias)
    y = torch.empty_like(xc)
    stats = torch.empty((N, num_groups, 2), dtype=torch.float32, device=dev) if want_stats else None
    lib = L.lib()
    with _device_guard(dev):
        need = lib.prb_group_norm_workspace_bytes(N, P, C, num_groups, code, 0)
        ws = _scratch(need, dev)
        rc = lib.prb_group_norm(_p(xc), _p(w), _p(b), _p(y), _p(stats), N, P, C, num_groups, eps,
                                ACTIVATIONS[activation], code, w_code, _p(ws), need, _raw_stream(dev))
    if rc:
        _raise(rc, "group_norm_fused")
    return y, stats


def group_norm_vjp(x: Tensor, grad_y: Tensor, stats: Tensor, num_groups: int, weight: Tensor | None = None,
                   bias: Tensor | None = None, activation: str | None = None, *, want_params: bool = True):
    """``(g_x, g_weight, g_bias)``; parameter gradients in the parameters' dtype, summed in fp32."""
    N, P, C, w_code = _norm_shape(x, num_groups, weight, bias, activation)
    code = _dtype_code(x)
    if tuple(grad_y.shape) != tuple(x.shape):
        raise ValueError(f"grad_y must be {tuple(x.shape)}, got {tuple(grad_y.shape)}")
    if tuple(stats.shape) != (N, num_groups, 2) or stats.dtype != torch.float32:
        raise ValueError(f"stats must be float32 {(N, num_groups, 2)}, got {stats.dtype} {tuple(stats.shape)}")
    dev = _check_cuda(x, grad_y, stats, weight, bias)
    xc, gy, w, b, st = _aligned(x), _aligned(grad_y.to(x.dtype)), _plain(weight), _plain(bias), _plain(stats)
    g_x = torch.empty_like(xc)
    g_w = torch.empty_like(w) if weight is not None and want_params else None
    g_b = torch.empty_like(b) if bias is not None and want_params else None
    lib = L.lib()
    with _device_guard(dev):
        need = lib.prb_group_norm_workspace_bytes(N, P, C, num_groups, code, 1)
        ws = _scratch(need, dev)
        rc = lib.prb_bwd_group_norm(_p(xc), _p(gy), _p(w), _p(b), _p(st), _p(g_x), _p(g_w), _p(g_b), N, P, C,
                                    num_groups, ACTIVATIONS[activation], code, w_code, _p(ws), need,
                                    _raw_stream(dev))
    if rc:
        _raise(rc, "group_norm_vjp")
    return g_x, g_w, g_b


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, num_groups, eps, activation):
        y, stats = group_norm_fused(x, num_groups, weight, bias, eps, activation)
        ctx.save_for_backward(x, weight, bias, stats)
        ctx.args = (num_groups, activation)
        return y

    @staticmethod
    def backward(ctx, grad_y):
        _once("group_norm")
        x, weight, bias, stats = ctx.saved_tensors
        num_groups, activation = ctx.args
        need = ctx.needs_input_grad
        g_x, g_w, g_b = group_norm_vjp(x, grad_y, stats, num_groups, weight, bias, activation,
                                       want_params=need[1] or need[2])
        return g_x if need[0] else None, g_w if need[1] else None, g_b if need[2] else None, None, None, None


def group_norm(x: Tensor, num_groups: int, weight: Tensor | None = None, bias: Tensor | None = None,
               eps: float = 1e-5, activation: str | None = None) -> Tensor:
    """Group norm with an activation over channel-last ``x (N, ..., C)``: the statistics of each of
    ``num_groups`` runs of ``C / num_groups`` channels over all positions of a sample, then
    ``activation(xhat * weight + bias)`` with activation ``None``, ``"silu"`` or ``"gelu"`` (exact).

    ``x`` float32 or bfloat16; ``weight`` and ``bias`` ``(C,)`` in float32 or ``x.dtype``.  For the norm
    over each head's channels of every token pass ``x`` as ``(B * T, C)``.  Differentiable in ``x``,
    ``weight`` and ``bias``."""
    return _GroupNorm.apply(x, weight, bias, int(num_groups), float(eps), activation)


# ------------------------------------------------------------------------------------- embedding

def _check_ids(ids: Tensor) -> None:
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"ids must be int32 or int64, got {ids.dtype}")


def embedding_fused(ids: Tensor, weight: Tensor, scale: float = 1.0) -> Tensor:
    """``scale * weight[ids]`` in ``weight.dtype``; ids outside the table give rows of zeros."""
    _check_ids(ids)
    if weight.dim() != 2 or weight.numel() == 0:
        raise ValueError(f"weight must be (vocab, channels), got {tuple(weight.shape)}")
    code = _dtype_code(weight)
    dev = _check_cuda(ids, weight)
    idc, w = ids.contiguous(), weight.contiguous()
    V, C = w.shape
    out = torch.empty((*ids.shape, C), dtype=w.dtype, device=dev)
    if ids.numel() == 0:
        return out
    with _device_guard(dev):
        rc = L.lib().prb_embedding(_p(idc), ids.dtype == torch.int64, _p(w), _p(out), ids.numel(), V, C, code, scale,
                                   _raw_stream(dev))
    if rc:
        _raise(rc, "embedding_fused")
    return out


def embedding_vjp(ids: Tensor, grad_out: Tensor, vocab: int, scale: float = 1.0) -> Tensor:
    """Dense gradient ``(vocab, channels)`` in ``grad_out.dtype``, each row's terms added in fp32 in the
    order of their positions (repeats bit for bit)."""
    _check_ids(ids)
    if tuple(grad_out.shape[:-1]) != tuple(ids.shape) or grad_out.dim() != ids.dim() + 1 or grad_out.shape[-1] < 1:
        raise ValueError(f"grad_out must be {tuple(ids.shape)} + (channels,), got {tuple(grad_out.shape)}")
    if vocab < 1:
        raise ValueError(f"vocab must be >= 1, got {vocab}")
    code = _dtype_code(grad_out)
    dev = _check_cuda(ids, grad_out)
    idc, g = ids.contiguous(), grad_out.contiguous()
    C = grad_out.shape[-1]
    if ids.numel() == 0:
        return torch.zeros(vocab, C, dtype=g.dtype, device=dev)
    out = torch.empty((vocab, C), dtype=g.dtype, device=dev)
    lib = L.lib()
    with _device_guard(dev):
        need = lib.prb_bwd_embedding_workspace_bytes(ids.numel(), vocab, C)
        ws = _scratch(need, dev)
        rc = lib.prb_bwd_embedding(_p(idc), ids.dtype == torch.int64, _p(g), _p(out), ids.numel(), vocab, C, code,
                                   scale, _p(ws), need, _raw_stream(dev))
    if rc:
        _raise(rc, "embedding_vjp")
    return out


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale):
        ctx.save_for_backward(ids)
        ctx.args = (weight.shape[0], scale, weight.dtype)
        return embedding_fused(ids, weight, scale)

    @staticmethod
    def backward(ctx, grad_out):
        _once("embedding")
        (ids,) = ctx.saved_tensors
        vocab, scale, dtype = ctx.args
        return None, embedding_vjp(ids, grad_out.to(dtype), vocab, scale), None


def embedding(ids: Tensor, weight: Tensor, scale: float = 1.0) -> Tensor:
    """Embedding lookup with scaling: ``scale * weight[ids]``, shape ``ids.shape + (C,)``, in
    ``weight.dtype`` (float32 or bfloat16; ids int32 or int64 on the same device).  Ids outside the table
    (padding) give rows of zeros and no gradient.  Differentiable in ``weight`` (dense gradient, a
    deterministic sum by sorted tokens)."""
    return _Embedding.apply(ids, weight, float(scale))
