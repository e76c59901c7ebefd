"""Linear attention with a decay for each head: a matrix-state sequence mixer next to the cells.

``S_t = w S_{t-1} + k_t v_t^T``, ``o_t = scale q_t S_t`` with ``w = exp(log_decay[h])``.  Unlike the
cells its recurrence is linear in the state, so there is nothing to iterate: one call evaluates the
whole sequence in chunks, and ``linear_attention_step`` is the single-token form on a pool of states
(the counterpart of ``decode_step``).  The reference's matrix-state cells are ``cells/para_m2rnn.py``
and ``cells/para_rwkv7.py``; this mixer has no counterpart there.

``linear_attention`` is differentiable; ``linear_attention_fused`` and
``linear_attention_reverse_vjp`` are the two operators behind it.
"""

from __future__ import annotations

import torch
from torch import Tensor

from . import _lib as L
from .ops import _attention_devices, _check_cuda, _dtype_code, gather_h0, validate_cu_seqlens

MAX_HEAD_DIM = 128


def _shapes(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor):
    """(B, T, Hq, Hkv, dk, dv) after the argument checks."""
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != 4:
            raise ValueError(f"{name} must be (B, T, heads, channels), got {tuple(t.shape)}")
        if t.dtype != q.dtype:
            raise TypeError(f"q, k, v must have one dtype, got {q.dtype} and {t.dtype} ({name})")
    B, T, Hq, dk = q.shape
    Hkv, dv = k.shape[2], v.shape[3]
    if tuple(k.shape) != (B, T, Hkv, dk) or tuple(v.shape) != (B, T, Hkv, dv):
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not fit together")
    _check_heads(Hq, Hkv, dk, dv, log_decay)
    if T < 1 or B < 1:
        raise ValueError("batch and time must be >= 1")
    return B, T, Hq, Hkv, dk, dv


def _check_heads(Hq: int, Hkv: int, dk: int, dv: int, log_decay: Tensor) -> None:
    if Hkv < 1 or Hq < 1 or Hq % Hkv:
        raise ValueError(f"query heads ({Hq}) must be a multiple of key / value heads ({Hkv})")
    if not (1 <= dk <= MAX_HEAD_DIM and 1 <= dv <= MAX_HEAD_DIM):
        raise TypeError(f"the CUDA backend covers head sizes 1..{MAX_HEAD_DIM}, got dk={dk}, dv={dv}")
    if log_decay.shape != (Hkv,):
        raise ValueError(f"log_decay must be ({Hkv},), one for each key / value head, got {tuple(log_decay.shape)}")


def _check_state(state: Tensor | None, shape: tuple[int, ...], name: str) -> Tensor | None:
    if state is None:
        return None
    if state.dtype != torch.float32:
        raise TypeError(f"{name} must be float32 (states are kept in 32 bits), got {state.dtype}")
    if tuple(state.shape) != shape:
        raise ValueError(f"{name} must be {shape}, got {tuple(state.shape)}")
    return state


def _offsets(cu_seqlens: Tensor | None, batch: int, time: int, dev):
    """(device int32 offsets, sequences, longest sequence).  Offsets are checked on the host, which
    reads a CUDA tensor back; while a CUDA graph is being captured that is not possible, so they
    have to be int32 on the device and the kernels clamp what a replay finds there."""
    if cu_seqlens is None:
        return None, batch, time
    if batch != 1:
        raise ValueError(f"cu_seqlens packs x with batch=1, got batch={batch}")
    if dev is not None and torch.cuda.is_current_stream_capturing():
        if not cu_seqlens.is_cuda or cu_seqlens.dtype != torch.int32 or not cu_seqlens.is_contiguous():
            raise RuntimeError("a CUDA graph needs cu_seqlens as a contiguous int32 CUDA tensor")
        if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2:
            raise ValueError(f"cu_seqlens must be (S+1,), got {tuple(cu_seqlens.shape)}")
        if cu_seqlens.device != dev:
            raise RuntimeError(f"tensors on different devices: {dev} and {cu_seqlens.device}")
        return cu_seqlens, cu_seqlens.numel() - 1, time
    cs = validate_cu_seqlens(cu_seqlens, time)
    longest = max(b - a for a, b in zip(cs[:-1], cs[1:]))
    return cu_seqlens.to(device=dev, dtype=torch.int32).contiguous(), len(cs) - 1, longest


def _decay(log_decay: Tensor) -> Tensor:
    return log_decay.detach().to(torch.float32).contiguous()


def _prepare(q, k, v, log_decay, state, cu_seqlens, scale):
    """Checks, and the trailing arguments of the native operators: (cu, sequences, longest, scale, sparse)."""
    B, T, Hq, Hkv, dk, dv = _shapes(q, k, v, log_decay)
    _dtype_code(q)
    dev = _check_cuda(q, k, v, log_decay, state)
    cu, n_seq, longest = _offsets(cu_seqlens, B, T, dev)
    _check_state(state, (n_seq, Hkv, dk, dv), "state")
    _attention_devices.add(dev)
    # checked offsets cover every token; those that a graph replays with may not, and tokens that no
    # sequence holds give zeros
    sparse = cu is not None and torch.cuda.is_current_stream_capturing()
    return (B, T, Hq, Hkv, dk, dv), cu, n_seq, longest, dk ** -0.5 if scale is None else float(scale), sparse


def linear_attention_fused(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, state: Tensor | None = None,
                           cu_seqlens: Tensor | None = None, *, scale: float | None = None,
                           want_state: bool = True):
    """``(o, final state or None)``: ``o (B,T,Hq,dv)`` in ``q.dtype``, states fp32 ``(n_seq,Hkv,dk,dv)``."""
    _, cu, n_seq, longest, scale, sparse = _prepare(q, k, v, log_decay, state, cu_seqlens, scale)
    return L.native().attention_fwd(q, k, v, _decay(log_decay), state, cu, n_seq, longest, scale, want_state, sparse)


def linear_attention_reverse_vjp(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, grad_out: Tensor,
                                 state: Tensor | None = None, grad_state: Tensor | None = None,
                                 cu_seqlens: Tensor | None = None, *, scale: float | None = None,
                                 want_state: bool = False):
    """``(g_q, g_k, g_v, g_state or None)`` from the cotangents of the output and of the final state.
    Gradients of shared key / value heads are summed over their query heads in fp32."""
    shape, cu, n_seq, longest, scale, sparse = _prepare(q, k, v, log_decay, state, cu_seqlens, scale)
    B, T, Hq, Hkv, dk, dv = shape
    if tuple(grad_out.shape) != (B, T, Hq, dv):
        raise ValueError(f"grad_out must be {(B, T, Hq, dv)}, got {tuple(grad_out.shape)}")
    _check_state(grad_state, (n_seq, Hkv, dk, dv), "grad_state")
    _check_cuda(q, grad_out, grad_state)
    return L.native().attention_bwd(q, k, v, _decay(log_decay), grad_out, state, grad_state, cu, n_seq, longest, scale,
                                    want_state, sparse)


def linear_attention(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, state: Tensor | None = None,
                     cu_seqlens: Tensor | None = None, block_table: Tensor | None = None, *,
                     scale: float | None = None, return_state: bool = False):
    """Linear attention with a decay for each head over whole sequences, differentiable in ``q``, ``k``,
    ``v`` and ``state``.

    ``q (B,T,Hq,dk)``, ``k (B,T,Hkv,dk)``, ``v (B,T,Hkv,dv)`` in float32 or bfloat16 (views with a unit
    channel stride are read in place), ``Hq`` a multiple of ``Hkv`` (query head ``h`` reads state head
    ``h // (Hq // Hkv)``), ``dk, dv <= 128``; ``log_decay (Hkv,) <= 0`` is a fixed schedule, not a
    parameter; ``state (B,Hkv,dk,dv)`` float32 is the initial state.  With ``cu_seqlens`` the batch is
    packed ``(1,N,...)`` and ``state`` has one row for each sequence; with ``block_table`` ``state`` is a
    pool and row ``i`` starts from slot ``block_table[i]``.  ``scale`` defaults to ``dk ** -0.5``.
    Returns ``o (B,T,Hq,dv)``, or ``(o, final states)`` with ``return_state=True``."""
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise TypeError("log_decay is a fixed schedule of the heads and has no gradient: detach it")
    if block_table is not None:
        if state is None or state.dim() != 4:
            raise ValueError("block_table needs state as a pool (C, Hkv, dk, dv)")
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("block_table is checked on the host, which a CUDA graph cannot do: pass state's rows")
        rows = q.shape[0] if cu_seqlens is None else cu_seqlens.numel() - 1
        state = gather_h0(state, block_table, rows, (k.shape[2], k.shape[3], v.shape[3]))
    _, cu, n_seq, longest, scale, sparse = _prepare(q, k, v, log_decay, state, cu_seqlens, scale)
    out, s_out = L.native().attention(q, k, v, _decay(log_decay), state, cu, n_seq, longest, scale, return_state,
                                      sparse)
    return (out, s_out) if return_state else out


def linear_attention_step(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, state: Tensor, *,
                          scale: float | None = None, block_table: Tensor | None = None,
                          out: Tensor | None = None) -> Tensor:
    """One token for each row: updates ``state`` in place and returns ``o (B,Hq,dv)``.

    ``q (B,Hq,dk)``, ``k (B,Hkv,dk)``, ``v (B,Hkv,dv)`` (or with a time axis of length 1, which the
    result then has too); ``state`` is a contiguous float32 ``(B,Hkv,dk,dv)``, or with ``block_table``
    ``(B,)`` a pool ``(C,Hkv,dk,dv)`` whose named slots are updated.  Slots outside the pool mark padding
    rows: they touch no state and their outputs are zero.  A slot that several rows name takes
    them in row order.  ``out`` and ``state`` share no memory with one another or with an input (``out``
    may be ``v`` itself where ``Hq = Hkv``).  One launch, no allocation with ``out=``: CUDA graphs can
    capture it."""
    # this call is the latency of a token: its checks are kept short
    if (q.requires_grad or k.requires_grad or v.requires_grad or log_decay.requires_grad or state.requires_grad) \
            and torch.is_grad_enabled():
        raise RuntimeError("linear_attention_step has no backward: call it under torch.no_grad()")
    timed = q.dim() == 4
    if timed:
        if any(t.dim() != 4 or t.shape[1] != 1 for t in (q, k, v)):
            raise ValueError("linear_attention_step takes one token: time axes must have length 1")
        q, k, v = q[:, 0], k[:, 0], v[:, 0]
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError("q, k, v must be (B, heads, channels), got "
                         f"{tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"q, k, v must have one dtype, got {q.dtype}, {k.dtype}, {v.dtype}")
    B, Hq, dk = q.shape
    Hkv, dv = k.shape[1], v.shape[2]
    if k.shape != (B, Hkv, dk) or v.shape != (B, Hkv, dv):
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not fit together")
    _check_heads(Hq, Hkv, dk, dv, log_decay)
    if B < 1:
        raise ValueError("batch must be >= 1")
    if state.dtype != torch.float32:
        raise TypeError(f"state must be float32 (states are kept in 32 bits), got {state.dtype}")
    if state.dim() != 4 or state.shape[1:] != (Hkv, dk, dv) or state.shape[0] < 1:
        raise ValueError(f"state must be (slots, {Hkv}, {dk}, {dv}), got {tuple(state.shape)}")
    if not state.is_contiguous():
        raise ValueError("linear_attention_step updates state in place: it must be contiguous")
    if block_table is None and state.shape[0] != B:
        raise ValueError(f"state has {state.shape[0]} rows for a batch of {B}: pass block_table for a pool")
    if block_table is not None:
        if block_table.dim() != 1 or block_table.numel() != B:
            raise ValueError(f"block_table must be ({B},), got {tuple(block_table.shape)}")
        if block_table.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"block_table must be int32 or int64, got {block_table.dtype}")
    _dtype_code(q)
    dev = _check_cuda(q, k, v, log_decay, state)
    shape = (B, 1, Hq, dv) if timed else (B, Hq, dv)
    if out is None:
        out = torch.empty(shape, dtype=q.dtype, device=dev)
    elif out.shape != shape or out.dtype != q.dtype or out.device != dev or not out.is_contiguous():
        raise ValueError(f"out must be contiguous {shape} {q.dtype} on {dev}")
    elif out.data_ptr() in (q.data_ptr(), k.data_ptr()):
        raise ValueError("out must not be q or k: other heads still read them")
    if block_table is not None and not block_table.is_cuda:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a CUDA graph needs block_table on the device")
        block_table = block_table.to(dev)
    elif block_table is not None:
        _check_cuda(q, block_table)
    L.native().attention_step(q, k, v, _decay(log_decay), state, block_table, dk ** -0.5 if scale is None else scale,
                              out)
    return out
