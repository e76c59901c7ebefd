"""Layers: ``ParaRNN``, the sequence wrapper that trains with the parallel Newton solve and evaluates with
the sequential unroll (reference ``layers/para_rnn.py:187-288``); ``LinearAttention``, the matrix-state
mixer with a decay for each head; ``TokenEmbedding``, the input side of a token model."""

from __future__ import annotations

import copy
import math

import torch
from torch import Tensor, nn

from .attn_ops import linear_attention, linear_attention_step
from .config import NewtonConfig, NewtonStats
from .newton import newton_apply
from .sequential import sequential_apply
from .token_ops import ACTIVATIONS, embedding, group_norm


class TokenEmbedding(nn.Module):
    """``scale * weight[ids]``; ``scale`` defaults to ``sqrt(d)`` (unit variance at the usual
    ``1 / sqrt(d)`` initialisation).  Ids outside the table are padding: rows of zeros, no gradient."""

    def __init__(self, vocab: int, d: int, *, scale: float | None = None, device=None, dtype=None):
        super().__init__()
        self.scale = math.sqrt(d) if scale is None else float(scale)
        self.weight = nn.Parameter(torch.empty(vocab, d, device=device, dtype=dtype))
        nn.init.normal_(self.weight, std=d ** -0.5)

    def forward(self, ids: Tensor) -> Tensor:
        return embedding(ids, self.weight, self.scale)


class LinearAttention(nn.Module):
    """Linear attention mixer: projections, ``linear_attention`` with a fixed decay schedule
    (``1 - 2^-3`` to ``1 - 2^-9`` over the key / value heads), a group norm over every head's channels
    with an activation, output projection.  ``forward`` takes whole (or packed) sequences, ``step``
    one token for each row on a pool of states."""

    def __init__(self, d_model: int, n_heads: int, *, n_kv_heads: int | None = None, d_value: int | None = None,
                 activation: str | None = "silu", eps: float = 1e-5, device=None, dtype=None):
        super().__init__()
        n_kv_heads = n_heads if n_kv_heads is None else n_kv_heads
        if n_heads < 1 or d_model % n_heads or n_kv_heads < 1 or n_heads % n_kv_heads:
            raise ValueError(f"n_heads={n_heads} must divide d_model={d_model} and be a multiple of "
                             f"n_kv_heads={n_kv_heads}")
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {tuple(ACTIVATIONS)}, got {activation!r}")
        kw = {"device": device, "dtype": dtype}
        self.n_heads, self.n_kv_heads = n_heads, n_kv_heads
        self.d_key = d_model // n_heads
        self.d_value = self.d_key if d_value is None else d_value
        self.activation, self.eps = activation, eps
        self.W_qkv = nn.Linear(d_model, n_heads * self.d_key + n_kv_heads * (self.d_key + self.d_value), bias=False, **kw)
        self.W_o = nn.Linear(n_heads * self.d_value, d_model, bias=False, **kw)
        self.norm_weight = nn.Parameter(torch.ones(n_heads * self.d_value, **kw))
        self.norm_bias = nn.Parameter(torch.zeros(n_heads * self.d_value, **kw))
        spread = torch.linspace(3.0, 9.0, n_kv_heads, device=device)
        self.register_buffer("log_decay", torch.log1p(-torch.exp2(-spread)).float())

    def _apply(self, fn, *args, **kw):
        # the schedule stays in float32 when the module is cast
        kept = self.log_decay
        super()._apply(fn, *args, **kw)
        if self.log_decay.dtype != kept.dtype and not self.log_decay.is_meta:
            self.log_decay = kept.to(self.log_decay.device)
        return self

    def zero_state(self, rows: int) -> Tensor:
        return torch.zeros(rows, self.n_kv_heads, self.d_key, self.d_value, device=self.W_qkv.weight.device)

    def _qkv(self, x: Tensor):
        y = self.W_qkv(x)
        nq, nk = self.n_heads * self.d_key, self.n_kv_heads * self.d_key
        return (y[..., :nq].unflatten(-1, (self.n_heads, self.d_key)),
                y[..., nq:nq + nk].unflatten(-1, (self.n_kv_heads, self.d_key)),
                y[..., nq + nk:].unflatten(-1, (self.n_kv_heads, self.d_value)))

    def _out(self, o: Tensor) -> Tensor:
        lead = o.shape[:-2]
        h = group_norm(o.reshape(-1, self.n_heads * self.d_value), self.n_heads, self.norm_weight, self.norm_bias,
                       self.eps, self.activation)
        return self.W_o(h.view(*lead, -1))

    def forward(self, x: Tensor, state: Tensor | None = None, cu_seqlens: Tensor | None = None,
                block_table: Tensor | None = None, *, return_state: bool = False):
        q, k, v = self._qkv(x)
        r = linear_attention(q, k, v, self.log_decay, state, cu_seqlens, block_table, return_state=return_state)
        return (self._out(r[0]), r[1]) if return_state else self._out(r)

    @torch.no_grad()
    def step(self, x: Tensor, state: Tensor, *, block_table: Tensor | None = None) -> Tensor:
        """``x (B, d_model)`` -> ``(B, d_model)``; the named slots of ``state`` are updated in place."""
        q, k, v = self._qkv(x)
        return self._out(linear_attention_step(q, k, v, self.log_decay, state, block_table=block_table))


class ParaRNN(nn.Module):
    """``embedding`` (a ``TokenEmbedding``) makes the layer take token ids in the place of vectors."""

    def __init__(self, cell: nn.Module, *, config: NewtonConfig | None = None, num_layers: int = 1,
                 batch_first: bool = True, output_hidden: bool = True, embedding: nn.Module | None = None):
        super().__init__()
        if embedding is not None and embedding.weight.shape[1] != cell.d_in:
            raise ValueError(f"embedding has {embedding.weight.shape[1]} channels, the cell takes {cell.d_in}")
        if num_layers < 1:
            raise ValueError("num_layers must be >= 1")
        if num_layers > 1 and cell.d_in != cell.d_h:
            raise ValueError("stacking needs d_in == d_h")
        self.cells = nn.ModuleList([cell] + [copy.deepcopy(cell) for _ in range(num_layers - 1)])
        for extra in self.cells[1:]:
            extra.reset_parameters()
        self.embedding = embedding
        self.config = config or NewtonConfig()
        self.batch_first = batch_first
        self.output_hidden = output_hidden
        self.last_stats: NewtonStats | None = None

    @property
    def cell(self) -> nn.Module:
        return self.cells[0]

    def forward(self, x: Tensor, h0: Tensor | None = None) -> Tensor:
        if not self.batch_first:
            x = x.transpose(0, 1)
        if x.dtype in (torch.int32, torch.int64):
            if self.embedding is None:
                raise TypeError("ParaRNN takes token ids only with an embedding")
            x = self.embedding(x)
        out = x
        for i, cell in enumerate(self.cells):
            h0_i = h0 if (h0 is not None and i == 0) else None
            slot = getattr(cell, "hidden_slot", None)
            hidden = slot is not None and (self.output_hidden or i + 1 < len(self.cells))
            if self.training:
                stats = NewtonStats()
                # the hidden slot straight from the solve: its backward takes the (B,T,d) cotangent
                out = newton_apply(cell, out, self.config, h0=h0_i, stats=stats,
                                   output_slot=slot if hidden else None)
                self.last_stats = stats
            else:
                states = sequential_apply(cell, out, h0_i)
                out = states[:, :, slot] if hidden else states
        if not self.batch_first:
            out = out.transpose(0, 1)
        return out
