"""Refusals of the token-model operators and the host-side logic around them, on the CPU: every check that
names an argument comes before any CUDA work, and CPU tensors are refused instead of computed."""

import ctypes

import pytest
import torch

import pararnn_b200 as prb
from pararnn_b200 import _lib, attn_ops, token_ops

B, T, HQ, HKV, DK, DV = 2, 5, 4, 2, 16, 8


def qkv(**kw):
    shapes = {"q": (B, T, HQ, DK), "k": (B, T, HKV, DK), "v": (B, T, HKV, DV), "g": (HKV,)}
    shapes.update(kw)
    return [torch.zeros(*s) for s in shapes.values()]


@pytest.mark.parametrize("change, error, text", [
    ({"q": (B, T, DK)}, ValueError, "q must be"),
    ({"k": (B, T, HKV, DK + 1)}, ValueError, "do not fit"),
    ({"v": (B, T + 1, HKV, DV)}, ValueError, "do not fit"),
    ({"q": (B, T, 3, DK)}, ValueError, "multiple"),
    ({"q": (B, T, HQ, 130), "k": (B, T, HKV, 130)}, TypeError, "head sizes"),
    ({"v": (B, T, HKV, 129)}, TypeError, "head sizes"),
    ({"g": (HQ,)}, ValueError, "log_decay"),
    ({"q": (B, 0, HQ, DK), "k": (B, 0, HKV, DK), "v": (B, 0, HKV, DV)}, ValueError, ">= 1"),
    ({"q": (0, T, HQ, DK), "k": (0, T, HKV, DK), "v": (0, T, HKV, DV)}, ValueError, ">= 1"),
])
def test_attention_refuses_shapes(change, error, text):
    with pytest.raises(error, match=text):
        prb.linear_attention(*qkv(**change))


def test_attention_refuses_types_devices_and_states():
    q, k, v, g = qkv()
    with pytest.raises(TypeError, match="one dtype"):
        prb.linear_attention(q, k.bfloat16(), v, g)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        prb.linear_attention(q.half(), k.half(), v.half(), g)
    with pytest.raises(RuntimeError, match="CUDA"):
        prb.linear_attention(q, k, v, g)
    with pytest.raises(TypeError, match="log_decay"):
        prb.linear_attention(q, k, v, g.requires_grad_(True))
    with pytest.raises(ValueError, match="pool"):
        prb.linear_attention(q, k, v, g.detach(), None, None, torch.zeros(B))
    with pytest.raises(TypeError, match="32 bits"):
        attn_ops._check_state(torch.zeros(B, HKV, DK, DV).bfloat16(), (B, HKV, DK, DV), "state")
    with pytest.raises(ValueError, match="state must be"):
        attn_ops._check_state(torch.zeros(B, HKV, DV, DK), (B, HKV, DK, DV), "state")


@pytest.mark.parametrize("cu, text", [
    ([0, 3], "cu_seqlens\\[-1\\]"), ([1, 5], "cu_seqlens\\[0\\]"), ([0, 3, 3, 5], "strictly"), ([0, 4, 2, 5], "strictly"),
    ([5], "S\\+1"),
])
def test_offsets_are_checked(cu, text):
    with pytest.raises(ValueError, match=text):
        attn_ops._offsets(torch.tensor(cu), 1, 5, None)


def test_offsets_pack_one_row_and_give_the_longest_sequence():
    with pytest.raises(ValueError, match="batch=1"):
        attn_ops._offsets(torch.tensor([0, 5]), 2, 5, None)
    assert attn_ops._offsets(None, 3, 7, None) == (None, 3, 7)


def step_args(**kw):
    a = dict(q=torch.zeros(B, HQ, DK), k=torch.zeros(B, HKV, DK), v=torch.zeros(B, HKV, DV), log_decay=torch.zeros(HKV),
             state=torch.zeros(B, HKV, DK, DV))
    a.update(kw)
    return a


@pytest.mark.parametrize("change, error, text", [
    (dict(q=torch.zeros(B, 2, HQ, DK)), ValueError, "one token"),
    (dict(q=torch.zeros(B, DK)), ValueError, "heads, channels"),
    (dict(k=torch.zeros(B, HKV, DK).bfloat16()), TypeError, "one dtype"),
    (dict(v=torch.zeros(B + 1, HKV, DV)), ValueError, "do not fit"),
    (dict(state=torch.zeros(B, HKV, DK, DV).bfloat16()), TypeError, "32 bits"),
    (dict(state=torch.zeros(B, HKV, DV, DK)), ValueError, "state must be"),
    (dict(state=torch.zeros(B, HKV, DV, DK).transpose(2, 3)), ValueError, "contiguous"),
    (dict(state=torch.zeros(B + 3, HKV, DK, DV)), ValueError, "block_table"),
    (dict(block_table=torch.zeros(B + 1, dtype=torch.int32)), ValueError, "block_table"),
    (dict(block_table=torch.zeros(B)), TypeError, "int32 or int64"),
    (dict(q=torch.zeros(B, HQ, DK, requires_grad=True)), RuntimeError, "no backward"),
    (dict(), RuntimeError, "CUDA"),
])
def test_step_refuses(change, error, text):
    with pytest.raises(error, match=text):
        prb.linear_attention_step(**step_args(**change))


@pytest.mark.parametrize("kw, error, text", [
    (dict(num_groups=3), ValueError, "divide"),
    (dict(num_groups=0), ValueError, "divide"),
    (dict(x=torch.zeros(8)), ValueError, "N, ..., C"),
    (dict(x=torch.zeros(0, 8)), ValueError, "empty"),
    (dict(activation="relu6"), ValueError, "activation"),
    (dict(weight=torch.zeros(7)), ValueError, "weight"),
    (dict(weight=torch.zeros(8).half()), TypeError, "weight"),
    (dict(weight=torch.zeros(8), bias=torch.zeros(8).bfloat16(), x=torch.zeros(2, 8).bfloat16()), TypeError, "one dtype"),
    (dict(x=torch.zeros(2, 8).half()), TypeError, "float32 or bfloat16"),
    (dict(), RuntimeError, "CUDA"),
])
def test_group_norm_refuses(kw, error, text):
    args = dict(x=torch.zeros(2, 8), num_groups=2)
    args.update(kw)
    with pytest.raises(error, match=text):
        prb.group_norm(**args)


def test_group_norm_vjp_refuses():
    x = torch.zeros(2, 3, 8)
    # the arguments that the forward has too are checked first, and a CPU tensor ends there
    with pytest.raises(ValueError, match="divide"):
        token_ops.group_norm_vjp(x, x, torch.zeros(2, 3, 2), 3)
    with pytest.raises(RuntimeError, match="CUDA"):
        token_ops.group_norm_vjp(x, x, torch.zeros(2, 2, 2), 2)


@pytest.mark.parametrize("ids, weight, error, text", [
    (torch.zeros(3), torch.zeros(4, 2), TypeError, "ids"),
    (torch.zeros(3, dtype=torch.long), torch.zeros(4), ValueError, "weight"),
    (torch.zeros(3, dtype=torch.long), torch.zeros(0, 2), ValueError, "weight"),
    (torch.zeros(3, dtype=torch.long), torch.zeros(4, 2).half(), TypeError, "float32 or bfloat16"),
    (torch.zeros(3, dtype=torch.long), torch.zeros(4, 2), RuntimeError, "CUDA"),
])
def test_embedding_refuses(ids, weight, error, text):
    with pytest.raises(error, match=text):
        prb.embedding(ids, weight)
    if weight.dim() == 2 and weight.numel():
        with pytest.raises(error):
            token_ops.embedding_vjp(ids, torch.zeros(3, 2, dtype=weight.dtype), 4)


def test_c_entry_points_check_arguments_before_any_gpu_work():
    lib = _lib.lib()
    null = None
    buf = ctypes.create_string_buffer(512)
    p = (ctypes.addressof(buf) + 255) & ~255
    h = ctypes.byref(_lib.Heads(p, 1, 1, 1))
    bad, ws, unsupported = -1, -2, -3

    def fwd(q=h, decay=p, out=p, rows=1, time=4, n_seq=1, longest=4, hq=2, hkv=2, dk=8, dv=8, dtype=1, cu=null):
        return lib.prb_linear_attention(q, h, h, decay, null, cu, out, null, rows, time, n_seq, longest, hq, hkv, dk, dv,
                                        dtype, 1.0, null, 0, null)

    assert fwd(q=null) == bad and fwd(decay=null) == bad and fwd(out=null) == bad
    assert fwd(rows=0) == bad and fwd(time=0) == bad and fwd(dtype=7) == bad and fwd(longest=5) == bad
    assert fwd(n_seq=2) == bad  # rectangular: one sequence for each row
    assert fwd(hq=3) == unsupported and fwd(dk=129) == unsupported and fwd(dv=136) == unsupported
    assert fwd(rows=1, time=1 << 20, longest=1 << 20) == ws  # cut into segments: needs a workspace
    n = lib.prb_linear_attention_workspace_bytes(1, 1 << 20, 1, 1 << 20, 2, 2, 8, 8, 1, 0, 0)
    assert n > 0 and lib.prb_linear_attention_workspace_bytes(1, 1 << 20, 1, 1 << 20, 2, 2, 8, 8, 1, 0, 1) > 0
    assert lib.prb_linear_attention_workspace_bytes(64, 128, 64, 128, 8, 8, 64, 64, 1, 0, 1) == 0
    assert lib.prb_bwd_linear_attention(h, h, h, null, p, null, null, null, p, p, p, null, 1, 4, 1, 4, 2, 2, 8, 8, 1, 1.0,
                                        null, 0, null) == bad
    step = lambda **k: lib.prb_linear_attention_step(  # noqa: E731
        p, p, p, p, k.get("state", p), k.get("table"), 0, p, k.get("rows", 2), k.get("slots", 2), 2, k.get("hkv", 2), 8,
        k.get("dv", 8), 0, 1.0, null)
    assert step(state=null) == bad and step(rows=0) == bad and step(slots=3) == bad
    assert step(hkv=4) == unsupported and step(dv=200) == unsupported
    norm = lambda **k: lib.prb_group_norm(  # noqa: E731
        k.get("x", p), null, null, p, null, k.get("n", 2), k.get("pos", 3), k.get("c", 8), k.get("g", 2), 1e-5,
        k.get("act", 0), k.get("dtype", 0), 0, null, 0, null)
    assert norm(x=null) == bad and norm(x=p + 4) == bad and norm(n=0) == bad and norm(g=3) == bad
    assert norm(act=3) == bad and norm(dtype=2) == bad and norm() == ws
    assert lib.prb_group_norm_workspace_bytes(4, 1, 64, 8, 1, 0) == 0
    assert lib.prb_group_norm_workspace_bytes(4, 1, 64, 8, 1, 1) > 0
    assert lib.prb_embedding(null, 1, p, p, 4, 4, 4, 0, 1.0, null) == bad
    assert lib.prb_embedding(p, 1, p, p, 0, 4, 4, 0, 1.0, null) == bad
    assert lib.prb_embedding(p, 1, p, p, 1 << 32, 4, 4, 0, 1.0, null) == unsupported
    assert lib.prb_bwd_embedding(p, 1, p, p, 4, 4, 4, 0, 1.0, null, 0, null) == ws
    assert lib.prb_bwd_embedding_workspace_bytes(1000, 10, 16) > lib.prb_bwd_embedding_workspace_bytes(10, 10, 16) > 0


def test_layers_are_built_and_refuse_what_they_cannot_do():
    layer = prb.LinearAttention(64, 4, n_kv_heads=2, d_value=32)
    assert layer.W_qkv.weight.shape == (4 * 16 + 2 * (16 + 32), 64) and layer.W_o.weight.shape == (64, 4 * 32)
    assert layer.log_decay.shape == (2,) and bool((layer.log_decay < 0).all())
    assert "log_decay" in layer.state_dict() and not layer.log_decay.requires_grad
    assert layer.zero_state(3).shape == (3, 2, 16, 32)
    schedule = layer.log_decay.clone()
    assert torch.equal(layer.bfloat16().log_decay, schedule) and layer.W_o.weight.dtype == torch.bfloat16
    for bad in (dict(n_heads=3), dict(n_heads=4, n_kv_heads=3)):
        with pytest.raises(ValueError):
            prb.LinearAttention(64, **bad)
    with pytest.raises(ValueError, match="activation"):
        prb.LinearAttention(64, 4, activation="relu")
    emb = prb.TokenEmbedding(10, 16)
    assert emb.scale == 4.0 and emb.weight.shape == (10, 16)
    rnn = prb.ParaRNN(prb.ParaNLRU(16, 16), embedding=emb)
    with pytest.raises(ValueError, match="embedding"):
        prb.ParaRNN(prb.ParaNLRU(8, 8), embedding=emb)
    with pytest.raises(RuntimeError, match="CUDA"):
        rnn(torch.zeros(2, 3, dtype=torch.long))
    with pytest.raises(TypeError, match="embedding"):
        prb.ParaRNN(prb.ParaNLRU(16, 16))(torch.zeros(2, 3, dtype=torch.long))


def test_fake_kernels_on_meta_tensors():
    ns = torch.ops.pararnn_b200
    m = lambda *s, dtype=torch.bfloat16: torch.empty(*s, dtype=dtype, device="meta")  # noqa: E731
    q, k, v, g = m(1, T, HQ, DK), m(1, T, HKV, DK), m(1, T, HKV, DV), m(HKV, dtype=torch.float32)
    cu = m(4, dtype=torch.int32)
    o, s = ns.linear_attention_fused(q, k, v, g, None, cu)
    assert o.shape == (1, T, HQ, DV) and o.dtype == torch.bfloat16 and s.shape == (3, HKV, DK, DV)
    gq, gk, gv, gs = ns.reverse_linear_attention_vjp(q, k, v, g, o)
    assert (gq.shape, gk.shape, gv.shape, gs.shape) == (q.shape, k.shape, v.shape, (1, HKV, DK, DV))
    assert gs.dtype == torch.float32
    out = ns.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, m(1, HKV, DK, DV, dtype=torch.float32))
    assert out.shape == (1, HQ, DV)
    y, st = ns.group_norm_fused(m(3, 7, 8), 2)
    assert y.shape == (3, 7, 8) and st.shape == (3, 2, 2)
    gx, gw, gb = ns.group_norm_vjp(m(3, 7, 8), y, st, 2, m(8), m(8))
    assert gx.shape == y.shape and gw.shape == gb.shape == (8,)
    e = ns.embedding_fused(m(2, 5, dtype=torch.int64), m(11, 8), 2.0)
    assert e.shape == (2, 5, 8) and ns.embedding_vjp(m(2, 5, dtype=torch.int64), e, 11).shape == (11, 8)
