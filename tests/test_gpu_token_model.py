"""The token-model operators as they are used together: embedding -> linear attention mixer (projections,
linear attention, group norm with its activation) -> gradients, against the same model in 64 bits on the
CPU; prompt and single-token forms of the mixer; token ids into ``ParaRNN``."""

import pytest
import torch

import pararnn_b200 as prb
from token_util import attention_oracle, norm_oracle

pytestmark = pytest.mark.gpu


def model64(params, ids, layer, scale, cu=None):
    """The embedding and the mixer in float64; ``params``: name -> leaf."""
    x = params["emb"][ids] * scale
    y = x @ params["W_qkv"].t()
    nq, nk = layer.n_heads * layer.d_key, layer.n_kv_heads * layer.d_key
    q = y[..., :nq].unflatten(-1, (layer.n_heads, layer.d_key))
    k = y[..., nq:nq + nk].unflatten(-1, (layer.n_kv_heads, layer.d_key))
    v = y[..., nq + nk:].unflatten(-1, (layer.n_kv_heads, layer.d_value))
    o, _ = attention_oracle(q, k, v, layer.log_decay.cpu(), cu=cu)
    h = norm_oracle(o.reshape(-1, layer.n_heads * layer.d_value), layer.n_heads, params["norm_weight"],
                    params["norm_bias"], layer.eps, layer.activation)
    return h.view(*ids.shape, -1) @ params["W_o"].t()


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("kw", [dict(n_heads=4), dict(n_heads=4, n_kv_heads=2, d_value=24, activation="gelu")])
def test_embedding_mixer_and_all_gradients_match_64_bits(kw, packed):
    """Five stages (lookup, projection, attention, norm, projection) of sums with at most 300 terms, each within
    2^-15 of the sum of its terms' sizes in fp32; the norm divides by a spread of at least an eighth of its
    inputs' size.  Against the largest entry: 5 * 2^-15 * 2^3 < 2^-9."""
    torch.manual_seed(0)
    V, D, B, T = 50, 64, 1 if packed else 2, 210
    emb = prb.TokenEmbedding(V, D).cuda()
    layer = prb.LinearAttention(D, **kw).cuda()
    with torch.no_grad():
        layer.norm_bias.uniform_(-0.2, 0.2)
    ids = torch.randint(0, V, (B, T))
    cu = [0, 3, 140, 210] if packed else None
    out = layer(emb(ids.cuda()), cu_seqlens=None if cu is None else torch.tensor(cu))
    grad = torch.randn(out.shape)
    named = {"emb": emb.weight, "W_qkv": layer.W_qkv.weight, "W_o": layer.W_o.weight,
             "norm_weight": layer.norm_weight, "norm_bias": layer.norm_bias}
    got = torch.autograd.grad(out, list(named.values()), grad.cuda())
    leaves = {n: p.detach().cpu().double().requires_grad_(True) for n, p in named.items()}
    want = model64(leaves, ids, layer, emb.scale, cu)
    near = lambda a, b: float((a.detach().double().cpu() - b.detach()).abs().max() / b.detach().abs().max())  # noqa: E731
    assert near(out, want) <= 2 ** -9
    for n, a, b in zip(named, got, torch.autograd.grad(want, list(leaves.values()), grad.double())):
        assert near(a, b) <= 2 ** -9, n


def test_mixer_prompt_then_steps_equal_the_whole_sequence():
    """A server's run: prompts in one packed call, the states into pool slots, then tokens one by one.  In fp32
    both forms add the same terms; the bound is that of the test above."""
    torch.manual_seed(1)
    layer = prb.LinearAttention(64, 4, n_kv_heads=2).cuda()
    lens, more = [17, 1, 133], 4
    xs = [torch.randn(n + more, 64, device="cuda") for n in lens]
    cu = torch.tensor([0, 17, 18, 151])
    pool = layer.zero_state(6)
    slots = torch.tensor([4, 0, 2], device="cuda")
    with torch.no_grad():
        whole = [layer(x[None]) for x in xs]
        y, s = layer(torch.cat([x[:n] for x, n in zip(xs, lens)])[None], cu_seqlens=cu, return_state=True)
        pool.index_copy_(0, slots, s)
        size = max(float(w.abs().max()) for w in whole)
        for i, n in enumerate(lens):
            assert float((y[0, cu[i]:cu[i + 1]] - whole[i][0, :n]).abs().max()) <= 2 ** -9 * size
        for t in range(more):
            y = layer.step(torch.stack([x[n + t] for x, n in zip(xs, lens)]), pool, block_table=slots)
            for i, n in enumerate(lens):
                assert float((y[i] - whole[i][0, n + t]).abs().max()) <= 2 ** -9 * size


def test_para_rnn_takes_token_ids():
    torch.manual_seed(2)
    emb = prb.TokenEmbedding(40, 32).cuda()
    rnn = prb.ParaRNN(prb.ParaNLRU(32, 32), embedding=emb).cuda()
    ids = torch.randint(-1, 40, (2, 70), device="cuda")
    out = rnn(ids)
    vectors = torch.where((ids >= 0)[..., None], emb.weight[ids.clamp(min=0)] * emb.scale, 0.0)
    x = vectors.detach().requires_grad_(True)
    want = rnn(x)
    assert torch.equal(out, want)
    g = torch.randn_like(out)
    (gx,) = torch.autograd.grad(want, [x], g)
    (gw,) = torch.autograd.grad(out, [emb.weight], g)
    ref = torch.zeros(40, 32, dtype=torch.float64, device="cuda")
    live = ids.flatten() >= 0
    ref.index_add_(0, ids.flatten()[live], gx.double().flatten(0, 1)[live] * emb.scale)
    size = torch.zeros_like(ref).index_add_(0, ids.flatten()[live], gx.double().abs().flatten(0, 1)[live] * emb.scale)
    assert float(((gw.double() - ref).abs() - 140 * 2 ** -23 * size).max()) <= 0
    rnn.eval()
    assert rnn(ids).shape == out.shape


def test_a_training_step_in_a_graph():
    """Forward, backward and the gradients' operators captured through autograd with leaves of their own."""
    torch.manual_seed(3)
    q, k, v = (torch.randn(2, 300, 2, 64, device="cuda").bfloat16().requires_grad_(True) for _ in range(3))
    w = torch.ones(128, device="cuda").bfloat16().requires_grad_(True)
    g = torch.tensor([-0.05, -0.3], device="cuda")
    do = torch.randn(600, 128, device="cuda").bfloat16()

    def step():
        o = prb.linear_attention(q, k, v, g)
        y = prb.group_norm(o.view(600, 128), 2, w, activation="silu")
        return torch.autograd.grad(y, [q, k, v, w], do)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for _ in range(2):
        with torch.no_grad():
            q.copy_(torch.randn_like(q))
            do.copy_(torch.randn_like(do))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, step()):
            assert torch.equal(a, b)


def test_double_backward_is_refused():
    x = torch.randn(4, 8, device="cuda", requires_grad=True)
    y = prb.group_norm(x, 2)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(y.sum(), [x], create_graph=True)


def test_custom_ops_match_the_functions():
    ns = torch.ops.pararnn_b200
    q, k, v = (torch.randn(1, 50, 2, 64, device="cuda").bfloat16() for _ in range(3))
    g = torch.tensor([-0.05, -0.3], device="cuda")
    o, s = ns.linear_attention_fused(q, k, v, g)
    want = prb.linear_attention(q, k, v, g, return_state=True)
    assert torch.equal(o, want[0]) and torch.equal(s, want[1])
    pool, ref = s.clone(), s.clone()
    a = ns.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, pool)
    b = prb.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, ref)
    assert torch.equal(a, b) and torch.equal(pool, ref)
    x = torch.randn(6, 64, device="cuda")
    assert torch.equal(ns.group_norm_fused(x, 4, None, None, 1e-5, "silu")[0], prb.group_norm(x, 4, activation="silu"))
    w, ids = torch.randn(9, 64, device="cuda"), torch.randint(0, 9, (5,), device="cuda")
    assert torch.equal(ns.embedding_fused(ids, w, 2.0), prb.embedding(ids, w, 2.0))
