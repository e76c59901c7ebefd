"""The token-model operators inside a compiled function: the compiler breaks its graph at them and the results are those
of the plain call."""

import warnings

import pytest
import torch

import pararnn_b200 as prb

pytestmark = pytest.mark.gpu


def compiled(f, *args):
    torch._dynamo.reset()
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")  # the compiler tells of each break once
        return torch.compile(f, backend="aot_eager")(*args)


def test_compiled_mixer_with_embedding_and_gradients():
    torch.manual_seed(0)
    emb, mixer = prb.TokenEmbedding(20, 64).cuda(), prb.LinearAttention(64, 4, n_kv_heads=2).cuda()
    ids = torch.randint(0, 20, (2, 70), device="cuda")
    leaves = [emb.weight, mixer.W_qkv.weight, mixer.norm_weight, mixer.norm_bias]

    def model(i):
        return mixer(torch.tanh(emb(i))).sin()

    want, got = model(ids), compiled(model, ids)
    g = torch.randn_like(want)
    # the same kernels; the elementwise parts may be put together in another order of roundings
    assert float((got - want).abs().max()) <= 2 ** -18 * float(want.abs().max())
    for a, b in zip(torch.autograd.grad(got, leaves, g), torch.autograd.grad(want, leaves, g)):
        assert float((a - b).abs().max()) <= 2 ** -16 * float(b.abs().max())


def test_compiled_norm_and_step():
    x = torch.randn(6, 64, device="cuda", requires_grad=True)
    w = torch.rand(64, device="cuda")
    assert torch.equal(compiled(lambda t: prb.group_norm(t, 4, w, activation="gelu"), x),
                       prb.group_norm(x, 4, w, activation="gelu"))
    q, k, v = (torch.randn(3, 2, 32, device="cuda") for _ in range(3))
    g = torch.tensor([-0.1, -0.4], device="cuda")
    pool = torch.randn(3, 2, 32, 32, device="cuda")
    ref = pool.clone()
    with torch.no_grad():
        a = compiled(lambda s: prb.linear_attention_step(q, k, v, g, s) + 1, pool)
        b = prb.linear_attention_step(q, k, v, g, ref) + 1
    assert torch.equal(a, b) and torch.equal(pool, ref)
