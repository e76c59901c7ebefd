"""Group norm with an activation and the embedding lookup against their 64-bit definitions.

Tolerances, with u = half a step of the I/O type:

* norm, forward: mean and variance are exact to about n 2^-24 of their terms for n <= 2^13 added pairwise
  or per thread; xhat carries that relative error of (|x - mean| rstd + |mean| rstd 2^-23), the activation
  has slope <= 1.13 and its own error of 2^-21.  |error| <= u |y| + 2^-15 (1 + |xhat w| + |b| + |mean| rstd).
* norm, backward: dx = rstd (w du - m1 - xhat m2), all in fp32 with the same statistics:
  |error| <= u |dx| + 2^-13 rstd max|w dy| (1 + |xhat|) (1 + max |mean| rstd); dw and db are sums of N terms of
  which each has an error of 2^-15 of its size: |error| <= u |dw| + 2^-13 sum |dy| (1 + |xhat|).
* embedding: one product and one rounding, |error| <= (u + 2^-24) |y|; the gradient adds n terms in fp32:
  |error| <= u |g| + n 2^-24 sum |dy|.
"""

import math

import pytest
import torch

import pararnn_b200 as prb
from pararnn_b200 import token_ops
from token_util import norm_oracle, unit

pytestmark = pytest.mark.gpu

SHAPES = [  # N, positions, C, groups
    (1, 1, 1, 1), (5, 1, 24, 3), (300, 1, 1024, 8), (7, 1, 1000, 8), (3, 1, 2048, 1), (64, 1, 96, 12),
    (2000, 1, 2560, 20), (2, 1, 6000, 2), (2, 1, 20, 20),
    (3, 2, 32, 4), (2, 37, 96, 12), (4, 300, 256, 32), (1, 2000, 40, 8), (2, 9, 4400, 2), (5, 64, 6, 3), (2, 50, 33, 3),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("act", [None, "silu", "gelu"])
def test_group_norm_matches_the_definition(shape, act, dtype):
    N, P, C, G = shape
    gen = torch.Generator().manual_seed(C + P)
    x = (torch.randn(N, P, C, generator=gen) * 1.5 + torch.randn(C, generator=gen)).to(dtype).double()
    w = (1 + 0.3 * torch.randn(C, generator=gen)).to(dtype).double()
    b = (0.3 * torch.randn(C, generator=gen)).to(dtype).double()
    dy = torch.randn(N, P, C, generator=gen).to(dtype).double()
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = norm_oracle(*leaves[:1], G, *leaves[1:], 1e-5, act)
    want = torch.autograd.grad(y, leaves, dy)
    y = y.detach()
    z = x.view(N, P, G, -1)
    mean, var = z.mean((1, 3), keepdim=True), z.var((1, 3), keepdim=True, correction=0)
    rstd = (var + 1e-5).rsqrt()
    xhat = ((z - mean) * rstd).view_as(x)
    lift = (mean.abs() * rstd).expand_as(z).reshape(x.shape)
    rs = rstd.expand_as(z).reshape(x.shape)
    dev = [t.to("cuda", dtype).requires_grad_(True) for t in (x, w, b)]
    got = prb.group_norm(dev[0], G, dev[1], dev[2], activation=act)
    u = unit(dtype)

    def near(a, e, tol, what):
        over = float(((a.detach().double().cpu() - e).abs() - tol).max())
        assert over <= 0, f"{what}: over its bound by {over}"

    near(got, y, u * y.abs() + 2 ** -15 * (1 + (xhat * w).abs() + b.abs() + lift), "y")
    grads = torch.autograd.grad(got, dev, dy.to("cuda", dtype))
    size = 2 ** -13 * rs * (w * dy).abs().max() * (1 + xhat.abs()) * (1 + float(lift.max()))
    near(grads[0], want[0], u * want[0].abs() + size, "dx")
    terms = (dy.abs() * (1 + xhat.abs()) * (1 + lift)).sum((0, 1))
    near(grads[1], want[1], u * want[1].abs() + 2 ** -13 * terms, "dw")
    near(grads[2], want[2], u * want[2].abs() + 2 ** -13 * terms, "db")
    again = torch.autograd.grad(prb.group_norm(dev[0], G, dev[1], dev[2], activation=act), dev, dy.to("cuda", dtype))
    assert all(torch.equal(a, c) for a, c in zip(grads, again))


@pytest.mark.parametrize("positions", [1, 50])
def test_group_norm_without_parameters_with_fp32_ones_and_through_views(positions):
    x = torch.randn(6, positions, 64, device="cuda").bfloat16()
    want = norm_oracle(x.double().cpu(), 4, None, None, 1e-3, None)
    got = prb.group_norm(x, 4, eps=1e-3)
    assert float((got.double().cpu() - want).abs().max()) <= float(want.abs().max()) * 2 ** -8 + 2 ** -12
    w = torch.rand(64, device="cuda") + 0.5
    a = prb.group_norm(x, 4, w, None, activation="silu")
    wide = torch.empty(6, positions, 2, 64, device="cuda", dtype=torch.bfloat16)
    wide[:, :, 0] = x
    assert torch.equal(a, prb.group_norm(wide[:, :, 0], 4, w, None, activation="silu"))
    flat = torch.empty(x.numel() + 1, device="cuda", dtype=torch.bfloat16)
    flat[1:] = x.flatten()
    assert torch.equal(a, prb.group_norm(flat[1:].view_as(x), 4, w, None, activation="silu"))
    # the layout (N, H, W, C) is the same data
    if positions == 50:
        assert torch.equal(a, prb.group_norm(x.view(6, 5, 10, 64), 4, w, activation="silu").view_as(a))


@pytest.mark.parametrize("positions", [1, 64])
def test_group_norm_with_a_mean_far_above_its_spread(positions):
    # the variance must not be formed as a difference of squares: spread 1 around 4096
    gen = torch.Generator().manual_seed(0)
    x = (4096 + torch.randn(3, positions, 256, generator=gen)).float()
    want = norm_oracle(x.double(), 2, None, None, 1e-5, None)
    got = prb.group_norm(x.cuda(), 2)
    # each x - mean has an absolute error of about the mean's rounding, 2^-12 of the spread
    assert float((got.double().cpu() - want).abs().max()) <= 2 ** -10


@pytest.mark.parametrize("positions", [1, 40])
def test_group_norm_keeps_non_finite_samples_to_themselves(positions):
    x = torch.randn(5, positions, 64, device="cuda")
    want = prb.group_norm(x, 4, activation="gelu")
    y = x.clone()
    y[2, 0, 3], y[3, 0, 17] = float("nan"), float("inf")
    got = prb.group_norm(y, 4, activation="gelu")
    same = [0, 1, 4]
    assert torch.equal(got[same], want[same])
    assert torch.equal(got[2, :, 16:], want[2, :, 16:]) and torch.isnan(got[2, :, :16]).all()
    assert torch.equal(got[3, :, :16], want[3, :, :16]) and torch.equal(got[3, :, 32:], want[3, :, 32:])
    flat = torch.full((2, positions, 64), 3.25, device="cuda")  # no spread at all: xhat = 0
    assert not prb.group_norm(flat, 4).any()


EMBED = [(1, 1, 1), (1, 5, 8), (33, 1, 24), (500, 7, 257), (2000, 3, 768), (4000, 5000, 64), (300, 60000, 40),
         (70000, 11, 16)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("ids_type", [torch.int32, torch.int64])
@pytest.mark.parametrize("shape", EMBED)
def test_embedding_and_its_gradient(shape, dtype, ids_type):
    N, V, C = shape
    gen = torch.Generator().manual_seed(N + C)
    ids = (torch.rand(N, generator=gen) ** 2 * V).long().clamp(0, V - 1)
    if N > 40:  # padding ids
        ids[3], ids[17], ids[30] = -1, V, -100
    table = torch.randn(V, C, generator=gen).to(dtype)
    dy = torch.randn(N, C, generator=gen).to(dtype)
    scale = 1.7
    live = (ids >= 0) & (ids < V)
    want = torch.where(live[:, None], table.double()[ids.clamp(0, V - 1)] * scale, 0.0)
    w = table.cuda().requires_grad_(True)
    got = prb.embedding(ids.to("cuda", ids_type), w, scale)
    u = unit(dtype)
    # scale is a float32 number to the kernel
    tol = (u + 2 ** -23) * want.abs()
    assert got.dtype == dtype and float(((got.detach().double().cpu() - want).abs() - tol).max()) <= 0
    (g,) = torch.autograd.grad(got, [w], dy.cuda())
    add = torch.zeros(V, C, dtype=torch.float64).index_add_(0, ids[live], dy.double()[live] * scale)
    size = torch.zeros(V, C, dtype=torch.float64).index_add_(0, ids[live], dy.double()[live].abs() * scale)
    count = torch.bincount(ids[live], minlength=V).double()[:, None]
    tol = u * add.abs() + (count + 2) * 2 ** -23 * size
    assert float(((g.double().cpu() - add).abs() - tol).max()) <= 0
    for _ in range(2):
        (again,) = torch.autograd.grad(prb.embedding(ids.to("cuda", ids_type), w, scale), [w], dy.cuda())
        assert torch.equal(again, g)


def test_embedding_of_one_token_repeated_and_of_none():
    w = torch.randn(10, 32, device="cuda", requires_grad=True)
    ids = torch.full((3, 5000), 4, device="cuda")
    out = prb.embedding(ids, w, 0.5)
    assert out.shape == (3, 5000, 32) and torch.equal(out[2, 7], 0.5 * w[4])
    (g,) = torch.autograd.grad(out, [w], torch.ones_like(out))
    # 15000 ones: every partial sum is a whole number, so the sum is exact
    assert torch.equal(g[4], torch.full((32,), 7500.0, device="cuda")) and not g[[0, 1, 2, 3, 5, 6, 7, 8, 9]].any()
    none = prb.embedding(torch.empty(0, 3, dtype=torch.long, device="cuda"), w)
    assert none.shape == (0, 3, 32)
    (g,) = torch.autograd.grad(none, [w], torch.empty_like(none))
    assert g.shape == w.shape and not g.any()


def test_embedding_order_of_a_long_list_spans_bitmap_windows():
    # more positions than one bitmap window holds, one id that is everywhere and rare ones between
    N, V, C = 600_001, 50, 4
    ids = torch.zeros(N, dtype=torch.int32, device="cuda")
    ids[::1000] = torch.arange(len(ids[::1000]), device="cuda", dtype=torch.int32) % V
    dy = torch.ones(N, C, device="cuda")
    got = token_ops.embedding_vjp(ids, dy, V)
    want = torch.bincount(ids.long(), minlength=V).float()[:, None].expand(V, C)
    assert torch.equal(got, want)  # whole numbers below 2^24: exact


def test_token_ops_capture_and_replay():
    ids = torch.randint(0, 100, (400,), device="cuda")
    w = torch.randn(100, 64, device="cuda")
    gw, gb = torch.ones(64, device="cuda"), torch.zeros(64, device="cuda")
    dy = torch.randn(400, 64, device="cuda")

    def run():
        x = token_ops.embedding_fused(ids, w, 2.0)
        y, st = token_ops.group_norm_fused(x, 4, gw, gb, activation="silu")
        gx, a, b = token_ops.group_norm_vjp(x, dy, st, 4, gw, gb, "silu")
        return y, a, b, token_ops.embedding_vjp(ids, gx, 100, 2.0)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for seed in range(3):
        torch.manual_seed(seed)
        ids.copy_(torch.randint(0, 100 if seed else 2, (400,), device="cuda"))
        w.copy_(torch.randn(100, 64, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, run()):
            assert torch.equal(a, b)
    assert math.isfinite(float(outs[0].sum()))
