"""Group norm over many samples: several pieces, CTAs that walk several samples, groups that lie across channel blocks."""

import pytest
import torch

import pararnn_b200 as prb
from token_util import norm_oracle, unit

pytestmark = pytest.mark.gpu

# N, positions, C, groups
SHAPES = [(70000, 2, 24, 3),     # more samples than one launch takes: the pieces add to the same rows
          (3000, 1, 2048, 1),    # a row wider than the one-pass kernels take
          (900, 1, 99, 3),       # odd groups beyond 32 channels
          (700, 5, 2600, 26),    # 100 channels a group across blocks of 512 and 1024
          (9000, 3, 512, 256),   # many small groups
          (40, 300, 1200, 8)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_outputs_and_gradients_over_many_samples(shape, dtype):
    """xhat in fp32 is exact to 2^-15 of 1 + |xhat| + |mean| rstd (sums of at most 2^14 terms, added per thread and
    joined pairwise; slope at most 1.1): |error| <= u |y| + 2^-15 (1 + |xhat w| + |b| + |mean| rstd); dx likewise with
    rstd max |w dy|; dw and db add N x positions terms with that error each, their own additions in chains of at most
    N positions / 2^8 + 2^8 terms of 2^-24: all below 2^-13 of the sum of the terms' sizes."""
    N, P, C, G = shape
    gen = torch.Generator().manual_seed(C)
    x = (torch.randn(N, P, C, generator=gen) * 1.5 + torch.randn(C, generator=gen)).to(dtype)
    w = (1 + 0.3 * torch.randn(C, generator=gen)).to(dtype)
    b = (0.3 * torch.randn(C, generator=gen)).to(dtype)
    dy = torch.randn(N, P, C, generator=gen).to(dtype)
    dev = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    got = prb.group_norm(dev[0], G, dev[1], dev[2], activation="silu")
    grads = torch.autograd.grad(got, dev, dy.cuda())
    # 64 bits, on the GPU for speed
    wide = [t.detach().double().requires_grad_(True) for t in dev]
    y = norm_oracle(wide[0], G, wide[1], wide[2], 1e-5, "silu")
    want = torch.autograd.grad(y, wide, dy.cuda().double())
    x, w, b, dy = wide[0].detach(), wide[1].detach(), wide[2].detach(), dy.cuda().double()
    z = x.view(N, P, G, -1)
    mean, rstd = z.mean((1, 3), keepdim=True), (z.var((1, 3), keepdim=True, correction=0) + 1e-5).rsqrt()
    xhat = ((z - mean) * rstd).view_as(x)
    lift = (mean.abs() * rstd).expand_as(z).reshape(x.shape)
    u = unit(dtype)

    def near(a, e, tol, what):
        over = float(((a.detach().double() - e.detach()).abs() - tol).max())
        assert over <= 0, f"{what}: over its bound by {over}"

    near(got, y, u * y.detach().abs() + 2 ** -15 * (1 + (xhat * w).abs() + b.abs() + lift), "y")
    size = 2 ** -13 * rstd.expand_as(z).reshape(x.shape) * (w * dy).abs().max() * (1 + xhat.abs()) * (1 + lift.max())
    near(grads[0], want[0], u * want[0].abs() + size, "dx")
    terms = (dy.abs() * (1 + xhat.abs()) * (1 + lift)).sum((0, 1))
    near(grads[1], want[1], u * want[1].abs() + 2 ** -13 * terms, "dw")
    near(grads[2], want[2], u * want[2].abs() + 2 ** -13 * terms, "db")
    again = torch.autograd.grad(prb.group_norm(dev[0], G, dev[1], dev[2], activation="silu"), dev, dy.to(dtype))
    assert all(torch.equal(a, c) for a, c in zip(grads, again))


def test_samples_keep_their_bits_whatever_stands_beside_them():
    """A sample's output and gradient do not depend on how many samples share a CTA or a piece."""
    x = torch.randn(66000, 2, 16, device="cuda")
    dy = torch.randn_like(x)

    def run(lo, hi):
        leaf = x[lo:hi].clone().requires_grad_(True)
        y = prb.group_norm(leaf, 2, activation="gelu")
        return y.detach(), torch.autograd.grad(y, [leaf], dy[lo:hi])[0]

    whole = run(0, 66000)
    for lo, hi in ((0, 1), (65530, 65540), (65999, 66000), (100, 900)):
        for a, b in zip(run(lo, hi), whole):
            assert torch.equal(a, b[lo:hi])


def test_a_row_of_twelve_million_channels():
    x = torch.randn(1, 12_000_000, device="cuda", requires_grad=True)
    y = prb.group_norm(x, 2_400_000)
    dy = torch.randn_like(y)
    (gx,) = torch.autograd.grad(y, [x], dy)
    wide = x.detach().double().requires_grad_(True)
    want = norm_oracle(wide, 2_400_000, None, None, 1e-5, None)
    (wx,) = torch.autograd.grad(want, [wide], dy.double())
    z = wide.detach().view(-1, 5)
    rstd = (z.var(1, correction=0) + 1e-5).rsqrt()
    # five terms a group, all in fp32: 2^-19 of 1 + |xhat| + |mean| rstd <= 4 + |mean| rstd; dx the same times rstd |dy|
    lift = ((4 + z.mean(1).abs() * rstd) * 2 ** -19)[:, None]
    assert bool(((y.detach().double() - want.detach()).view(-1, 5).abs() <= lift).all())
    size = lift * (rstd * dy.double().view(-1, 5).abs().amax(1))[:, None] * 8
    assert bool(((gx.double() - wx).view(-1, 5).abs() <= size).all())
