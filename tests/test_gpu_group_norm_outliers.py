"""Group norm over positions of which a few lie far from the rest, the first ones among them."""

import pytest
import torch

import pararnn_b200 as prb
from token_util import norm_oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("C", [64, 66, 33, 1024])  # vectors of four, two and one channel, several groups a CTA
@pytest.mark.parametrize("size", [10.0, 1e3, 1e5])
@pytest.mark.parametrize("where", [[0], [0, 1, 2, 3], [2500], [0, 4095]])
def test_positions_far_from_the_rest(C, size, where):
    """fp32.  A batch of at most 8 positions x 4 channels has its squares summed about its own mean, with an error of
    (32 + 2) 2^-24 of its M2; each join of (count, mean, M2) adds at most 4 roundings of 2^-24, and there are at most
    4096 / 8 + 32 of them in a chain, of terms that are all positive: below 2^-14 of M2 at the very worst, 2^-15 of
    rstd.  mean is exact to 2^-21 of the largest |x|, which is at most |mean| + |x - mean|.  So
    |error| <= 2^-15 (|xhat| + 1) + 2^-20 (|mean| + |x - mean|) rstd <= 2^-14 (1 + |xhat| + |mean| rstd)."""
    gen = torch.Generator(device="cuda").manual_seed(C)
    x = torch.randn(3, 4096, C, generator=gen, device="cuda")
    x[:, where] += size
    check(x, 3 if C % 3 == 0 else 4)


def test_a_long_sample_with_a_first_position_far_from_the_rest():
    """A million positions: a thread has some thousand values.  Squares about the first of them would lose
    1e-3 of the variance in the rounding of their sum; the bound is the one above (110 batches a thread)."""
    x = torch.randn(1, 1 << 20, 256, generator=torch.Generator(device="cuda").manual_seed(0), device="cuda")
    x[:, 0] += 1e3
    check(x, 8)


def check(x, groups):
    y = prb.group_norm(x, groups)
    wide = x.double()
    want = norm_oracle(wide, groups, None, None, 1e-5, None)
    z = wide.view(*x.shape[:2], groups, -1)
    lift = z.mean((1, 3), keepdim=True).abs() * (z.var((1, 3), keepdim=True, correction=0) + 1e-5).rsqrt()
    tol = 2 ** -14 * (1 + want.abs() + lift.expand_as(z).reshape(x.shape))
    over = float(((y.double() - want).abs() - tol).max())
    assert over <= 0, f"over its bound by {over}"
