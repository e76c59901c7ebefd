"""Group norm with any of its parameters left out, and any of its gradients requested, against 64 bits."""

import itertools

import pytest
import torch

import pararnn_b200 as prb
from token_util import norm_oracle

pytestmark = pytest.mark.gpu

GIVEN = [(False, False), (True, False), (False, True), (True, True)]


@pytest.mark.parametrize("has_w,has_b", GIVEN)
@pytest.mark.parametrize("positions", [1, 9])
@pytest.mark.parametrize("act", [None, "silu"])
def test_every_choice_of_parameters_and_gradients(has_w, has_b, positions, act):
    """fp32, 32 channels a group: a group's mean and variance are sums of at most 32 x 9 terms, so xhat is exact to
    2^-15 of its size; a gradient adds at most 6 x 9 products of size |dy| (1 + |xhat|) with that error, and the
    activation's slope is at most 1.1: all of it within 2^-12 of the largest such sum."""
    gen = torch.Generator().manual_seed(positions)
    n = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    x, dy = n(6, positions, 64), n(6, positions, 64)
    w, b = (1 + 0.3 * n(64) if has_w else None), (0.3 * n(64) if has_b else None)
    given = [t for t in (x, w, b) if t is not None]
    wide = [t.double().requires_grad_(True) for t in given]
    it = iter(wide[1:])
    want_y = norm_oracle(wide[0], 2, next(it) if has_w else None, next(it) if has_b else None, 1e-5, act)
    want = torch.autograd.grad(want_y, wide, dy.double())
    for picked in itertools.product([False, True], repeat=len(given)):
        dev = [t.cuda().requires_grad_(p) for t, p in zip(given, picked)]
        it = iter(dev[1:])
        y = prb.group_norm(dev[0], 2, next(it) if has_w else None, next(it) if has_b else None, activation=act)
        assert float((y.detach().double().cpu() - want_y.detach()).abs().max()) <= 2 ** -12 * 8
        assert y.requires_grad == any(picked)
        if not any(picked):
            continue
        y.backward(dy.cuda())
        for t, p, e in zip(dev, picked, want):
            if not p:
                assert t.grad is None
                continue
            assert t.grad.shape == e.shape
            size = max(1.0, float(dy.abs().max())) * 8 * (1 if e.dim() == 3 else 6 * positions)
            assert float((t.grad.double().cpu() - e).abs().max()) <= 2 ** -12 * size
