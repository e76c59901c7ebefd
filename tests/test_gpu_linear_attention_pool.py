"""The single-token call on pools of states that other calls hold too."""

import pytest
import torch

import pararnn_b200 as prb

pytestmark = pytest.mark.gpu


def inputs(rows=3, heads=2, d=32):
    torch.manual_seed(0)
    q, k, v = (torch.randn(rows, 4, heads, d, device="cuda") for _ in range(3))
    return q, k, v, torch.tensor([-0.1, -0.4], device="cuda"), torch.randn(rows, heads, d, d, device="cuda")


@pytest.mark.parametrize("through_view", [False, True])
def test_a_step_invalidates_what_a_backward_pass_saved(through_view):
    q, k, v, g, pool = inputs()
    q.requires_grad_(True)
    o = prb.linear_attention(q, k, v, g, pool)
    with torch.no_grad():
        target = pool[:] if through_view else pool
        prb.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, target)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()
    # without a step in between the pass is fine
    o = prb.linear_attention(q, k, v, g, pool)
    o.sum().backward()
    assert torch.isfinite(q.grad).all()


def test_a_step_counts_as_a_write_of_state_and_output():
    q, k, v, g, pool = inputs()
    out = torch.empty(3, 2, 32, device="cuda")
    before = pool._version, out._version
    prb.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, pool, out=out)
    assert pool._version > before[0] and out._version > before[1]
    with torch.inference_mode():
        states = torch.zeros_like(pool)
        prb.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, states)
    # an inference tensor has no version: outside the mode the step serves it as before
    prb.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, states)
    assert states.any()
