"""Bounded waits of the linear attention sweeps that run out: every role of the CTA leaves, the launch ends, the status
word says so, and the next calls are right.  The limit is lowered through the library's test hook to a single poll,
which no wait for a tile survives; nothing is made to hang."""

import pytest
import torch

from pararnn_b200 import _lib
from pararnn_b200 import attn_ops as la

pytestmark = pytest.mark.gpu


def problem(B, T, share, dk, dv, lens=None):
    g = torch.Generator().manual_seed(T + dk + dv)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k, v, do = (n(B, T, h, d).to("cuda", torch.bfloat16)
                   for h, d in ((2 * share, dk), (2, dk), (2, dv), (2 * share, dv)))
    cu = None if lens is None else torch.tensor([0] + lens).cumsum(0)
    rows = B if lens is None else len(lens)
    s0, ds = (n(rows, 2, dk, dv).cuda() for _ in range(2))
    return (q, k, v, torch.tensor([-0.01, -0.2], device="cuda")), do, s0, ds, cu


def run(p, want_state):
    args, do, s0, ds, cu = p
    r = la.linear_attention_fused(*args, s0, cu, want_state=want_state)
    return r + la.linear_attention_reverse_vjp(*args, do, s0, ds, cu, want_state=want_state)


@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128), (128, 64), (64, 128)])
@pytest.mark.parametrize("want_state", [False, True])
@pytest.mark.parametrize("shape", [dict(B=2, T=700, share=1), dict(B=1, T=2500, share=3),  # whole, in segments
                                   dict(B=1, T=500, share=2, lens=[130, 1, 200, 169]),
                                   dict(B=1, T=3000, share=3, lens=[2100, 900])])
def test_a_wait_that_runs_out_ends_the_launch_and_is_reported(shape, dk, dv, want_state, prb_options):
    lib = _lib.lib()
    p = problem(dk=dk, dv=dv, **shape)
    want = run(p, want_state)
    torch.cuda.synchronize()
    assert lib.prb_linear_attention_status(1) == 0
    args, do, s0, ds, cu = p
    for call in (lambda: la.linear_attention_fused(*args, s0, cu, want_state=want_state),
                 lambda: la.linear_attention_reverse_vjp(*args, do, s0, ds, cu, want_state=want_state)):
        prb_options("spin_limit", 1)
        call()
        torch.cuda.synchronize()
        prb_options("spin_limit", 0)
        assert lib.prb_linear_attention_status(0) == 1 and lib.prb_linear_attention_poll(1) == 1
        assert lib.prb_linear_attention_status(1) == 0
    for a, b in zip(run(p, want_state), want):
        assert (a is None) == (b is None) and (a is None or torch.equal(a, b))
    torch.cuda.synchronize()
    assert lib.prb_linear_attention_status(1) == 0


def test_the_status_waits_for_sweeps_on_other_streams(prb_options):
    """torch's streams are non-blocking: a read on the legacy stream alone would not see what has not run yet."""
    lib = _lib.lib()
    p = problem(2, 700, 1, 64, 64)
    run(p, False)
    torch.cuda.synchronize()
    assert lib.prb_linear_attention_status(1) == 0
    side = torch.cuda.Stream()
    prb_options("spin_limit", 1)
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)  # about 10 ms
        la.linear_attention_fused(*p[0], p[2], want_state=False)
    prb_options("spin_limit", 0)
    assert lib.prb_linear_attention_status(1) == 1
    assert side.query()


def fail_once(prb_options, p):
    prb_options("spin_limit", 1)
    la.linear_attention_fused(*p[0], p[2], want_state=False)
    torch.cuda.synchronize()
    prb_options("spin_limit", 0)


def test_the_next_call_of_any_kind_reports_it(prb_options):
    """A model of linear attention layers alone calls no other check: the next prompt, gradient or token raises, once."""
    import pararnn_b200 as prb

    p = problem(2, 700, 1, 64, 64)
    (q, k, v, g), do, s0, ds, _ = p
    pool = torch.zeros(2, 2, 64, 64, device="cuda")
    leaf = q.clone().requires_grad_(True)
    out = prb.linear_attention(leaf, k, v, g)
    for call in (lambda: prb.linear_attention(q, k, v, g), lambda: la.linear_attention_reverse_vjp(q, k, v, g, do),
                 lambda: prb.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, pool),
                 lambda: torch.autograd.grad(out, [leaf], do, retain_graph=True)):
        fail_once(prb_options, p)
        with pytest.raises(RuntimeError, match="bounded device-side wait ran out in an earlier linear attention"):
            call()
        call()


def test_replays_are_reported_by_the_check(prb_options):
    """A graph keeps the limit that it was captured with."""
    from pararnn_b200 import ops

    p = problem(2, 700, 1, 64, 64)
    run(p, False)
    ops.check_pending_backward()
    graph = torch.cuda.CUDAGraph()
    prb_options("spin_limit", 1)
    with torch.cuda.graph(graph):
        la.linear_attention_fused(*p[0], p[2], want_state=False)
        ops.check_pending_backward()  # nothing to wait for inside a capture
    prb_options("spin_limit", 0)
    for _ in range(2):
        graph.replay()
        with pytest.raises(RuntimeError, match="linear attention"):
            ops.check_pending_backward()
    ops.check_pending_backward()
