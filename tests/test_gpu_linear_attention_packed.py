"""Packed batches of linear attention whose sequences must not see one another: non-finite neighbours in grouped
backward passes (a ragged chunk is visited once for each query head)."""

import pytest
import torch

from pararnn_b200 import attn_ops as la

pytestmark = pytest.mark.gpu


def case(lens, Hq, Hkv, dk, dv, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    N = sum(lens)
    q, k, v, do = (n(1, N, h, d).to("cuda", dtype) for h, d in ((Hq, dk), (Hkv, dk), (Hkv, dv), (Hq, dv)))
    s0, ds = (n(len(lens), Hkv, dk, dv).cuda() for _ in range(2))
    cu = [0]
    for length in lens:
        cu.append(cu[-1] + length)
    return [q, k, v, do], s0, ds, -0.02 - 0.1 * torch.rand(Hkv, generator=g).cuda(), cu


# 129 to 150 tokens: a whole chunk and a ragged one; the last case is long enough to be cut into segments
@pytest.mark.parametrize("lens", [[5, 70], [129, 40], [127, 1, 150], [1430, 300]])
@pytest.mark.parametrize("share", [1, 2, 3, 5])
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128), (64, 128), (40, 96)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_sequence_behind_another_never_reaches_it(lens, share, dk, dv, dtype, bad):
    """All inputs of the last sequence are bad: the outputs, gradients and states of the earlier ones keep their
    bits.  Eight calls, since an order that is missing between warps shows in some runs only."""
    xs, s0, ds, g, cu = case(lens, share * 2, 2, dk, dv, dtype, seed=sum(lens) + share)
    offsets = torch.tensor(cu, dtype=torch.int32)
    at, S = cu[-2], len(lens) - 1

    def run(x):
        o, s = la.linear_attention_fused(*x[:3], g, s0, offsets)
        return (o, s) + la.linear_attention_reverse_vjp(*x[:3], g, x[3], s0, ds, offsets, want_state=True)

    want = run(xs)
    dirty = [x.clone() for x in xs]
    for x in dirty:
        x[0, at:] = bad
    for _ in range(8):
        got = run(dirty)
        for name, a, b in zip(("o", "state", "dq", "dk", "dv", "dstate"), got, want):
            a, b = (a[:S], b[:S]) if name.endswith("state") else (a[0, :at], b[0, :at])
            assert torch.isfinite(b).all() and torch.equal(a, b), name
