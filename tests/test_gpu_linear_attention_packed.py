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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N", [300, 3000])
def test_offsets_out_of_order_give_no_token_to_two_sequences(N, dtype):
    """What a replay finds in its offsets: one below an earlier one counts as that one.  40 sequences, so that the
    scan passes from one warp-load of sequences to the next; 3000 tokens are long enough for segments."""
    xs, _, _, g, _ = case([N], 2, 1, 64, 64, dtype, seed=N)
    S = 40 if N == 300 else 4
    tail = [N - 40] * (S - 3)
    wild, plain = [0, 200, 50, N - 40] + tail, [0, 200, 200, N - 40] + tail
    wilder, full = [-5, N + 9, 3, N - 40] + tail, [0] + [N] * S
    s0, ds = torch.randn(S, 1, 64, 64).cuda(), torch.randn(S, 1, 64, 64).cuda()
    cu = torch.tensor(plain, dtype=torch.int32, device="cuda")

    def run():
        o, s = la.linear_attention_fused(*xs[:3], g, s0, cu)
        return (o, s) + la.linear_attention_reverse_vjp(*xs[:3], g, xs[3], s0, ds, cu, want_state=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = run()

    def replay(offsets):
        cu.copy_(torch.tensor(offsets, dtype=torch.int32))
        graph.replay()
        return [x.clone() for x in outs]

    for a, b in ((wild, plain), (wilder, full)):
        for x, y in zip(replay(a), replay(b)):
            assert torch.equal(x, y)
    got = replay(wild)
    assert not got[0][:, N - 40:].any() and torch.equal(got[1][1], s0[1]) and torch.equal(got[1][3:], s0[3:])
    if N == 300:
        # bf16: neither call is cut into segments, the bits are the same.  fp32: the capture, which only knows that no
        # sequence is longer than 300, cuts and the call does not; each is within 2 (dk + 64 + chunks + 16) 2^-24 of the
        # sum of the terms' sizes (chunks of 64: at most 5, and one more addition for a segment), so they differ by at
        # most twice that, 2 * 2 * (64 + 64 + 6 + 16) * 2^-24 < 2^-14; the sizes' own rounding is far below the rest
        args = [x[:, :N - 40] for x in xs[:3]], s0[[0, 2]], torch.tensor([0, 200, N - 40])
        want = la.linear_attention_fused(*args[0], g, *args[1:])
        size = la.linear_attention_fused(*[x.abs() for x in args[0]], g, args[1].abs(), args[2])
        for x, y, z in zip((got[0][:, :N - 40], got[1][[0, 2]]), want, size):
            if dtype == torch.bfloat16:
                assert torch.equal(x, y)
            else:
                assert bool(((x - y).abs() <= 2 ** -14 * z).all())
