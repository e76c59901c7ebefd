"""Linear attention with a decay for each head against the 64-bit recurrence: outputs, states and
gradients over types, head layouts, lengths, packed batches, strides and non-finite neighbours.

Tolerances.  With A = the same operator on absolute values (an upper bound of every sum of absolute
terms), u = half a step of the I/O type:

* fp32: the operands are exact, the longest chain of additions has dk + 64 + (one per chunk) terms, each
  rounded to 2^-24 relative, twice that where a product is rounded first, so
  |error| <= 2 (dk + 64 + chunks + 16) 2^-24 A.
* bf16: the result is rounded once (u |o|); scores and state are rounded once to bf16 as operands of the
  tensor cores (u A); the accumulation has at most 128 + 128 terms at 2^-23 (the tensor core
  truncates).  |error| <= u |o| + u A + 2^-14 A.
* states are sums in fp32 of operands held to 2^-17 or better: |error| <= 2^-15 A for bf16 inputs, the
  fp32 bound for fp32 ones.
"""

import pytest
import torch

import pararnn_b200 as prb
from pararnn_b200 import attn_ops as la
from token_util import attention_grads, attention_oracle, unit

pytestmark = pytest.mark.gpu


def make(B, T, Hq, Hkv, dk, dv, dtype, seed, n_state=None, decay=None):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    cast = lambda x: x.to(dtype).double()  # noqa: E731
    q, k, v, do = (cast(n(B, T, H, d)) for H, d in ((Hq, dk), (Hkv, dk), (Hkv, dv), (Hq, dv)))
    if decay is None:
        decay = -torch.rand(Hkv, generator=g) * 0.5
        decay[0] = -1e-3
    decay = torch.as_tensor(decay, dtype=torch.float32).expand(Hkv).contiguous()
    rows = B if n_state is None else n_state
    return q, k, v, do, decay, n(rows, Hkv, dk, dv).double(), n(rows, Hkv, dk, dv).double()


def cuda(x, dtype):
    return None if x is None else x.to("cuda", dtype)


def bound(dtype, dk, T, magnitude, value):
    if dtype == torch.float32:
        return 2 * (dk + 64 + T / 64 + 16) * 2 ** -24 * magnitude
    return unit(dtype) * (value.abs() + magnitude) + 2 ** -14 * magnitude


def state_bound(dtype, dk, T, magnitude):
    return (2 ** -15 if dtype == torch.bfloat16 else 2 * (64 + T / 64 + 16) * 2 ** -24) * magnitude


def near(got, want, tol, what):
    got = got.double().cpu()
    assert torch.isfinite(got).all(), what
    over = ((got - want).abs() - tol).max()
    assert float(over) <= 1e-30, f"{what}: {float((got - want).abs().max())} is over its bound by {float(over)}"


CASES = [
    # B, T, Hq, Hkv, dk, dv
    (1, 1, 1, 1, 64, 64),
    (2, 63, 2, 2, 64, 64),
    (1, 129, 2, 1, 128, 128),
    (2, 128, 3, 3, 128, 64),
    (1, 300, 4, 2, 64, 128),
    (3, 65, 2, 2, 16, 56),
    (1, 257, 3, 1, 40, 96),
    (1, 70, 2, 2, 7, 13),
    (1, 1500, 1, 1, 32, 64),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("with_state", [False, True])
def test_forward_and_backward_match_the_recurrence(case, dtype, with_state):
    B, T, Hq, Hkv, dk, dv = case
    q, k, v, do, decay, s0, ds = make(*case, dtype, seed=T)
    if not with_state:
        s0 = ds = None
    o, last = attention_oracle(q, k, v, decay, s0)
    absl = lambda x: None if x is None else x.abs()  # noqa: E731
    mag_o, mag_s = attention_oracle(q.abs(), k.abs(), v.abs(), decay, absl(s0))
    got_o, got_s = la.linear_attention_fused(cuda(q, dtype), cuda(k, dtype), cuda(v, dtype), decay.cuda(),
                                             cuda(s0, torch.float32))
    near(got_o, o, bound(dtype, dk, T, mag_o, o), "o")
    near(got_s, last, state_bound(dtype, dk, T, mag_s), "state")
    want = attention_grads(q, k, v, decay, do, s0, ds)
    mags = attention_grads(q.abs(), k.abs(), v.abs(), decay, do.abs(), absl(s0), absl(ds))
    got = la.linear_attention_reverse_vjp(cuda(q, dtype), cuda(k, dtype), cuda(v, dtype), decay.cuda(),
                                          cuda(do, dtype), cuda(s0, torch.float32), cuda(ds, torch.float32),
                                          want_state=with_state)
    for name, g, w, m, d in zip(("dq", "dk", "dv"), got, want, mags, (dv, dv, dk)):
        near(g, w, bound(dtype, d * (Hq // Hkv), T, m, w), name)
    if with_state:
        near(got[3], want[3], state_bound(dtype, dv * (Hq // Hkv), T, mags[3]), "dstate")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lens", [[1], [1, 1, 1], [130, 1, 64, 127], [5, 600, 33], [2048, 3]])
def test_packed_sequences_are_independent(lens, dtype):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    N, S, Hq, Hkv, dk, dv = cu[-1], len(lens), 4, 2, 64, 64
    q, k, v, do, decay, s0, ds = make(1, N, Hq, Hkv, dk, dv, dtype, seed=N, n_state=S)
    o, last = attention_oracle(q, k, v, decay, s0, cu=cu)
    mag_o, mag_s = attention_oracle(q.abs(), k.abs(), v.abs(), decay, s0.abs(), cu=cu)
    t = torch.tensor(cu, dtype=torch.int32)
    args = [cuda(x, dtype) for x in (q, k, v)] + [decay.cuda()]
    for offsets in (t, t.cuda().long()):
        got_o, got_s = la.linear_attention_fused(*args, s0.float().cuda(), offsets)
        near(got_o, o, bound(dtype, dk, N, mag_o, o), "o")
        near(got_s, last, state_bound(dtype, dk, N, mag_s), "state")
    want = attention_grads(q, k, v, decay, do, s0, ds, cu=cu)
    mags = attention_grads(q.abs(), k.abs(), v.abs(), decay, do.abs(), s0.abs(), ds.abs(), cu=cu)
    got = la.linear_attention_reverse_vjp(*args, cuda(do, dtype), s0.float().cuda(), ds.float().cuda(), t,
                                          want_state=True)
    for name, g, w, m in zip(("dq", "dk", "dv"), got, want, mags):
        near(g, w, bound(dtype, 2 * 64, N, m, w), name)
    near(got[3], want[3], state_bound(dtype, 2 * 64, N, mags[3]), "dstate")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("decay", [0.0, -1e-4, -3.0, -200.0, float("-inf")])
def test_decays_from_none_to_no_memory(decay, dtype):
    B, T, H, d = 1, 300, 2, 64
    q, k, v, do, g, s0, _ = make(B, T, H, H, d, d, dtype, seed=3, decay=decay)
    o, last = attention_oracle(q, k, v, g, s0)
    mag_o, mag_s = attention_oracle(q.abs(), k.abs(), v.abs(), g, s0.abs())
    got_o, got_s = la.linear_attention_fused(cuda(q, dtype), cuda(k, dtype), cuda(v, dtype), g.cuda(),
                                             s0.float().cuda())
    near(got_o, o, bound(dtype, d, T, mag_o, o), "o")
    near(got_s, last, state_bound(dtype, d, T, mag_s), "state")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_rows_cut_into_segments(dtype):
    # one head and thousands of tokens: the time axis is split over CTAs; against the 64-bit recurrence
    B, T, H, d = 1, 5000, 1, 64
    q, k, v, do, g, s0, ds = make(B, T, H, H, d, d, dtype, seed=9, decay=-2e-3)
    o, last = attention_oracle(q, k, v, g, s0)
    mag_o, mag_s = attention_oracle(q.abs(), k.abs(), v.abs(), g, s0.abs())
    args = [cuda(x, dtype) for x in (q, k, v)] + [g.cuda()]
    got_o, got_s = la.linear_attention_fused(*args, s0.float().cuda())
    near(got_o, o, bound(dtype, d, T, mag_o, o), "o")
    near(got_s, last, state_bound(dtype, d, T, mag_s), "state")
    want = attention_grads(q, k, v, g, do, s0, ds)
    mags = attention_grads(q.abs(), k.abs(), v.abs(), g, do.abs(), s0.abs(), ds.abs())
    got = la.linear_attention_reverse_vjp(*args, cuda(do, dtype), s0.float().cuda(), ds.float().cuda(),
                                          want_state=True)
    for name, a, w, m in zip(("dq", "dk", "dv"), got, want, mags):
        near(a, w, bound(dtype, d, T, m, w), name)
    near(got[3], want[3], state_bound(dtype, d, T, mags[3]), "dstate")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_later_positions_never_reach_earlier_outputs(dtype, bad):
    B, T, H, d = 2, 200, 2, 64
    q, k, v, do, g, s0, _ = make(B, T, H, H, d, d, dtype, seed=11)
    clean = [cuda(x, dtype) for x in (q, k, v, do)]
    at = 150
    want = la.linear_attention_fused(*clean[:3], g.cuda())[0]
    dirty = [x.clone() for x in clean]
    for x in dirty[:3]:
        x[0, at:] = bad
    got, state = la.linear_attention_fused(*dirty[:3], g.cuda())
    # equal up to the order of the sums where the row was added again without the masked positions
    tol = 2 ** -7 if dtype == torch.bfloat16 else 2 ** -16
    assert float((got[0, :at] - want[0, :at]).abs().max()) <= tol * float(want.abs().max())
    assert torch.equal(got[1], want[1])
    assert torch.isfinite(state[1]).all() and not torch.isfinite(state[0]).any()
    # backwards: gradients of k and v look at later positions only
    wk, wv = la.linear_attention_reverse_vjp(*clean[:3], g.cuda(), clean[3])[1:3]
    dirty = [x.clone() for x in clean]
    dirty[0][0, :50] = bad
    dirty[3][0, :50] = bad
    gk, gv = la.linear_attention_reverse_vjp(dirty[0], *clean[1:3], g.cuda(), dirty[3])[1:3]
    for a, w in ((gk, wk), (gv, wv)):
        assert float((a[0, 50:] - w[0, 50:]).abs().max()) <= tol * float(w.abs().max())
        assert torch.equal(a[1], w[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_views_give_the_same_bits(dtype):
    B, T, H, d = 2, 150, 3, 64
    g = torch.full((H,), -0.1, device="cuda")
    torch.manual_seed(0)
    qkv = torch.randn(B, T, 3, H, d, device="cuda").to(dtype)
    q, k, v = qkv.unbind(2)
    want = la.linear_attention_fused(q.contiguous(), k.contiguous(), v.contiguous(), g)
    for a, b, c in ((q, k, v), tuple(x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v))):
        got = la.linear_attention_fused(a, b, c, g)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # odd offsets and broadcast heads are copied
    flat = torch.randn(B * T * H * d + 3, device="cuda").to(dtype)
    odd = flat[3:].view(B, T, H, d)
    assert torch.equal(la.linear_attention_fused(odd, k, v, g)[0], la.linear_attention_fused(odd.clone(), k, v, g)[0])
    one = k[:, :, :1].expand(B, T, H, d)
    assert torch.equal(la.linear_attention_fused(q, one, v, g)[0],
                       la.linear_attention_fused(q, one.contiguous(), v, g)[0])


def test_autograd_entry_gives_the_operator_gradients_and_refuses_a_learned_decay():
    B, T, Hq, Hkv, d = 2, 90, 4, 2, 64
    q, k, v, do, g, s0, ds = make(B, T, Hq, Hkv, d, d, torch.float32, seed=5)
    leaves = [x.float().cuda().requires_grad_(True) for x in (q, k, v, s0)]
    o, s = prb.linear_attention(*leaves[:3], g.cuda(), leaves[3], return_state=True)
    got = torch.autograd.grad([o, s], leaves, [do.float().cuda(), ds.float().cuda()])
    want = la.linear_attention_reverse_vjp(*[x.detach() for x in leaves[:3]], g.cuda(), do.float().cuda(),
                                           leaves[3].detach(), ds.float().cuda(), want_state=True)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    with pytest.raises(TypeError, match="log_decay"):
        prb.linear_attention(*leaves[:3], g.cuda().requires_grad_(True))
    # against differences of the loss, in fp32: the central difference of a linear functional of v is exact
    # up to the rounding of two forward passes
    with torch.no_grad():
        e = torch.randn_like(leaves[2])
        f = lambda x: (prb.linear_attention(leaves[0], leaves[1], x, g.cuda(), leaves[3]).double()  # noqa: E731
                       * do.cuda()).sum()
        diff = float(f(leaves[2] + e) - f(leaves[2] - e)) / 2
    (gv,) = torch.autograd.grad(prb.linear_attention(leaves[0], leaves[1], leaves[2], g.cuda(), leaves[3]),
                                [leaves[2]], do.float().cuda())
    dot = float((gv.double() * e.double()).sum())
    size = float((gv.double().abs() * e.double().abs()).sum())
    assert abs(diff - dot) <= 2 ** -14 * size


def test_capture_replay_with_new_inputs_and_offsets():
    H, d, N = 2, 64, 300
    torch.manual_seed(1)
    q, k, v, do = (torch.randn(1, N, H, d, device="cuda").bfloat16() for _ in range(4))
    g = torch.tensor([-0.01, -0.2], device="cuda")
    cu = torch.tensor([0, 100, 300], dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        la.linear_attention_fused(q, k, v, g, None, cu)
        la.linear_attention_reverse_vjp(q, k, v, g, do, None, None, cu)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, s = la.linear_attention_fused(q, k, v, g, None, cu)
        grads = la.linear_attention_reverse_vjp(q, k, v, g, do, None, None, cu)[:3]
    for offsets, fill in (([0, 100, 300], 1.0), ([0, 1, 300], 0.5), ([0, 200, 300], 2.0)):
        cu.copy_(torch.tensor(offsets, dtype=torch.int32))
        q.mul_(fill)
        graph.replay()
        torch.cuda.synchronize()
        want = la.linear_attention_fused(q, k, v, g, None, cu.clone())
        assert torch.equal(o, want[0]) and torch.equal(s, want[1])
        for a, b in zip(grads, la.linear_attention_reverse_vjp(q, k, v, g, do, None, None, cu.clone())[:3]):
            assert torch.equal(a, b)
    # offsets that leave tokens behind the last sequence, an empty sequence, or the range: clamped
    cu.copy_(torch.tensor([0, 0, 120], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    want = la.linear_attention_fused(q[:, :120], k[:, :120], v[:, :120], g)
    assert torch.equal(o[:, :120], want[0]) and not o[:, 120:].any()
    assert torch.equal(s[1], want[1][0]) and not s[0].any()
    cu.copy_(torch.tensor([0, 4000, -7], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, la.linear_attention_fused(q, k, v, g)[0])


def test_two_streams_at_once():
    torch.manual_seed(2)
    xs = [[torch.randn(2, 1000, 2, 64, device="cuda").bfloat16() for _ in range(3)] for _ in range(2)]
    g = torch.tensor([-0.01, -0.2], device="cuda")
    want = [la.linear_attention_fused(*x, g) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for st, x in zip(streams, xs):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got.append(la.linear_attention_fused(*x, g))
    torch.cuda.synchronize()
    for i, (o, s) in enumerate(got):
        assert torch.equal(o, want[i % 2][0]) and torch.equal(s, want[i % 2][1])


# --------------------------------------------------------------------------------- single tokens

def step_want(q, k, v, decay, pool, slots, scale=None):
    """Rows in order, 64 bits; padding rows give zeros."""
    pool = pool.clone()
    share = q.shape[1] // k.shape[1]
    scale = q.shape[2] ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape[0], q.shape[1], v.shape[2], dtype=torch.float64)
    for r, s in enumerate(slots):
        if 0 <= s < pool.shape[0]:
            pool[s] = pool[s] * torch.exp(decay.double())[:, None, None] + k[r][:, :, None] * v[r][:, None]
            out[r] = scale * torch.einsum("hgk,hkv->hgv", q[r].view(k.shape[1], share, -1), pool[s]).flatten(0, 1)
    return out, pool


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1), (1, 8, 8, 128, 128), (3, 4, 2, 64, 96), (5, 3, 1, 7, 13),
                                   (70, 8, 8, 128, 128), (70, 8, 8, 64, 24), (300, 2, 1, 16, 40)])
def test_step_updates_the_pool_in_place(shape, dtype):
    B, Hq, Hkv, dk, dv = shape
    C = B + 5
    q, k, v, _, decay, _, _ = make(B, 1, Hq, Hkv, dk, dv, dtype, seed=B + dk)
    pool = torch.randn(C, Hkv, dk, dv, generator=torch.Generator().manual_seed(1))
    slots = torch.randperm(C, generator=torch.Generator().manual_seed(2))[:B]
    if B > 3:  # padding rows on both sides of the pool, and one slot that three rows name
        slots[1], slots[2] = -1, C
        slots[B // 2] = slots[B - 1] = slots[0]
    o, new = step_want(q[:, 0], k[:, 0], v[:, 0], decay, pool.double(), slots.tolist())
    args = [cuda(x, dtype) for x in (q, k, v)] + [decay.cuda()]
    mags = step_want(q[:, 0].abs(), k[:, 0].abs(), v[:, 0].abs(), decay, pool.double().abs(), slots.tolist())
    for bt in (slots.int().cuda(), slots.cuda()):
        p = pool.cuda()
        got = prb.linear_attention_step(*args, p, block_table=bt)
        assert got.shape == (B, 1, Hq, dv)
        # fp32 arithmetic, dk terms; one rounding to the output's type
        near(got[:, 0], o, unit(dtype) * o.abs() + (dk + 8) * 2 ** -23 * mags[0], "o")
        near(p, new, 2 ** -21 * mags[1], "pool")
    if B <= 3:
        p = pool[slots].cuda()
        out = torch.empty(B, Hq, dv, device="cuda", dtype=dtype)
        got = prb.linear_attention_step(*[x[:, 0] for x in args[:3]], args[3], p, out=out)
        assert got is out
        near(out, o, unit(dtype) * o.abs() + (dk + 8) * 2 ** -23 * mags[0], "o")


def test_step_leaves_other_slots_and_padding_as_they_were():
    pool = torch.randn(6, 2, 64, 64, device="cuda")
    before = pool.clone()
    x = torch.randn(3, 2, 64, device="cuda")
    g = torch.tensor([-0.1, -0.2], device="cuda")
    out = prb.linear_attention_step(x, x, x, g, pool, block_table=torch.tensor([-1, 4, 1 << 40], device="cuda"))
    assert not out[0].any() and not out[2].any() and out[1].any()
    keep = [0, 1, 2, 3, 5]
    assert torch.equal(pool[keep], before[keep]) and not torch.equal(pool[4], before[4])


def test_prompt_then_steps_equal_one_long_prompt():
    """The run as a server uses it: packed prompts, states into a pool, then tokens one by one."""
    Hq, Hkv, d, lens, more = 4, 2, 64, [37, 130, 1], 5
    g = torch.tensor([-0.02, -0.3])
    torch.manual_seed(4)
    full = [[torch.randn(1, n + more, h, d).bfloat16() for h in (Hq, Hkv, Hkv)] for n in lens]
    cu = torch.tensor([0, 37, 167, 168], dtype=torch.int32)
    packed = [torch.cat([f[i][:, :n] for f, n in zip(full, lens)], 1).cuda() for i in range(3)]
    pool = torch.zeros(7, Hkv, d, d, device="cuda")
    slots = torch.tensor([5, 0, 3], device="cuda")
    o, s = prb.linear_attention(*packed, g.cuda(), None, cu, return_state=True)
    pool.index_copy_(0, slots, s)
    for t in range(more):
        q, k, v = (torch.cat([f[i][:, n + t] for f, n in zip(full, lens)]).cuda() for i in range(3))
        step = prb.linear_attention_step(q, k, v, g.cuda(), pool, block_table=slots)
        for r, n in enumerate(lens):
            x = [y.double() for y in full[r]]
            want, _ = attention_oracle(*[y[:, :n + t + 1] for y in x], g)
            mag, _ = attention_oracle(*[y[:, :n + t + 1].abs() for y in x], g)
            near(step[r], want[0, -1], bound(torch.bfloat16, d, n, mag[0, -1], want[0, -1]), f"step {t} row {r}")
    # and the pool as the initial state of another packed call
    o2, s2 = prb.linear_attention(*packed, g.cuda(), pool, cu, slots, return_state=True)
    want = prb.linear_attention(*packed, g.cuda(), pool[slots], cu, return_state=True)
    assert torch.equal(o2, want[0]) and torch.equal(s2, want[1])


def test_step_in_a_graph():
    B, H, d = 4, 2, 64
    q, k, v = (torch.randn(B, H, d, device="cuda").bfloat16() for _ in range(3))
    g = torch.tensor([-0.1, -0.2], device="cuda")
    pool, bt, out = torch.zeros(9, H, d, d, device="cuda"), torch.arange(B, device="cuda"), torch.empty_like(v)
    prb.linear_attention_step(q, k, v, g, pool, block_table=bt, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        prb.linear_attention_step(q, k, v, g, pool, block_table=bt, out=out)
    pool.zero_()
    ref = torch.zeros_like(pool)
    for slots in ([0, 1, 2, 3], [3, 2, 8, -1], [0, 0, 4, 5]):
        bt.copy_(torch.tensor(slots))
        graph.replay()
        want = prb.linear_attention_step(q, k, v, g, ref, block_table=bt.clone())
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(pool, ref)


def test_first_call_of_a_fresh_thread():
    """The tensor-core path encodes tensor maps through the driver, which needs the device's context
    in the calling thread; a new thread has none until something binds it."""
    import threading

    q, k, v = (torch.randn(1, 200, 2, 64, device="cuda").bfloat16() for _ in range(3))
    g = torch.tensor([-0.1, -0.2], device="cuda")
    want = la.linear_attention_fused(q, k, v, g)
    torch.cuda.synchronize()
    got = []
    th = threading.Thread(target=lambda: got.append(la.linear_attention_fused(q, k, v, g)))
    th.start()
    th.join()
    torch.cuda.synchronize()
    assert torch.equal(got[0][0], want[0]) and torch.equal(got[0][1], want[1])


@pytest.mark.parametrize("dk,dv", [(128, 64), (64, 128), (128, 128), (40, 96)])
@pytest.mark.parametrize("share", [1, 3])
def test_segments_of_every_tile_shape(dk, dv, share):
    """Rows long enough to be cut into segments, in every combination of 64- and 128-channel tiles: the state
    sweep, the fold and the sweep from the segments' states, forwards and backwards, against the 64-bit recurrence."""
    dtype, T = torch.bfloat16, 2300
    q, k, v, do, g, s0, ds = make(1, T, share, 1, dk, dv, dtype, seed=dk + share, decay=-3e-3)
    o, last = attention_oracle(q, k, v, g, s0)
    mag_o, mag_s = attention_oracle(q.abs(), k.abs(), v.abs(), g, s0.abs())
    args = [cuda(x, dtype) for x in (q, k, v)] + [g.cuda()]
    got_o, got_s = la.linear_attention_fused(*args, s0.float().cuda())
    near(got_o, o, bound(dtype, dk, T, mag_o, o), "o")
    near(got_s, last, state_bound(dtype, dk, T, mag_s), "state")
    want = attention_grads(q, k, v, g, do, s0, ds)
    mags = attention_grads(q.abs(), k.abs(), v.abs(), g, do.abs(), s0.abs(), ds.abs())
    got = la.linear_attention_reverse_vjp(*args, cuda(do, dtype), s0.float().cuda(), ds.float().cuda(),
                                          want_state=True)
    for name, a, w, m in zip(("dq", "dk", "dv"), got, want, mags):
        near(a, w, bound(dtype, 128 * share, T, m, w), name)
    near(got[3], want[3], state_bound(dtype, dk * share, T, mags[3]), "dstate")
    # a state's terms are held to 2^-24 (three parts of the decayed key) and added in at most 24 truncating
    # steps of 2^-23 a visit and one rounding a visit: 2^-18 of the sum of their sizes, against the 2^-17
    # that two parts alone would leave
    assert float(((got_s.double().cpu() - last).abs() / mag_s).max()) <= 2 ** -18


def test_both_kernel_families_agree_in_bf16(prb_options):
    """The tensor-core sweeps against the CUDA-core ones on the same bf16 inputs, at head sizes that both take."""
    q, k, v, do, g, s0, ds = make(2, 333, 4, 2, 64, 96, torch.bfloat16, seed=21)
    args = [cuda(x, torch.bfloat16) for x in (q, k, v)] + [g.cuda()]
    more = (cuda(do, torch.bfloat16), s0.float().cuda(), ds.float().cuda())
    a = la.linear_attention_fused(*args, s0.float().cuda()) + la.linear_attention_reverse_vjp(*args, *more, want_state=True)
    prb_options("kernel_family", "lookback")
    b = la.linear_attention_fused(*args, s0.float().cuda()) + la.linear_attention_reverse_vjp(*args, *more, want_state=True)
    o, last = attention_oracle(q, k, v, g, s0)
    mag_o, mag_s = attention_oracle(q.abs(), k.abs(), v.abs(), g, s0.abs())
    for got in (a, b):
        near(got[0], o, bound(torch.bfloat16, 64, 333, mag_o, o), "o")
        near(got[1], last, state_bound(torch.bfloat16, 64, 333, mag_s), "state")
    for x, y in zip(a, b):
        assert float((x.double() - y.double()).norm() / y.double().norm()) <= 2 ** -7


def test_step_refuses_an_output_that_other_heads_still_read():
    x = torch.randn(2, 2, 64, device="cuda")
    with pytest.raises(ValueError, match="out"):
        prb.linear_attention_step(x, x.clone(), x.clone(), torch.zeros(2, device="cuda"),
                                  torch.zeros(2, 2, 64, 64, device="cuda"), out=x)
