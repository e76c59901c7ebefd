"""Cases of the token-model operators: linear attention with a decay for each head (whole prompts,
training, single tokens), group norm with an activation over channel-last tensors, and the embedding
lookup with its gradient.

``run`` computes a case in its plain form, or, where ``own`` is true, through the calls that a user of
``pararnn_b200`` makes.  Sizes: 8 heads of 64 and of 128 channels, 12 heads of 64 (d = 768), d = 1024,
sequences up to 32768 and a vocabulary of 50304 are those of the recurrent workloads; the others are
generic odd sizes.
"""

import math
import os
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
_CHUNK = 64


# ------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # a serving engine takes in a handful of new requests: short ragged prompts, packed
        dict(name="prefill_packed_short", op="prefill", dtype="bf16", batch=1, tokens=739, seqs=5, hq=12, hkv=12,
             dk=64, dv=64, state=False),
        # one long document, the state carried in from the part before it
        dict(name="prefill_long", op="prefill", dtype="bf16", batch=1, tokens=32768, seqs=0, hq=8, hkv=8, dk=128,
             dv=128, state=True),
        # full-precision evaluation with grouped heads at an odd length
        dict(name="prefill_fp32_grouped", op="prefill", dtype="fp32", batch=2, tokens=1021, seqs=0, hq=8, hkv=2,
             dk=64, dv=96, state=True),
        # training step of a mixer layer, 8 heads of 64
        dict(name="train_8x64", op="train", dtype="bf16", batch=16, tokens=4096, seqs=0, hq=8, hkv=8, dk=64, dv=64,
             state=False),
        # training step of a wider layer on longer sequences
        dict(name="train_8x128", op="train", dtype="bf16", batch=4, tokens=8192, seqs=0, hq=8, hkv=8, dk=128,
             dv=128, state=False),
        # packed training batch with grouped heads and learned initial states
        dict(name="train_packed_grouped", op="train", dtype="bf16", batch=1, tokens=5003, seqs=6, hq=12, hkv=4,
             dk=64, dv=128, state=True),
        # one user's next token: latency
        dict(name="step_single", op="step", dtype="bf16", batch=1, slots=4, hq=8, hkv=8, dk=128, dv=128),
        # a full serving batch on a pool of states
        dict(name="step_pool", op="step", dtype="bf16", batch=192, slots=256, hq=8, hkv=8, dk=128, dv=128),
        # the norm over each head's channels behind the mixer, with its activation, in training
        dict(name="norm_heads", op="norm", dtype="bf16", batch=32768, length=1, channels=1024, groups=8,
             act="silu"),
        # channel-last feature maps in front of a world model: statistics over positions
        dict(name="norm_maps", op="norm", dtype="bf16", batch=16, length=4096, channels=256, groups=32, act="silu"),
        # token embeddings of the 12-layer stack, natural-text token frequencies
        dict(name="embed_vocab", op="embed", dtype="bf16", tokens=32768, vocab=50304, channels=768, zipf=True),
        # a small table at odd sizes in full precision
        dict(name="embed_small", op="embed", dtype="fp32", tokens=1531, vocab=997, channels=257, zipf=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prefill", "prefill", "train", "train", "step", "norm", "embed"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    if op in ("prefill", "train"):
        hkv = rng.choice([1, 2, 3, 4, 6, 8])
        hq = hkv * rng.choice([1, 1, 1, 2, 3])
        dk, dv = rng.choice([16, 32, 40, 64, 64, 96, 128, 128]), rng.choice([16, 32, 56, 64, 64, 96, 128, 128])
        budget = (1 << 24) if dtype == "bf16" else (1 << 21)
        tokens = _log_int(rng, 1, min(32768, budget // (hq * max(dk, dv))))
        packed = rng.random() < 0.4
        batch = 1 if packed else max(1, min(rng.choice([1, 2, 3, 5, 8]), budget // (tokens * hq * max(dk, dv))))
        seqs = min(tokens, rng.randint(1, 9)) if packed else 0
        return dict(op=op, dtype=dtype, batch=batch, tokens=tokens, seqs=seqs, hq=hq, hkv=hkv, dk=dk, dv=dv,
                    state=rng.random() < 0.5)
    if op == "step":
        batch = _log_int(rng, 1, 192)
        hkv = rng.choice([1, 2, 4, 8])
        return dict(op=op, dtype=dtype, batch=batch, slots=batch + rng.randint(0, 64), hq=hkv * rng.choice([1, 1, 3]),
                    hkv=hkv, dk=rng.choice([16, 40, 64, 128]), dv=rng.choice([16, 56, 64, 128]))
    if op == "norm":
        groups = rng.choice([1, 2, 4, 8, 12, 32])
        channels = groups * rng.choice([2, 8, 16, 40, 64, 128])
        rows = _log_int(rng, 1, (1 << 24) // channels)
        length = 1 if rng.random() < 0.5 else _log_int(rng, 1, rows)
        return dict(op=op, dtype=dtype, batch=max(1, rows // length), length=length, channels=channels,
                    groups=groups, act=rng.choice(["none", "silu", "gelu"]))
    vocab, channels = _log_int(rng, 2, 50304), _log_int(rng, 1, 768)
    return dict(op=op, dtype=dtype, tokens=_log_int(rng, 1, 32768), vocab=vocab, channels=channels,
                zipf=rng.random() < 0.5)


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] in ("prefill", "train"):
        n = case["batch"] * case["tokens"]
        hq, hkv, dk, dv = case["hq"], case["hkv"], case["dk"], case["dv"]
        states = 4 * (case["seqs"] or case["batch"]) * hkv * dk * dv
        qkvo = size * n * (hq * (dk + dv) + hkv * (dk + dv))
        flops = 2 * n * (hq + hkv) * dk * dv
        if case["op"] == "prefill":
            return {"bytes": qkvo + states * (2 if case["state"] else 1), "flops": flops}
        return {"bytes": 2 * qkvo + (2 * states if case["state"] else 0), "flops": 3 * flops}
    if case["op"] == "step":
        b, hq, hkv, dk, dv = case["batch"], case["hq"], case["hkv"], case["dk"], case["dv"]
        return {"bytes": 8 * b * hkv * dk * dv + size * b * (hq + hkv) * (dk + dv),
                "flops": b * (2 * hq + 3 * hkv) * dk * dv}
    if case["op"] == "norm":
        n = case["batch"] * case["length"] * case["channels"]
        return {"bytes": 4 * size * n, "flops": 30 * n}
    rows = case["tokens"] * case["channels"]
    return {"bytes": size * (3 * rows + case["vocab"] * case["channels"]), "flops": 3 * rows}


# ----------------------------------------------------------------------------------------- inputs

def _offsets(case, seed):
    """Cumulative lengths of the packed sequences: every one has a token, the cuts are random."""
    gen = torch.Generator().manual_seed(seed)
    cuts = torch.randperm(case["tokens"] - 1, generator=gen)[: case["seqs"] - 1] + 1
    return torch.cat([torch.zeros(1, dtype=torch.long), cuts.sort().values, torch.tensor([case["tokens"]])])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, to=dtype):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(to)

    st = dict(case)
    if case["op"] in ("prefill", "train", "step"):
        hq, hkv, dk, dv = case["hq"], case["hkv"], case["dk"], case["dv"]
        # decays 1 - 2^-3 (a memory of some 8 tokens) to 1 - 2^-9 over the heads
        spread = torch.linspace(3.0, 9.0, hkv, dtype=torch.float64) if hkv > 1 else torch.tensor([6.0]).double()
        st["log_decay"] = torch.log1p(-torch.exp2(-spread)).float().cuda()
        lead = (case["batch"],) if case["op"] == "step" else (case["batch"], case["tokens"])
        st["q"], st["k"], st["v"] = normal(*lead, hq, dk), normal(*lead, hkv, dk), normal(*lead, hkv, dv)
        if case["op"] == "step":
            st["pool"] = normal(case["slots"], hkv, dk, dv, to=torch.float32)
            st["block_table"] = torch.randperm(case["slots"], generator=gen, device="cuda")[: case["batch"]].int()
            return st
        st["offsets"] = None
        rows = case["batch"]
        if case["seqs"]:
            rows = case["seqs"]
            # the scheduler that packs the batch keeps the offsets on the host
            st["offsets"] = _offsets(case, seed).int()
        st["s0"] = normal(rows, hkv, dk, dv, to=torch.float32) if case["state"] else None
        if case["op"] == "train":
            st["grad"] = normal(*lead, hq, dv)
            for name in ("q", "k", "v", "s0"):
                if st[name] is not None:
                    st[name].requires_grad_(True)
        return st
    if case["op"] == "norm":
        c = case["channels"]
        st["x"] = (normal(case["batch"], case["length"], c, to=torch.float32)
                   + normal(1, 1, c, to=torch.float32)).to(dtype).requires_grad_(True)
        st["w"] = (1 + normal(c, scale=0.2, to=torch.float32)).to(dtype).requires_grad_(True)
        st["b"] = normal(c, scale=0.2).requires_grad_(True)
        st["grad"] = normal(case["batch"], case["length"], c)
        return st
    v = case["vocab"]
    if case["zipf"]:
        u = torch.rand(case["tokens"], generator=gen, device="cuda", dtype=torch.float64)
        ids = (torch.exp(u * math.log(v)) - 1).long().clamp(0, v - 1)
    else:
        ids = torch.randint(0, v, (case["tokens"],), generator=gen, device="cuda")
    st["ids"] = ids
    st["table"] = normal(v, case["channels"], scale=0.02).requires_grad_(True)
    st["grad"] = normal(case["tokens"], case["channels"])
    return st


# ------------------------------------------------------------------------------------- plain form

def _power(log_decay, n):
    """exp(n log_decay) in 64 bits with a trailing axis over n; 0 where n is negative."""
    n = n.to(log_decay.device).double()
    shape = (-1,) + (1,) * n.dim()
    return torch.where(n < 0, 0.0, torch.exp(n.clamp(min=0) * log_decay.double().view(shape)))


def _mix(a, b, c, s0, log_decay, lengths, first):
    """sum_{j<=i} w^(i-j) (a_i.b_j) c_j + w^(i+first) a_i s0 over (rows, time, heads, channels), in
    blocks of time, and the state w^(L-1+first) s0 + sum_j w^(L-j-first) b_j c_j^T behind each row's
    last position."""
    rows, time, heads, _ = a.shape
    blocks = -(-time // _CHUNK)

    def cut(x):
        x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, blocks * _CHUNK - time))
        return x.view(rows, blocks, _CHUNK, heads, -1).permute(0, 3, 1, 2, 4)

    a, b, c = cut(a), cut(b), cut(c)
    pos = torch.arange(_CHUNK)
    near = _power(log_decay, pos[:, None] - pos[None, :]).float()
    inner = torch.matmul(torch.matmul(a, b.transpose(-1, -2)) * near[None, :, None], c)
    # what each block adds to the state, as seen at its own end
    to_end = _power(log_decay, _CHUNK - pos - first).float()
    added = torch.matmul((b * to_end[None, :, None, :, None]).transpose(-1, -2), c)
    m = torch.arange(blocks)
    between = _power(log_decay, _CHUNK * (m[:, None] - m[None, :] - 1)).float()
    before = torch.matmul(between[None], added.flatten(3)).view_as(added)
    if s0 is not None:
        since = _power(log_decay, _CHUNK * m).float()
        before = before + since[None, :, :, None, None] * s0[:, :, None]
    outer = torch.matmul(a, before) * _power(log_decay, pos + first).float()[None, :, None, :, None]
    out = (inner + outer).permute(0, 2, 3, 1, 4).reshape(rows, blocks * _CHUNK, heads, -1)[:, :time]
    at = torch.arange(blocks * _CHUNK, device=a.device)
    left = lengths[:, None] - at[None, :] - first
    weight = _power(log_decay, left).permute(1, 0, 2) * (at[None, None] < lengths[:, None, None])
    weight = weight.float().view(rows, heads, blocks * _CHUNK, 1)
    last = torch.matmul((b.flatten(2, 3) * weight).transpose(-1, -2), c.flatten(2, 3))
    if s0 is not None:
        last = last + _power(log_decay, lengths - 1 + first).t().float()[:, :, None, None] * s0
    return out, last


def _spread(x, index):
    """Packed (1, tokens, ...) to one row for each sequence, zeros behind its last token."""
    return torch.where((index >= 0)[..., None, None], x[0][index.clamp(min=0)], 0.0)


def _turn(x, lengths):
    """Each row's first `lengths` positions in the opposite order."""
    at = lengths[:, None] - 1 - torch.arange(x.shape[1], device=x.device)[None]
    at = torch.where(at < 0, torch.arange(x.shape[1], device=x.device)[None], at)
    return torch.take_along_dim(x, at[..., None, None], 1)


def _plain_attention(st):
    q, k, v = st["q"].detach().float(), st["k"].detach().float(), st["v"].detach().float()
    s0 = None if st["s0"] is None else st["s0"].detach()
    grad = st["grad"].float() if st["op"] == "train" else None
    index = None
    lengths = torch.full((q.shape[0],), q.shape[1], device=q.device)
    if st["offsets"] is not None:
        cu = st["offsets"].long().to(q.device)
        lengths = cu[1:] - cu[:-1]
        at = torch.arange(int(lengths.max()), device=q.device)
        index = torch.where(at[None] < lengths[:, None], cu[:-1, None] + at[None], -1)
        q, k, v = _spread(q, index), _spread(k, index), _spread(v, index)
        grad = None if grad is None else _spread(grad, index)
    share = st["hq"] // st["hkv"]
    scale = st["dk"] ** -0.5
    g = st["log_decay"]
    g_all = g.repeat_interleave(share)
    k_all, v_all = k.repeat_interleave(share, 2), v.repeat_interleave(share, 2)
    s_all = None if s0 is None else s0.repeat_interleave(share, 1)
    dtype = st["q"].dtype

    def packed(x):
        return (x if index is None else x[index >= 0][None]).to(dtype)

    o, last = _mix(q, k_all, v_all, s_all, g_all, lengths, 1)
    o = packed(o * scale)
    if st["op"] == "prefill":
        return o, last[:, ::share].contiguous()
    dq, _ = _mix(grad, v_all, k_all, None if s_all is None else s_all.transpose(-1, -2), g_all, lengths, 1)
    back = [_turn(x, lengths) for x in (k_all, v_all, q, grad)]
    dk, _ = _mix(back[1], back[3], back[2], None, g_all, lengths, 0)
    dv, ds = _mix(back[0], back[2], back[3], None, g_all, lengths, 0)

    def shared(x):
        return scale * _turn(x, lengths).unflatten(2, (st["hkv"], share)).sum(3)

    out = (o, packed(dq * scale), packed(shared(dk)), packed(shared(dv)))
    return out if s0 is None else out + (scale * ds.unflatten(1, (st["hkv"], share)).sum(2),)


def _plain_step(st):
    rows = st["block_table"].long()
    q, k, v = st["q"].float(), st["k"].float(), st["v"].float()
    new = torch.exp(st["log_decay"])[None, :, None, None] * st["pool"][rows] + k[..., None] * v[:, :, None, :]
    st["pool"][rows] = new
    share = st["hq"] // st["hkv"]
    o = torch.matmul(q[:, :, None], new.repeat_interleave(share, 1))[:, :, 0] * st["dk"] ** -0.5
    return o.to(st["q"].dtype), st["pool"]


def _activate(u, act):
    """The activation and its derivative."""
    if act == "silu":
        s = torch.sigmoid(u)
        return u * s, s * (1 + u * (1 - s))
    if act == "gelu":
        c = 0.5 * (1 + torch.erf(u * math.sqrt(0.5)))
        return u * c, c + u * torch.exp(-0.5 * u * u) * (1 / math.sqrt(2 * math.pi))
    return u, torch.ones_like(u)


def _norm(st, to):
    """Output and gradients of the group norm, computed in the type `to`."""
    n, length, c = st["x"].shape
    x, dy = st["x"].detach().to(to), st["grad"].to(to)
    w, b = st["w"].detach().to(to), st["b"].detach().to(to)
    x = x.view(n, length, st["groups"], -1)
    mean = x.mean((1, 3), keepdim=True)
    rstd = torch.rsqrt((x - mean).square().mean((1, 3), keepdim=True) + 1e-5)
    hat = (x - mean) * rstd
    y, slope = _activate(hat.view(n, length, c) * w + b, st["act"])
    du = dy * slope
    dhat = (du * w).view_as(hat)
    dx = rstd * (dhat - dhat.mean((1, 3), keepdim=True) - hat * (dhat * hat).mean((1, 3), keepdim=True))
    return y, dx.view(n, length, c), (du * hat.view(n, length, c)).sum((0, 1)), du.sum((0, 1))


def _embed_scale(case):
    return math.sqrt(case["channels"])


def _plain_embed(st):
    scale = _embed_scale(st)
    table = st["table"].detach().float()
    out = table[st["ids"]] * scale
    grad = torch.zeros_like(table).index_add_(0, st["ids"], st["grad"].float() * scale)
    return out.to(st["table"].dtype), grad.to(st["table"].dtype)


# -------------------------------------------------------------------------------- the framework's

def _run_own(st):
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pararnn-torch_b200")
    if root not in sys.path:  # the package is not installed, it lies below the repository's root
        sys.path.insert(0, root)
    import pararnn_b200 as prb

    if st["op"] == "prefill":
        return prb.linear_attention(st["q"], st["k"], st["v"], st["log_decay"], st["s0"], st["offsets"],
                                    return_state=True)
    if st["op"] == "train":
        o = prb.linear_attention(st["q"], st["k"], st["v"], st["log_decay"], st["s0"], st["offsets"])
        leaves = [st["q"], st["k"], st["v"]] + ([] if st["s0"] is None else [st["s0"]])
        return (o.detach(), *torch.autograd.grad(o, leaves, st["grad"]))
    if st["op"] == "step":
        o = prb.linear_attention_step(st["q"], st["k"], st["v"], st["log_decay"], st["pool"],
                                      block_table=st["block_table"])
        return o, st["pool"]
    if st["op"] == "norm":
        y = prb.group_norm(st["x"], st["groups"], st["w"], st["b"],
                           activation=None if st["act"] == "none" else st["act"])
        return (y.detach(), *torch.autograd.grad(y, [st["x"], st["w"], st["b"]], st["grad"]))
    y = prb.embedding(st["ids"], st["table"], scale=_embed_scale(st))
    return (y.detach(), *torch.autograd.grad(y, [st["table"]], st["grad"]))


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        if state["op"] in ("prefill", "train"):
            return _plain_attention(state)
        if state["op"] == "step":
            return _plain_step(state)
        if state["op"] == "norm":
            return tuple(x.to(state["x"].dtype) for x in _norm(state, torch.float32))
        return _plain_embed(state)


# --------------------------------------------------------------------------- 64-bit by definition

def _exact_attention(st):
    """Sums over all earlier positions, head by head, from the definition without blocks of state."""
    scale, share = st["dk"] ** -0.5, st["hq"] // st["hkv"]
    q, k, v = (st[n].detach().double() for n in ("q", "k", "v"))
    train = st["op"] == "train"
    do = st["grad"].double() if train else None
    o = q.new_zeros(*q.shape[:3], st["dv"])
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    rows = range(st["batch"])
    spans = [(r, 0, st["tokens"]) for r in rows]
    if st["offsets"] is not None:
        cu = st["offsets"].tolist()
        spans = [(0, x, y) for x, y in zip(cu[:-1], cu[1:])]
    last = q.new_zeros(len(spans), st["hkv"], st["dk"], st["dv"])
    ds = torch.zeros_like(last)
    for n, (r, lo, hi) in enumerate(spans):
        for h in range(st["hkv"]):
            g = st["log_decay"][h].double()
            power = torch.exp(g * torch.arange(hi - lo + 1, device=q.device).double())
            kk, vv = k[r, lo:hi, h], v[r, lo:hi, h]
            s0 = None if st["s0"] is None else st["s0"][n, h].detach().double()
            last[n, h] = (kk * power[:-1].flip(0)[:, None]).t() @ vv
            if s0 is not None:
                last[n, h] += power[-1] * s0
            for hq in range(h * share, (h + 1) * share):
                for i0 in range(0, hi - lo, 2048):
                    i1 = min(hi - lo, i0 + 2048)
                    sl = slice(lo + i0, lo + i1)
                    gap = torch.arange(i0, i1, device=q.device)[:, None] - torch.arange(i1, device=q.device)[None]
                    decay = torch.where(gap >= 0, power[gap.clamp(min=0)], 0.0) * scale
                    a = (q[r, sl, hq] @ kk[:i1].t()) * decay
                    o[r, sl, hq] = a @ vv[:i1]
                    far = scale * power[i0 + 1:i1 + 1, None]
                    if s0 is not None:
                        o[r, sl, hq] += far * (q[r, sl, hq] @ s0)
                    if train:
                        da = (do[r, sl, hq] @ vv[:i1].t()) * decay
                        dq[r, sl, hq] = da @ kk[:i1]
                        dk[r, lo:lo + i1, h] += da.t() @ q[r, sl, hq]
                        dv[r, lo:lo + i1, h] += a.t() @ do[r, sl, hq]
                        if s0 is not None:
                            dq[r, sl, hq] += far * (do[r, sl, hq] @ s0.t())
                            ds[n, h] += (far * q[r, sl, hq]).t() @ do[r, sl, hq]
    if not train:
        return o, last
    return (o, dq, dk, dv) if st["s0"] is None else (o, dq, dk, dv, ds)


def _exact_norm(st):
    """The gradients through 64-bit differentiation of the definition."""
    n, length, c = st["x"].shape
    x, w, b = (st[k].detach().double().requires_grad_(True) for k in ("x", "w", "b"))
    z = x.reshape(n, length, st["groups"], -1)
    var, mean = torch.var_mean(z, (1, 3), correction=0, keepdim=True)
    u = ((z - mean) / torch.sqrt(var + 1e-5)).reshape(n, length, c) * w + b
    if st["act"] == "silu":
        u = u / (1 + torch.exp(-u))
    elif st["act"] == "gelu":
        u = u * torch.special.ndtr(u)
    return (u.detach(), *torch.autograd.grad(u, [x, w, b], st["grad"].double()))


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] in ("prefill", "train"):
        with torch.no_grad():
            return _exact_attention(st)
    if case["op"] == "norm":
        return _exact_norm(st)
    if case["op"] == "step":
        pool, o = st["pool"].double(), []
        for row, slot in enumerate(st["block_table"].tolist()):
            kv = torch.einsum("hk,hv->hkv", st["k"][row].double(), st["v"][row].double())
            pool[slot] = pool[slot] * torch.exp(st["log_decay"].double())[:, None, None] + kv
            q = st["q"][row].double().view(case["hkv"], -1, case["dk"])
            o.append(torch.einsum("hgk,hkv->hgv", q, pool[slot]).flatten(0, 1) / math.sqrt(case["dk"]))
        return torch.stack(o), pool
    scale = _embed_scale(case)
    table = st["table"].detach().double()
    out = torch.nn.functional.embedding(st["ids"], table) * scale
    one = torch.sparse_coo_tensor(torch.stack([st["ids"], torch.arange(case["tokens"], device="cuda")]),
                                  torch.full((case["tokens"],), scale, dtype=torch.float64, device="cuda"),
                                  (case["vocab"], case["tokens"]))
    return out, torch.sparse.mm(one, st["grad"].double())
