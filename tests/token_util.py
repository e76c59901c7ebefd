"""64-bit oracles of the token-model operators (linear attention with a decay for each head, group norm
with an activation, embedding), on the CPU, from the definitions: token by token, no chunks."""

import torch


def attention_oracle(q, k, v, log_decay, state=None, scale=None, cu=None):
    """(o, final states) in float64, differentiable; S_t = w S_{t-1} + k_t v_t^T, o_t = scale q_t S_t."""
    B, T, Hq, dk = q.shape
    Hkv, dv = k.shape[2], v.shape[3]
    share = Hq // Hkv
    scale = dk ** -0.5 if scale is None else scale
    w = torch.exp(log_decay.double())[:, None, None]
    spans = [(b, 0, T) for b in range(B)] if cu is None else [(0, a, b) for a, b in zip(cu[:-1], cu[1:])]
    rows = [[None] * T for _ in range(B)]
    last = []
    for n, (b, lo, hi) in enumerate(spans):
        s = q.new_zeros(Hkv, dk, dv) if state is None else state[n]
        for t in range(lo, hi):
            s = w * s + k[b, t][:, :, None] * v[b, t][:, None, :]
            rows[b][t] = scale * torch.einsum("hgk,hkv->hgv", q[b, t].view(Hkv, share, dk), s).reshape(Hq, dv)
        last.append(s)
    zero = q.new_zeros(Hq, dv)
    o = torch.stack([torch.stack([zero if x is None else x for x in r]) for r in rows])
    return o, torch.stack(last)


def attention_grads(q, k, v, log_decay, grad, state=None, grad_state=None, scale=None, cu=None):
    """float64 gradients (q, k, v, state or None) by differentiating the recurrence."""
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    s = None if state is None else state.clone().requires_grad_(True)
    o, last = attention_oracle(*leaves, log_decay, s, scale, cu)
    total = (o * grad).sum()
    if grad_state is not None:
        total = total + (last * grad_state).sum()
    got = torch.autograd.grad(total, leaves + ([] if s is None else [s]))
    return (*got, None) if s is None else got


def norm_oracle(x, groups, w, b, eps, act):
    N, C = x.shape[0], x.shape[-1]
    z = x.reshape(N, -1, groups, C // groups)
    mean = z.mean((1, 3), keepdim=True)
    var = ((z - mean) ** 2).mean((1, 3), keepdim=True)
    u = ((z - mean) / torch.sqrt(var + eps)).reshape(x.shape)
    u = u * (1 if w is None else w) + (0 if b is None else b)
    if act == "silu":
        return u * torch.sigmoid(u)
    if act == "gelu":
        return u * torch.special.ndtr(u)
    return u


def unit(dtype):
    """Half a step of the type: the largest relative error of one rounding."""
    return torch.finfo(dtype).eps / 2
