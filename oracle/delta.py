"""The gated delta rule and the group norm with an activation in 64 bits on the
CPU: definitions in torch, differentiable, for the tests.  They share no code
with the kernels."""
from __future__ import annotations

import torch


def gated_delta(q, k, v, g, beta, lens, scale, h0=None):
    """Token by token.  q, k [T, Hk, K], v [T, H, V], g, beta [T, H], the first
    sequence at row 0; returns o [sum(lens), H, V] and the states
    [N, H, K, V]."""
    q, k, v, g, beta = (x.double() for x in (q, k, v, g, beta))
    H, V, K = v.shape[1], v.shape[2], q.shape[2]
    q, k = (x.repeat_interleave(H // x.shape[1], 1) for x in (q, k))
    o, states, t = [], [], 0
    for n, rows in enumerate(lens):
        S = torch.zeros(H, K, V, dtype=torch.float64) if h0 is None else h0[n].double()
        for t in range(t, t + rows):
            S = torch.exp(g[t])[:, None, None] * S
            u = beta[t][:, None] * (v[t] - torch.einsum("hkv,hk->hv", S, k[t]))
            S = S + torch.einsum("hk,hv->hkv", k[t], u)
            o.append(scale * torch.einsum("hkv,hk->hv", S, q[t]))
        t = sum(lens[:n + 1])
        states.append(S)
    o = torch.stack(o) if o else torch.zeros(0, H, V, dtype=torch.float64)
    return o, torch.stack(states) if states else torch.zeros(0, H, K, V, dtype=torch.float64)


def group_norm(x, num_groups, weight=None, bias=None, eps=1e-5, activation=None):
    """Channels-last group norm and activation of x [N, ..., C]."""
    x = x.double()
    z = x.reshape(x.shape[0], -1, num_groups, x.shape[-1] // num_groups)
    mean = z.mean((1, 3), keepdim=True)
    var = ((z - mean) ** 2).mean((1, 3), keepdim=True)
    y = ((z - mean) / torch.sqrt(var + eps)).reshape(x.shape)
    if weight is not None:
        y = y * weight.double()
    if bias is not None:
        y = y + bias.double()
    if activation == "relu":
        return torch.where(y > 0, y, torch.zeros_like(y))
    return y * torch.sigmoid(y) if activation == "silu" else y
