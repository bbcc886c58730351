"""Performance cases of the gated delta rule and of the group norm with an
activation, each with its plain form.

``listed()`` names the cases, ``draw(rng)`` gives another one of the same
ranges.  With ``own`` false, ``run`` computes an operator from elementary torch
operations in 32 bits (angles of decays in 64); with ``own`` true it calls the
package.  ``exact`` is the operator's definition in 64 bits.  The kinds:

* ``chunk``  the gated delta rule over packed sequences, forward alone
             (``ssla_amd.delta.chunk_gated_delta``), or with ``grad``
             forward and backward;
* ``sites``  ragged histories of many sites at once, their states gathered from
             and written back to a resident table
             (``ssla_amd.delta.sparse_delta_scan``);
* ``step``   one token of each active site or slot
             (``ssla_amd.delta.sparse_delta_step``);
* ``norm``   group norm with an activation, channels last
             (``ssla_amd.norm.group_norm_act``), forward alone or with ``grad``
             forward and backward.

The rule, per sequence and head, state S in R^{K x V}:

    S <- exp(g_t) S;  u_t = beta_t (v_t - S^T k_t);  S <- S + k_t u_t^T
    o_t = scale S^T q_t
"""
import math
import random

import torch
import torch.nn.functional as F

own = False
DEV = "cuda"
BT = 64
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # the last rows of a stream's window: a call that is all latency
        dict(name="chunk_short", kind="chunk", dtype="bf16", N=1, T=77, Hk=2, H=2, K=64, V=64, ragged=False,
             state=True, grad=False),
        # the headline's sizes: eight 4096-token sequences, eight heads of 64, prefill
        dict(name="chunk_prefill", kind="chunk", dtype="bf16", N=8, T=32768, Hk=8, H=8, K=64, V=64, ragged=False,
             state=True, grad=False),
        # a ragged serving batch of 128-wide heads, two value heads to a key head
        dict(name="chunk_ragged_wide", kind="chunk", dtype="bf16", N=21, T=16411, Hk=2, H=4, K=128, V=128,
             ragged=True, state=False, grad=False),
        # one long recording in one call
        dict(name="chunk_long", kind="chunk", dtype="fp16", N=1, T=65536, Hk=4, H=4, K=64, V=128, ragged=False,
             state=True, grad=False),
        # a training step of the attention at the headline's sizes
        dict(name="chunk_train", kind="chunk", dtype="bf16", N=8, T=32768, Hk=8, H=8, K=64, V=64, ragged=False,
             state=True, grad=True),
        # the same in fp32 on a ragged batch with shared key heads
        dict(name="chunk_train_fp32", kind="chunk", dtype="fp32", N=12, T=8209, Hk=2, H=4, K=64, V=64, ragged=True,
             state=True, grad=True),
        # 64 bins of the 76x60 grid in one call
        dict(name="sites_64_bins", kind="sites", dtype="fp32", sites=4560, n=4510, T=58475, Hk=4, H=4, K=32, V=32),
        # the sites of a deep stage: few of them, long histories
        dict(name="sites_deep", kind="sites", dtype="bf16", sites=80, n=71, T=9001, Hk=4, H=4, K=32, V=32),
        # one online bin on the 76x60 grid
        dict(name="step_bin", kind="step", dtype="fp32", sites=4560, n=912, Hk=4, H=4, K=32, V=32),
        # a token for each of a thousand streams with wide heads
        dict(name="step_streams", kind="step", dtype="bf16", sites=1200, n=1024, Hk=4, H=8, K=128, V=128),
        # the head-wise norm of the attention's output at the headline's sizes
        dict(name="norm_heads", kind="norm", dtype="bf16", N=32768, L=1, C=512, G=8, act="silu", grad=False),
        # a training step of the norm of eight dense grids of a 76x60 stage
        dict(name="norm_grid_train", kind="norm", dtype="fp32", N=8, L=4560, C=64, G=8, act="relu", grad=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("chunk", "chunk", "train", "sites", "step", "norm"))
    H = rng.choice((1, 2, 3, 4, 8))
    Hk = rng.choice([h for h in range(1, H + 1) if H % h == 0])
    dtype = rng.choice(("bf16", "fp16", "fp32"))
    K, V = rng.choice((16, 32, 40, 64, 64, 96, 128)), rng.choice((16, 32, 56, 64, 64, 128, 128))
    if kind in ("chunk", "train"):
        most = (2 if kind == "chunk" else 1) * 32768 * 8 * 64 * 64
        T = min(_log(rng, 33, 65536), most // (H * K * V), 65536 if kind == "chunk" else 32768)
        N = min(_log(rng, 1, 32), max(1, T // 24))
        return dict(kind="chunk", dtype=dtype, N=N, T=T, Hk=Hk, H=H, K=K, V=V, ragged=rng.random() < 0.6,
                    state=rng.random() < 0.6, grad=kind == "train")
    if kind == "sites":
        K, V = min(K, 64), min(V, 64)
        sites = _log(rng, 40, 4560)
        n = max(1, int(sites * rng.uniform(0.2, 1.0)))
        return dict(kind=kind, dtype=dtype, sites=sites, n=n, T=min(n * _log(rng, 2, 120), 58475 * 4 // H), Hk=Hk, H=H,
                    K=K, V=V)
    if kind == "step":
        sites = min(_log(rng, 8, 4560), 1200 * 8 * 128 * 128 // (H * K * V))
        return dict(kind=kind, dtype=dtype, sites=sites, n=max(1, int(sites * rng.uniform(0.1, 1.0))), Hk=Hk, H=H, K=K,
                    V=V)
    G, per = rng.choice((1, 2, 4, 8)), rng.choice((4, 8, 12, 16, 32, 64))
    L = rng.choice((1, _log(rng, 2, 18240)))
    return dict(kind="norm", dtype=dtype, N=max(1, _log(rng, 1, 32768 * 512) // (G * per * L)), L=L, C=G * per, G=G,
                act=rng.choice(("none", "relu", "silu")), grad=rng.random() < 0.5)


# ------------------------------------------------------------------ inputs --
def _lengths(case, seed):
    """Rows of the sequences: equal, or ragged (an empty one now and then)."""
    N, T = case["N"] if case["kind"] == "chunk" else case["n"], case["T"]
    if case.get("ragged", True) is False:
        return [T // N + (i < T % N) for i in range(N)]
    rng = random.Random(seed * 1000003 + T)
    share = [rng.expovariate(1.0) + 0.02 for _ in range(N)]
    cut = [0]
    for i in range(N):
        cut.append(cut[-1] + share[i])
    at = [int(c / cut[-1] * T) for c in cut]
    at[-1] = T
    return [b - a for a, b in zip(at, at[1:])]


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)

    if case["kind"] == "norm":
        s = dict(case, x=(randn(case["N"], case["L"], case["C"]) * 1.5 + randn(case["C"])).to(dt),
                 w=1 + 0.1 * randn(case["C"]), b=0.1 * randn(case["C"]))
        if case["grad"]:
            s["dy"] = randn(case["N"], case["L"], case["C"]).to(dt)
            s.update({n: s[n].requires_grad_() for n in ("x", "w", "b")})
        return s
    H, Hk, K, V = case["H"], case["Hk"], case["K"], case["V"]
    T = case["n"] if case["kind"] == "step" else case["T"]
    s = dict(case, scale=K ** -0.5,
             q=F.normalize(randn(T, Hk, K), dim=-1).to(dt), k=F.normalize(randn(T, Hk, K), dim=-1).to(dt),
             v=randn(T, H, V).to(dt), g=F.logsigmoid(randn(T, H) + 1) / 4, beta=torch.sigmoid(randn(T, H)))
    if case["kind"] != "step":
        lens = _lengths(case, seed)
        s["longest"] = max(lens)
        s["cu"] = torch.tensor([0] + lens, device=DEV).cumsum(0)
    if case["kind"] == "chunk":
        s["h0"] = 0.1 * randn(case["N"], H, K, V) if case["state"] else None
        if case["grad"]:
            s["do"] = randn(T, H, V).to(dt)
            s["dht"] = 0.1 * randn(case["N"], H, K, V) if case["state"] else None
            s.update({n: s[n].requires_grad_() for n in ("q", "k", "v", "g", "beta", "h0") if s[n] is not None})
    else:
        s["state"] = 0.1 * randn(case["sites"], H, K, V)
        s["at"] = torch.randperm(case["sites"], generator=gen, device=DEV)[:case["n"]].sort().values.int()
    return s


# ------------------------------------------------------------ plain forms --
def _inverse(A):
    """(I + A)^-1 of strictly lower triangular [.., BT, BT]: the inverses of the
    diagonal blocks, doubled in width until one block is left."""
    row = torch.arange(BT, device=A.device)
    inv, w = torch.eye(BT, device=A.device, dtype=A.dtype).expand_as(A), 1
    while w < BT:
        low = (row[:, None] // w % 2 == 1) & (row[:, None] // w - 1 == row[None, :] // w)
        inv = inv - inv @ (A * low) @ inv
        w *= 2
    return inv


def _plain_chunk(q, k, v, g, beta, cu, longest, scale, h0):
    """The rule by chunks of BT rows: inside a chunk the u_t solve a unit lower
    triangular system, from chunk to chunk the state is carried."""
    T, H, V = v.shape
    N, C, K = cu.numel() - 1, max(1, -(-longest // BT)), q.shape[-1]
    at = cu[:-1, None] + torch.arange(C * BT, device=cu.device)
    inside = at < cu[1:, None]
    at = at.clamp(max=T - 1)

    def rows(x):   # [T, heads, *] -> [C, N, H, BT, *]
        x = x.repeat_interleave(H // x.shape[1], 1)[at] * inside.view(N, -1, *[1] * (x.dim() - 1))
        return x.view(N, C, BT, *x.shape[2:]).movedim(3, 2).movedim(1, 0)

    q, k, v, beta = (rows(x.float()) for x in (q, k, v, beta))
    G = rows(g.double()).cumsum(-1)
    row = torch.arange(BT, device=cu.device)
    keep = row[:, None] >= row[None, :]
    decay = (G[..., :, None] - G[..., None, :]).masked_fill(~keep, -math.inf).exp().float()
    kt = k.transpose(-1, -2).contiguous()
    inv = _inverse((k @ kt) * decay * beta[..., None] * (row[:, None] > row[None, :]))
    qk = (q @ kt) * decay
    from_start, to_end = G.exp().float()[..., None], (G[..., -1:] - G).exp().float()[..., None]
    kin, qin, kout = beta[..., None] * from_start * k, from_start * q, (to_end * k).transpose(-1, -2).contiguous()
    bv, through = beta[..., None] * v, from_start[..., -1:, :]
    S = torch.zeros(N, H, K, V, device=cu.device) if h0 is None else h0.float()
    o = []
    for c in range(C):   # the state of a chunk needs the one before it
        u = inv[c] @ (bv[c] - kin[c] @ S)
        o.append(scale * (qin[c] @ S + qk[c] @ u))
        S = through[c] * S + kout[c] @ u
    o = torch.stack(o, 1).movedim(2, 3).reshape(N * C * BT, H, V)
    t = torch.arange(T, device=cu.device)
    n = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    return o[n * (C * BT) + t - cu[n]], S


def _token(S, q, k, v, g, beta):
    """One token of each row's state; returns the state and S^T q."""
    S = g.exp()[..., None, None] * S
    u = beta[..., None] * (v - (S * k[..., None]).sum(-2))
    S = S + k[..., None] * u[..., None, :]
    return S, (S * q[..., None]).sum(-2)


def _plain_sites(s):
    """Every site's history, token by token, all sites side by side."""
    q, k, v, g, beta = (x.float().repeat_interleave(s["H"] // x.shape[1], 1) for x in
                        (s["q"], s["k"], s["v"], s["g"], s["beta"]))
    at = s["at"].long()
    if s["kind"] == "step":
        S, o = _token(s["state"][at], q, k, v, g, beta)
    else:
        cu, S, o = s["cu"], s["state"][at], torch.zeros_like(v)
        for t in range(s["longest"]):   # a token's state needs the one before it
            row = (cu[:-1] + t).clamp(max=s["T"] - 1)
            on = (cu[:-1] + t < cu[1:])[:, None]
            S1, o1 = _token(S, q[row], k[row], v[row], g[row], beta[row])
            S = torch.where(on[..., None, None], S1, S)
            o.index_add_(0, row, o1 * on[..., None])
    s["state"][at] = S
    return (s["scale"] * o).to(s["v"].dtype), s["state"]


def _plain_norm(x, w, b, G, act):
    x = x.float().view(*x.shape[:2], G, -1)
    d = x - x.mean((1, 3), keepdim=True)
    y = (d * (d.square().mean((1, 3), keepdim=True) + 1e-5).rsqrt()).flatten(2) * w + b
    return y * torch.sigmoid(y) if act == "silu" else y.clamp(min=0) if act == "relu" else y


def run(s):
    if s["kind"] in ("sites", "step"):
        if not own:
            return _plain_sites(s)
        from ssla_amd.delta import sparse_delta_scan, sparse_delta_step
        x = s["q"], s["k"], s["v"], s["g"], s["beta"]
        if s["kind"] == "step":
            return sparse_delta_step(s["at"], *x, s["state"], scale=s["scale"]), s["state"]
        return sparse_delta_scan(*x, s["cu"], s["at"], s["state"], scale=s["scale"]), s["state"]
    if s["kind"] == "norm":
        if own:
            from ssla_amd.norm import group_norm_act
            y = group_norm_act(s["x"], s["G"], s["w"], s["b"], activation=None if s["act"] == "none" else s["act"])
        else:
            y = _plain_norm(s["x"], s["w"], s["b"], s["G"], s["act"]).to(s["x"].dtype)
        if not s["grad"]:
            return y
        return y.detach(), *torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])
    x = s["q"], s["k"], s["v"], s["g"], s["beta"]
    if own:
        from ssla_amd.delta import chunk_gated_delta
        o, ht = chunk_gated_delta(*x, s["cu"], scale=s["scale"], initial_state=s["h0"], output_final_state=True)
    else:
        o, ht = _plain_chunk(*x, s["cu"], s["longest"], s["scale"], s["h0"])
        o = o.to(s["v"].dtype)
    if not s["grad"]:
        return o, ht
    if s["h0"] is None:
        return o.detach(), ht.detach(), *torch.autograd.grad(o, x, s["do"])
    return o.detach(), ht.detach(), *torch.autograd.grad((o, ht), (*x, s["h0"]), (s["do"], s["dht"]))


# -------------------------------------------------------- 64-bit definition --
def _exact_rule(q, k, v, g, beta, lens, scale, S):
    """The definition, token by token, in 64 bits: the sequences side by side,
    a sequence that has ended standing still."""
    H = v.shape[1]
    q, k = (x.repeat_interleave(H // x.shape[1], 1) for x in (q, k))
    first = [0]
    for n in lens:
        first.append(first[-1] + n)
    order = sorted(range(len(lens)), key=lambda i: -lens[i])   # the sequences that go on: the first few
    start = torch.tensor([first[i] for i in order], device=DEV)
    back = torch.tensor(sorted(range(len(lens)), key=lambda i: order[i]), device=DEV)
    S, ended, o, rows = S[order], [], [], []
    left = len(lens)
    for t in range(max(lens)):
        while lens[order[left - 1]] <= t:
            left -= 1
        if S.shape[0] > left:
            ended.insert(0, S[left:])
            S = S[:left]
        r = start[:left] + t
        S = S * torch.exp(g[r])[:, :, None, None]
        miss = v[r] - torch.matmul(k[r].unsqueeze(2), S).squeeze(2)
        S = S + k[r].unsqueeze(3) * (beta[r].unsqueeze(2) * miss).unsqueeze(2)
        o.append(torch.matmul(q[r].unsqueeze(2), S).squeeze(2) * scale)
        rows.append(r)
    S = torch.cat([S, *ended])[back]
    rows = torch.cat(rows)
    return torch.cat(o)[torch.argsort(rows)], S


def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] == "norm":
        x, w, b = (s[n].detach().double().requires_grad_(s["grad"]) for n in ("x", "w", "b"))
        z = x.reshape(s["N"], s["L"], s["G"], s["C"] // s["G"])
        var, mean = torch.var_mean(z, dim=(1, 3), correction=0, keepdim=True)
        y = ((z - mean) / torch.sqrt(var + 1e-5)).reshape(x.shape) * w + b
        y = y / (1 + torch.exp(-y)) if s["act"] == "silu" else torch.where(y > 0, y, 0) if s["act"] == "relu" else y
        return (y.detach(), *torch.autograd.grad(y, (x, w, b), s["dy"].double())) if s["grad"] else y
    lens = [1] * s["n"] if s["kind"] == "step" else (s["cu"][1:] - s["cu"][:-1]).tolist()
    if max(lens) > (8192 if case.get("grad") else 65536):
        return None
    x = [s[n].detach().double().requires_grad_(bool(case.get("grad"))) for n in ("q", "k", "v", "g", "beta")]
    if s["kind"] != "chunk":
        table, at = s["state"].double(), s["at"].long()
        o, S = _exact_rule(*x, lens, s["scale"], table[at])
        table[at] = S
        return o, table
    shape = len(lens), s["H"], s["K"], s["V"]
    h0 = torch.zeros(shape, device=DEV, dtype=torch.float64) if s["h0"] is None else s["h0"].detach().double()
    if not s["grad"]:
        return _exact_rule(*x, lens, s["scale"], h0)
    h0.requires_grad_()
    o, ht = _exact_rule(*x, lens, s["scale"], h0)
    if s["h0"] is None:
        return o.detach(), ht.detach(), *torch.autograd.grad(o, x, s["do"].double())
    return o.detach(), ht.detach(), *torch.autograd.grad((o, ht), (*x, h0), (s["do"].double(), s["dht"].double()))


# -------------------------------------------------------------------- work --
def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    if case["kind"] == "norm":
        n, C = case["N"] * case["L"] * case["C"], case["C"]
        return {"bytes": n * size * (4 if case["grad"] else 2) + C * 4 * (4 if case["grad"] else 2),
                "flops": n * (24 if case["grad"] else 9)}
    H, Hk, K, V = case["H"], case["Hk"], case["K"], case["V"]
    T = case["n"] if case["kind"] == "step" else case["T"]
    inputs, out = T * ((2 * Hk * K + H * V) * size + 2 * H * 4), T * H * V * size
    # a token: the state's decay, S^T k, the update, S^T q
    flops = T * H * K * V * 7
    if case["kind"] != "chunk":
        return {"bytes": inputs + out + 2 * case["n"] * H * K * V * 4, "flops": flops}
    states = case["N"] * H * K * V * 4
    if not case["grad"]:
        return {"bytes": inputs + out + states * (2 if case["state"] else 1), "flops": flops}
    # and their gradients: each product's two factors, the states once more
    return {"bytes": 2 * inputs + 2 * out + states * (4 if case["state"] else 1), "flops": flops * 3}
