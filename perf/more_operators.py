"""Performance cases of the gated recurrence over long sequences, of the norms
around a block and of the counter-based dropout, each with its plain form.

``listed()`` names the cases, ``draw(rng)`` gives another one of the same
ranges.  With ``own`` false, ``run`` computes an operator from elementary torch
operations in 32 bits; with ``own`` true it calls the package.  ``exact`` is
the operator's definition in 64 bits.  The kinds:

* ``scan``   the gated recurrence over packed sequences, split along the time
             axis (``ssla_amd.scan.gated_scan``), or with ``grad`` forward and
             backward;
* ``step``   one token of each active row of a resident state table
             (``ssla_amd.scan.sparse_gated_step``);
* ``gated``  the norm of an attention's output by heads, times its output gate
             (``ssla_amd.norm.gated_norm``), or with ``grad`` both directions;
* ``block``  a residual stream's step from one block to the next: norm of the
             block's output, dropout, scale, sum, and the next block's norm
             (``ssla_amd.norm.residual_norm``), or with ``grad`` both directions;
* ``drop``   dropout by a counter-based generator (``ssla_amd.dropout.counter_dropout``),
             or with ``grad`` both directions.

The recurrence, per sequence and channel, a_t the gate of g_t:

    h_t = a_t h_{t-1} + u_t,   o_t = q_t h_t  (or h_t without a read-out gate)

The dropout's mask: 16 bits an element of Philox4x32-10 (Salmon et al., 2011),
eight elements a counter; an element is kept where its bits are at least
round(p 2^16).
"""
import math
import random

import numpy as np
import torch
import torch.nn.functional as F

own = False
DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # the last rows of a window through one 48-wide layer: a call that is all latency
        dict(name="scan_short", kind="scan", dtype="fp32", gdtype="fp32", gate="sigmoid", N=1, T=77, C=48, read=True,
             state=True, ragged=False, grad=False),
        # one long recording, 16-bit throughout
        dict(name="scan_long", kind="scan", dtype="bf16", gdtype="bf16", gate="sigmoid", N=1, T=65536, C=1024, read=True,
             state=True, ragged=False, grad=False),
        # a ragged serving batch, log gates kept in 32 bits
        dict(name="scan_ragged", kind="scan", dtype="bf16", gdtype="fp32", gate="log", N=21, T=16411, C=2048, read=False,
             state=True, ragged=True, grad=False),
        # training the 96-wide event layer: few channels, long ragged windows
        dict(name="scan_events_train", kind="scan", dtype="fp32", gdtype="fp32", gate="sigmoid", N=8, T=58475, C=96,
             read=True, state=False, ragged=True, grad=True),
        # training at the headline's batch: eight 4096-token sequences
        dict(name="scan_train", kind="scan", dtype="bf16", gdtype="bf16", gate="sigmoid", N=8, T=32768, C=1024, read=True,
             state=True, ragged=False, grad=True),
        # a token for each of the active rows of a resident table
        dict(name="step_rows", kind="step", dtype="bf16", gdtype="bf16", gate="sigmoid", rows=4560, n=912, C=2048,
             read=True),
        # the norm behind eight heads of 64 with its output gate, at the headline's sizes
        dict(name="gated_heads", kind="gated", dtype="bf16", T=32768, C=512, G=8, norm="rms", act="silu", grad=False),
        # the same in training, four heads of 256 (odd number of rows)
        dict(name="gated_train", kind="gated", dtype="bf16", T=16411, C=1024, G=4, norm="rms", act="silu", grad=True),
        # single tokens of 32 streams between two blocks
        dict(name="block_tokens", kind="block", dtype="bf16", rdtype="bf16", T=32, C=2048, norm="rms", post=True,
             scale=False, p=0.0, grad=False),
        # a training step between two blocks: residual stream in 32 bits, layer scale, dropout
        dict(name="block_train", kind="block", dtype="bf16", rdtype="fp32", T=32768, C=1024, norm="rms", post=True,
             scale=True, p=0.1, grad=True),
        # dropout of a small layer's events
        dict(name="drop_events", kind="drop", dtype="fp32", T=4510, C=48, p=0.25, grad=False),
        # dropout of a wide activation, both directions
        dict(name="drop_train", kind="drop", dtype="bf16", T=32768, C=2048, p=0.1, grad=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("scan", "scan", "train", "step", "gated", "block", "drop"))
    dtype = rng.choice(("bf16", "fp16", "fp32"))
    if kind in ("scan", "train"):
        C = rng.choice((12, 24, 30, 48, 96, 200, 512, 1000, 1024, 2048))
        T = min(_log(rng, 1, 65536 if kind == "scan" else 32768), (1 << (26 if kind == "scan" else 25)) // C)
        return dict(kind="scan", dtype=dtype, gdtype=rng.choice((dtype, "fp32")), gate=rng.choice(("sigmoid", "log", "value")),
                    N=min(_log(rng, 1, 64), T), T=T, C=C, read=rng.random() < 0.6, state=rng.random() < 0.6,
                    ragged=rng.random() < 0.6, grad=kind == "train")
    if kind == "step":
        rows = _log(rng, 1, 4560)
        return dict(kind=kind, dtype=dtype, gdtype=rng.choice((dtype, "fp32")), gate=rng.choice(("sigmoid", "log", "value")),
                    rows=rows, n=max(1, int(rows * rng.uniform(0.1, 1.0))), C=rng.choice((12, 30, 48, 96, 512, 1000, 2048)),
                    read=rng.random() < 0.5)
    grad = rng.random() < 0.5
    if kind == "gated":
        G, per = rng.choice((1, 2, 4, 8, 16)), rng.choice((12, 32, 50, 64, 128, 256))
        return dict(kind=kind, dtype=dtype, T=min(_log(rng, 1, 32768), (1 << 24) // (G * per)), C=G * per, G=G,
                    norm=rng.choice(("rms", "layer")), act=rng.choice(("silu", "sigmoid")), grad=grad)
    C = rng.choice((24, 48, 75, 96, 512, 1000, 1024, 2048, 4096))
    T = min(_log(rng, 1, 32768), (1 << 25) // C)
    p = rng.choice((0.1, 0.25, 0.5))
    if kind == "drop":
        return dict(kind=kind, dtype=dtype, T=T, C=C, p=p, grad=grad)
    return dict(kind=kind, dtype=dtype, rdtype=rng.choice((dtype, "fp32")), T=T, C=C, norm=rng.choice(("rms", "layer")),
                post=rng.random() < 0.5, scale=rng.random() < 0.5, p=rng.choice((0.0, p)), grad=grad)


# ------------------------------------------------------------------ inputs --
def _lengths(case, seed):
    """Rows of the sequences: equal, or ragged (an empty one now and then)."""
    N, T = case["N"], case["T"]
    if not case["ragged"]:
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
    dt, C = DTYPES[case["dtype"]], case["C"]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)

    def leaves(s, *names):
        if case.get("grad"):
            s.update({n: s[n].requires_grad_() for n in names if s[n] is not None})
        return s

    if case["kind"] in ("scan", "step"):
        T = case["T"] if case["kind"] == "scan" else case["n"]
        g = randn(T, C) + 2.0   # memories of a few to a few hundred rows
        g = {"sigmoid": g, "log": F.logsigmoid(g), "value": torch.sigmoid(g)}[case["gate"]].to(DTYPES[case["gdtype"]])
        s = dict(case, u=randn(T, C).to(dt), g=g, q=randn(T, C).to(dt) if case["read"] else None)
        if case["kind"] == "step":
            s["table"] = randn(case["rows"], C)
            s["at"] = torch.randperm(case["rows"], generator=gen, device=DEV)[:T].sort().values.int()
            return s
        lens = _lengths(case, seed)
        s["lens"] = lens
        s["cu"] = torch.tensor([0] + lens, device=DEV).cumsum(0)
        s["h0"] = randn(case["N"], C) if case["state"] else None
        if case["grad"]:
            s["do"] = randn(T, C).to(dt)
            s["dht"] = randn(case["N"], C) if case["state"] else None
        return leaves(s, "u", "g", "q", "h0")
    T = case["T"]
    s = dict(case, x=(randn(T, C) * 1.5 + 0.3 * randn(C)).to(dt))
    if case["grad"]:
        s["dy"] = randn(T, C).to(dt)
    if case["kind"] == "gated":
        s.update(z=randn(T, C).to(dt), w=1 + 0.1 * randn(C))
        return leaves(s, "x", "z", "w")
    s["seed"] = torch.randint(1 << 62, (1,), generator=gen, device=DEV)
    if case["kind"] == "drop":
        return leaves(s, "x")
    s.update(r=(2 * randn(T, C)).to(DTYPES[case["rdtype"]]), w=1 + 0.1 * randn(C),
             w2=1 + 0.1 * randn(C) if case["post"] else None, ls=0.5 + 0.1 * randn(C) if case["scale"] else None)
    if case["grad"]:
        s["ds"] = randn(T, C).to(s["r"].dtype)
    return leaves(s, "x", "r", "w", "w2", "ls")


# ------------------------------------------------------------ plain forms --
def _doubling(a, x, back=False):
    """h_t = a_t h_{t-1} + x_t (or from the end) over dim 0 by doubling spans:
    after k passes row t holds the 2^k rows up to it."""
    d, T = 1, a.shape[0]
    while d < T:
        lo, hi = (slice(d, None), slice(None, -d)) if not back else (slice(None, -d), slice(d, None))
        x, old = x.clone(), x
        x[lo] += a[lo] * old[hi]
        a, old = a.clone(), a
        a[lo] *= old[hi]
        d *= 2
    return x


def _gate(g, kind):
    return torch.sigmoid(g) if kind == "sigmoid" else torch.exp(g) if kind == "log" else g


def _plain_scan(s):
    """o, the final states and, with a gradient, those of u, g, q and h0."""
    u, g, cu, h0 = s["u"].detach().float(), s["g"].detach().float(), s["cu"], s["h0"]
    q = None if s["q"] is None else s["q"].detach().float()
    a = _gate(g, s["gate"])
    full = cu[1:] > cu[:-1]
    first, last = cu[:-1].clamp(max=s["T"] - 1), (cu[1:] - 1).clamp(min=0)
    entering = torch.zeros(s["N"], s["C"], device=DEV) if h0 is None else h0.detach()
    mine = torch.zeros_like(u).index_add_(0, first, entering * full[:, None])   # the state a first row starts from
    start = torch.zeros(s["T"], 1, device=DEV).index_add_(0, first, full[:, None].float()) > 0
    h = _doubling(a.masked_fill(start, 0), u + a * mine)
    ht = torch.where(full[:, None], h[last], entering)
    o = h if q is None else q * h
    out = [o.to(s["u"].dtype), ht]
    if not s["grad"]:
        return tuple(out)
    do = s["do"].float()
    e = do if q is None else do * q
    if s["dht"] is not None:
        e = e.index_add(0, last, s["dht"] * full[:, None])
    behind = torch.cat([torch.where(start, 0, a)[1:], torch.zeros(1, s["C"], device=DEV)])
    e = _doubling(behind, e, back=True)
    before = torch.where(start, mine, torch.cat([torch.zeros_like(h[:1]), h[:-1]]))
    dg = e * before
    dg = dg * a * torch.sigmoid(-g) if s["gate"] == "sigmoid" else dg * a if s["gate"] == "log" else dg
    out += [e.to(s["u"].dtype), dg.to(s["g"].dtype)]
    if q is not None:
        out.append((do * h).to(s["q"].dtype))
    if h0 is not None:
        out.append(torch.where(full[:, None], (a * e)[first], s["dht"]))
    return tuple(out)


def _plain_step(s):
    at = s["at"].long()
    h = _gate(s["g"].float(), s["gate"]) * s["table"][at] + s["u"].float()
    s["table"][at] = h
    return (h if s["q"] is None else h * s["q"].float()).to(s["u"].dtype), s["table"]


def _keep(shape, seed, p):
    """Which elements stay, in their order: 16 bits each of Philox4x32-10 with
    the counter index // 8."""
    n, low = shape[0] * shape[1], 0xffffffff
    i = torch.arange(-(-n // 8), device=DEV)
    c0, c1, c2, c3 = i & low, i >> 32, torch.zeros_like(i), torch.zeros_like(i)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        x, y = c0 * 0xD2511F53, c2 * 0xCD9E8D57   # (modulo 2^64)
        c0, c1, c2, c3 = ((y >> 32) & low) ^ c1 ^ k0, y & low, ((x >> 32) & low) ^ c3 ^ k1, x & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    bits = torch.stack([c0 & 0xffff, c0 >> 16, c1 & 0xffff, c1 >> 16, c2 & 0xffff, c2 >> 16, c3 & 0xffff, c3 >> 16], 1)
    return (bits.view(-1)[:n] >= round(p * 65536)).view(shape)


def _dropped(x, seed, p):
    if p == 0:
        return x
    return torch.where(_keep(x.shape, seed, p), x * (65536 / (65536 - round(p * 65536))), 0)


def _plain_norm(x, G, norm, w):
    x = x.unflatten(-1, (G, -1))
    if norm == "layer":
        x = x - x.mean(-1, keepdim=True)
    return (x * (x.square().mean(-1, keepdim=True) + 1e-5).rsqrt()).flatten(1) * w


def _plain_rows(s):
    """Outputs of the norms and the dropout, differentiable."""
    x, dt = s["x"].float(), s["x"].dtype
    if s["kind"] == "drop":
        return (_dropped(x, s["seed"], s["p"]).to(dt),)
    if s["kind"] == "gated":
        z = s["z"].float()
        return ((_plain_norm(x, s["G"], s["norm"], s["w"]) * torch.sigmoid(z) * (z if s["act"] == "silu" else 1)).to(dt),)
    y = _plain_norm(x, 1, s["norm"], s["w2"]) if s["post"] else x
    y = _dropped(y, s["seed"], s["p"])
    r = s["r"].float() + (y * s["ls"] if s["scale"] else y)
    return _plain_norm(r, 1, s["norm"], s["w"]).to(dt), r.to(s["r"].dtype)


def _own_rows(s):
    if s["kind"] == "drop":
        from ssla_amd.dropout import counter_dropout
        return (counter_dropout(s["x"], s["p"], s["seed"]),)
    from ssla_amd.norm import gated_norm, residual_norm
    if s["kind"] == "gated":
        return (gated_norm(s["x"], s["z"], s["G"], s["w"], eps=1e-5, activation=s["act"], kind=s["norm"]),)
    return residual_norm(s["x"], s["r"], s["w"], eps=1e-5, kind=s["norm"], scale=s["ls"], post_norm=s["post"],
                         post_weight=s["w2"], p=s["p"], seed=s["seed"])


def _leaves(s):
    return [s[n] for n in {"drop": ("x",), "gated": ("x", "z", "w"), "block": ("x", "r", "w", "w2", "ls"),
                           "scan": ("u", "g", "q", "h0")}[s["kind"]] if s[n] is not None]


def run(s):
    if s["kind"] == "step":
        if not own:
            return _plain_step(s)
        from ssla_amd.scan import sparse_gated_step
        return sparse_gated_step(s["at"], s["u"], s["g"], s["table"], q=s["q"], gate=s["gate"]), s["table"]
    if s["kind"] == "scan":
        if not own:
            return _plain_scan(s)
        from ssla_amd.scan import gated_scan
        o, ht = gated_scan(s["u"], s["g"], s["cu"], q=s["q"], gate=s["gate"], initial_state=s["h0"], output_final_state=True)
        if not s["grad"]:
            return o, ht
        got, given = ((o, ht), (s["do"], s["dht"])) if s["dht"] is not None else ((o,), (s["do"],))
        return o.detach(), ht.detach(), *torch.autograd.grad(got, _leaves(s), given)
    out = _own_rows(s) if own else _plain_rows(s)
    if not s["grad"]:
        return out
    given = (s["dy"], s["ds"]) if s["kind"] == "block" else (s["dy"],)
    return *(t.detach() for t in out), *torch.autograd.grad(out, _leaves(s), given)


# -------------------------------------------------------- 64-bit definition --
def _exact_scan(s):
    """Row by row, the sequences side by side; behind a sequence's end its state
    stands still."""
    lens, N, C = s["lens"], s["N"], s["C"]
    most = max(max(lens), 1)
    inside = torch.arange(most, device=DEV)[:, None] < torch.tensor(lens, device=DEV)
    rows = (s["cu"][:-1] + torch.arange(most, device=DEV)[:, None])[inside]

    def side(x, fill):
        out = torch.full((most, N, C), fill, dtype=torch.float64, device=DEV)
        out[inside] = x.detach().double()[rows]
        return out

    g = s["g"].detach().double()
    a = 1 / (1 + torch.exp(-g)) if s["gate"] == "sigmoid" else torch.exp(g) if s["gate"] == "log" else g
    slope = a * (1 - a) if s["gate"] == "sigmoid" else a if s["gate"] == "log" else torch.ones_like(g)
    A, U = side(a, 1.0), side(s["u"], 0.0)
    h = torch.zeros(N, C, dtype=torch.float64, device=DEV) if s["h0"] is None else s["h0"].detach().double()
    before = torch.empty_like(U) if s["grad"] else None
    H = torch.empty_like(U)
    for t in range(most):
        if s["grad"]:
            before[t] = h
        h = torch.addcmul(U[t], A[t], h, out=H[t])
    back = torch.empty(s["T"], dtype=torch.int64, device=DEV)
    back[rows] = torch.arange(rows.numel(), device=DEV)

    def packed(x):
        return x[inside][back]

    q = None if s["q"] is None else s["q"].detach().double()
    o, ht = packed(H), h.clone()
    if not s["grad"]:
        return o if q is None else q * o, ht
    do = s["do"].double()
    E = side(do if q is None else do * q, 0.0)
    c = torch.zeros_like(ht) if s["dht"] is None else s["dht"].double()
    for t in range(most - 1, -1, -1):
        E[t] += c
        c = A[t] * E[t]
    out = [o if q is None else q * o, ht, packed(E), packed(E * before) * slope]
    if q is not None:
        out.append(do * o)
    if s["h0"] is not None:
        out.append(c)
    return tuple(out)


def _exact_keep(shape, seed, p):
    """The mask from the published rounds, in unsigned 64-bit numbers."""
    n = shape[0] * shape[1]
    low, half = np.uint64(0xffffffff), np.uint64(32)
    x = [np.arange((n + 7) // 8, dtype=np.uint64), None, np.zeros((n + 7) // 8, np.uint64), np.zeros((n + 7) // 8, np.uint64)]
    x[0], x[1] = x[0] & low, x[0] >> half
    key = [seed & 0xffffffff, seed >> 32]
    for _ in range(10):
        p0, p1 = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(p1 >> half) ^ x[1] ^ np.uint64(key[0]), p1 & low, (p0 >> half) ^ x[3] ^ np.uint64(key[1]), p0 & low]
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    words = np.stack(x, 1).astype("<u4").view("<u2").reshape(-1)[:n]
    return torch.from_numpy(words >= round(p * 65536)).view(shape).to(DEV)


def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] == "step":
        h, g, at = s["table"].double(), s["g"].double(), s["at"].long()
        a = 1 / (1 + torch.exp(-g)) if s["gate"] == "sigmoid" else torch.exp(g) if s["gate"] == "log" else g
        h[at] = a * h[at] + s["u"].double()
        return (h[at] if s["q"] is None else h[at] * s["q"].double()), h
    if s["kind"] == "scan":
        return _exact_scan(s)
    d = {n: t.detach().double().requires_grad_(t.requires_grad) if torch.is_tensor(t) and t.is_floating_point() else t
         for n, t in s.items()}
    x = d["x"]

    def normed(v, groups, weight):
        v = v.reshape(v.shape[0], groups, -1)
        if s["norm"] == "layer":
            var, mean = torch.var_mean(v, dim=2, correction=0, keepdim=True)
            v = (v - mean) / torch.sqrt(var + 1e-5)
        else:
            v = v / torch.sqrt((v * v).mean(2, keepdim=True) + 1e-5)
        return v.reshape(x.shape) * weight

    def dropped(v):
        if s["p"] == 0:
            return v
        keep = _exact_keep(x.shape, int(s["seed"]), s["p"])
        return torch.where(keep, v / (1 - round(s["p"] * 65536) / 65536), torch.zeros_like(v))

    if s["kind"] == "drop":
        out = (dropped(x),)
    elif s["kind"] == "gated":
        act = 1 / (1 + torch.exp(-d["z"]))
        out = (normed(x, s["G"], d["w"]) * (act * d["z"] if s["act"] == "silu" else act),)
    else:
        y = dropped(normed(x, 1, d["w2"]) if s["post"] else x)
        r = d["r"] + (y * d["ls"] if s["scale"] else y)
        out = normed(r, 1, d["w"]), r
    if not s["grad"]:
        return out
    given = (d["dy"], d["ds"]) if s["kind"] == "block" else (d["dy"],)
    return *(t.detach() for t in out), *torch.autograd.grad(out, _leaves(d), given)


# -------------------------------------------------------------------- work --
def work(case):
    size, C = SIZE[case["dtype"]], case["C"]
    if case["kind"] in ("scan", "step"):
        n = (case["T"] if case["kind"] == "scan" else case["n"]) * C
        streams = size * (3 if case["read"] else 2) + SIZE[case["gdtype"]]   # u, g, q in, o out
        flops = 7 * n
        if case["kind"] == "step":
            return {"bytes": n * (streams + 8), "flops": flops}
        states = case["N"] * C * 4
        nbytes = n * streams + states * (2 if case["state"] else 1)
        if not case["grad"]:
            return {"bytes": nbytes, "flops": flops}
        # and do in, the gradients of u, g, q out, those of the states
        return {"bytes": nbytes + n * streams + states * (2 if case["state"] else 0), "flops": flops * 3}
    n = case["T"] * C
    if case["kind"] == "drop":
        return {"bytes": n * size * (4 if case["grad"] else 2), "flops": n * (4 if case["grad"] else 2)}
    if case["kind"] == "gated":
        return {"bytes": n * size * (6 if case["grad"] else 3) + 8 * C, "flops": n * (40 if case["grad"] else 14)}
    streams = 2 * size + 2 * SIZE[case["rdtype"]]   # x, r in, y and the sum out
    return {"bytes": n * streams * (2 if case["grad"] else 1) + 12 * C, "flops": n * (50 if case["grad"] else 18)}
