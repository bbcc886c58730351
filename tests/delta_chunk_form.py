"""The gated delta rule by chunks of 64 rows in 64 bits, forward and backward, with
a hook wherever the kernels round: what an operator's roundings may do to its
results is then a run with a model of them, and what a mistake would do a run with
the mistake.

``hook(name, x, terms, n)`` gets a value, the sum of the squares of the terms it is
a sum of, and how many roundings it takes, and returns the value to go on with.
A rounding is uniform in half a step of fp32 either way, 2^-24 / sqrt(3) of what is
rounded in the root mean square, and the partial sums of terms whose signs do not
know of each other have terms / 2 as their mean square, so n roundings are off by
sqrt(n terms / 6) 2^-24.  "operand" hooks (n = 0) get a value where it enters
a product."""
import torch

ROWS = 64


def exact(name, x, terms, n):
    return x


def roundings(seed):
    """Every rounding of fp32, independent of the others."""
    gen = torch.Generator().manual_seed(seed)

    def hook(name, x, terms, n):
        return x + (n * terms / 6).sqrt() * 2.0 ** -24 * torch.randn(x.shape, generator=gen, dtype=x.dtype) if n else x
    return hook


def two_parts(x):
    """x as two bf16, the third lost."""
    head = x.float().bfloat16().double()
    return head + (x - head).float().bfloat16().double()


def losing(which):
    """The mistake: one operand's third part is left out."""
    return lambda name, x, terms, n: two_parts(x) if name == which else x


def _mask(L, strict):
    return torch.ones(L, L, dtype=torch.float64).tril(-1 if strict else 0)


def _t(x):
    return x.transpose(-1, -2)


def forward(q, k, v, g, beta, scale, S, hook=exact):
    """One sequence: q, k [T, H, K] (a head for each of v's), v [T, H, V], g, beta
    [T, H], S [H, K, V].  Returns o, the final state and what the backward takes."""
    q, k, v, g, beta, S = (x.double() for x in (q, k, v, g, beta, S))
    q, k, v = (x.transpose(0, 1) for x in (q, k, v))
    g, beta = g.t(), beta.t()[..., None]
    K, o, saved = q.shape[-1], [], []
    for a in range(0, q.shape[1], ROWS):
        qc, kc, vc, b = (x[:, a:a + ROWS] for x in (q, k, v, beta))
        G = g[:, a:a + ROWS].cumsum(-1)
        L = G.shape[-1]
        E = (G[:, :, None] - G[:, None, :]).tril().exp()
        eG, end = G.exp()[..., None], (G[:, -1:] - G).exp()[..., None]
        A = hook("A", b * E * (kc @ _t(kc)), (b * E) ** 2 * (kc ** 2 @ _t(kc) ** 2), K + 6) * _mask(L, True)
        one = torch.eye(L, dtype=torch.float64) + A
        Tm = torch.linalg.solve_triangular(one, torch.eye(L, dtype=torch.float64).expand_as(one), upper=False)
        Tm = hook("Tm", Tm, (Tm ** 2 @ one ** 2 @ Tm ** 2) * _mask(L, True), L)
        So = hook("S operand", S, S, 0)
        R = hook("R", kc @ So, kc ** 2 @ So ** 2, K)
        X = hook("X", b * (vc - eG * R), (b * vc) ** 2 + (b * eG * R) ** 2, 6)
        Xo = hook("X operand", X, X, 0)
        To = hook("Tm operand", Tm, Tm, 0)
        u = hook("u", To @ Xo, To ** 2 @ Xo ** 2, L)
        uo = hook("u operand", u, u, 0)
        P = scale * E * _mask(L, False) * hook("P", qc @ _t(kc), qc ** 2 @ _t(kc) ** 2, K + 4)
        o.append(hook("o", scale * eG * (qc @ So) + P @ uo, (scale * eG) ** 2 * (qc ** 2 @ So ** 2) + P ** 2 @ uo ** 2,
                      K + L + 4))
        saved.append((a, qc, kc, vc, b, E, eG, end, Tm, P, S, u))
        through = eG[:, -1:]
        S = hook("S", through * S + _t(kc) @ (end * uo), (through * S) ** 2 + _t(kc) ** 2 @ (end * uo) ** 2, L + 6)
    return torch.cat(o, 1).transpose(0, 1), S, saved


def backward(saved, scale, do, D, hook=exact):
    """Gradients of q, k, v, g, beta and the initial state (heads not shared)."""
    do, D = do.double().transpose(0, 1), D.double()
    out = []
    for a, q, k, v, b, E, eG, end, Tm, P, S, u in reversed(saved):
        L, K, V = E.shape[-1], q.shape[-1], v.shape[-1]
        d = do[:, a:a + ROWS]
        Do, So, uo = hook("D operand", D, D, 0), hook("S operand", S, S, 0), hook("u operand", u, u, 0)
        du = hook("du", _t(P) @ d + end * (k @ Do), _t(P) ** 2 @ d ** 2 + end ** 2 * (k ** 2 @ Do ** 2), K + L + 4)
        dX = hook("dX", _t(Tm) @ du, _t(Tm) ** 2 @ du ** 2, L)
        Xo = hook("dX operand", dX, dX, 0)
        dP = scale * E * _mask(L, False) * hook("dP", d @ _t(uo), d ** 2 @ _t(uo) ** 2, V + 4)
        dN = -E * _mask(L, True) * hook("dN", Xo @ _t(uo), Xo ** 2 @ _t(uo) ** 2, V + 4)
        dS_q, dS_x, dS_u = d @ _t(So), Xo @ _t(So), uo @ _t(Do)
        q_S, q_P = scale * eG * dS_q, dP @ k
        dq = hook("dq", q_S + q_P, (scale * eG) ** 2 * (d ** 2 @ _t(So) ** 2) + dP ** 2 @ k ** 2, V + L + 4)
        nk, back = dN @ k, _t(dP) @ q + _t(b * dN) @ k
        back2 = _t(dP) ** 2 @ q ** 2 + _t(b * dN) ** 2 @ k ** 2
        dk = hook("dk", back + b * nk - b * eG * dS_x + end * dS_u,
                  back2 + b ** 2 * (dN ** 2 @ k ** 2) + (b * eG) ** 2 * (Xo ** 2 @ _t(So) ** 2)
                  + end ** 2 * (uo ** 2 @ _t(Do) ** 2), 2 * (V + L) + 8)
        dv = hook("dv", b * dX, (b * dX) ** 2, 1)

        def dot(x, y):
            return (x * y).sum(-1)
        parts = [(q, dq), (k, -(b * eG * dS_x)), (k, b * nk), (k, -back)]
        base = sum(dot(x, y) for x, y in parts)
        base2 = sum(dot(x ** 2, y ** 2) for x, y in parts)
        nxt, nxt2 = dot(k, end * dS_u), dot(k ** 2, (end * dS_u) ** 2)
        sd = eG[:, -1:] * (S * D)
        rest, rest2 = sd.sum((1, 2))[:, None], (sd ** 2).sum((1, 2))[:, None]

        def after(x):
            return x.flip(-1).cumsum(-1).flip(-1)
        # (the products' own roundings in dq, dk's pieces come with them: K + L of them a term)
        dg = hook("dg", after(base) + nxt.cumsum(-1) - nxt + rest, after(base2) + nxt2.cumsum(-1) - nxt2 + rest2,
                  2 * (K + L) + V + L)
        db = hook("dbeta", dot(dX, v) - eG[..., 0] * dot(k, dS_x) + dot(k, nk),
                  dot(dX ** 2, v ** 2) + eG[..., 0] ** 2 * dot(k ** 2, dS_x ** 2) + dot(k ** 2, nk ** 2), 2 * (K + L) + V)
        out.append((dq, dk, dv, dg, db))
        bX = b * eG * Xo
        D = hook("D", eG[:, -1:] * D + _t(q) @ (scale * eG * d) - _t(k) @ bX,
                 (eG[:, -1:] * D) ** 2 + _t(q) ** 2 @ (scale * eG * d) ** 2 + _t(k) ** 2 @ bX ** 2, 2 * L + 8)
    dq, dk, dv, dg, db = (torch.cat(x[::-1], 1).transpose(0, 1) for x in zip(*out))
    return dq, dk, dv, dg, db, D
