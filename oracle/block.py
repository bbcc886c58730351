"""The gated recurrence over packed sequences, the norms around a block and the
counter-based dropout in 64 bits on the CPU, for the tests.  They share no code
with the kernels.  The recurrence comes with how far a computation may be off
whose every step is off by a relative `eps`."""
from __future__ import annotations

import numpy as np
import torch


def _gate(g, kind):
    if kind == "value":
        return g, torch.ones_like(g)
    if kind == "log":
        return torch.exp(g), torch.exp(g)
    a = 1 / (1 + torch.exp(-g))
    return a, a / (1 + torch.exp(g))


def gated_scan(u, g, lens, q=None, gate="value", h0=None, do=None, dht=None, eps=0.0):
    """Rows 0 .. sum(lens) of u, g, q [T, C] as sequences of `lens` rows, each from
    its row of h0.  Returns a dict of (value, how far off): o and ht, and with do
    also du, dg, dq and dh0.  A state's step multiplies and adds once, each off by
    a relative eps of its terms' sizes: E_t = |a_t| E_{t-1} + eps H_t with H the
    recurrence of the absolute values."""
    u, g = u.double(), g.double()
    q = torch.ones_like(u) if q is None else q.double()
    T, C = u.shape
    N, most = len(lens), max([*lens, 1])
    a, slope = _gate(g, gate)
    first = torch.tensor([0, *lens]).cumsum(0)[:-1]
    t = torch.arange(most)
    inside = t[:, None] < torch.tensor(lens, dtype=torch.int64).reshape(1, N)
    rows = (first + t[:, None])[inside]

    def side(x, fill):   # [most, N, C]: behind an end the state stands still
        out = torch.full((most, N, C), fill, dtype=torch.float64)
        out[inside] = x[rows]
        return out

    def packed(x):
        out = torch.zeros(T, C, dtype=torch.float64)
        out[rows] = x[inside]
        return out

    A, U = side(a, 1.0), side(u, 0.0)
    live = inside[:, :, None].double()
    h = torch.zeros(N, C, dtype=torch.float64) if h0 is None else h0.double()
    size, off = h.abs(), torch.zeros_like(h)
    H, S, O, before = [], [], [], []   # states, sizes, how far off; and those before a row
    for i in range(most):
        before.append((h, size, off))
        h = A[i] * h + U[i]
        size = A[i].abs() * size + U[i].abs()
        off = A[i].abs() * off + eps * size * live[i]
        H.append(h), S.append(size), O.append(off)
    H, O = packed(torch.stack(H)), packed(torch.stack(O))
    out = {"o": (q * H, q.abs() * O + eps * (q * H).abs()), "ht": (h, off)}
    if do is None:
        return out
    do = do.double()
    D = side(do * q, 0.0)
    c = torch.zeros(N, C, dtype=torch.float64) if dht is None else dht.double()
    size, off = c.abs(), torch.zeros_like(c)
    E, dA, offE, offA = [], [], [], []
    for i in range(most - 1, -1, -1):
        e, esize, eoff = D[i] + c, D[i].abs() * (1 + eps) + size, off
        eoff = eoff + eps * esize * live[i]
        b, bsize, boff = before[i]
        E.append(e), offE.append(eoff)
        dA.append(e * b), offA.append(eoff * bsize + esize * boff + 2 * eps * esize * bsize)
        c, size = A[i] * e, A[i].abs() * esize
        off = A[i].abs() * eoff + eps * size * live[i]
    E, dA, offE, offA = (packed(torch.stack(x[::-1])) for x in (E, dA, offE, offA))
    out.update(du=(E, offE), dg=(dA * slope, offA * slope.abs() + 2 * eps * (dA * slope).abs()),
               dq=(do * H, do.abs() * O + eps * (do * H).abs()), dh0=(c, off))
    return out


def _norm(x, groups, weight, bias, eps, kind):
    v = x.reshape(x.shape[0], groups, -1)
    if kind == "layer":
        v = v - v.mean(2, keepdim=True)
    v = (v / torch.sqrt((v * v).mean(2, keepdim=True) + eps)).reshape(x.shape)
    v = v if weight is None else v * weight.double()
    return v if bias is None else v + bias.double()


def gated_norm(x, z, num_groups=1, weight=None, bias=None, eps=1e-5, activation="silu", kind="rms"):
    """Rows [N, C]; differentiable."""
    z = z.double()
    s = 1 / (1 + torch.exp(-z))
    return _norm(x.double(), num_groups, weight, bias, eps, kind) * (z * s if activation == "silu" else s)


def residual_norm(x, residual, weight=None, bias=None, eps=1e-5, kind="rms", scale=None, post_norm=False, post_weight=None,
                  keep=None, p=0.0):
    """(y, sum) of rows [N, C]; keep: the dropout's mask, or None."""
    v = _norm(x.double(), 1, post_weight, None, eps, kind) if post_norm else x.double()
    if keep is not None:
        v = torch.where(keep, v * dropout_scale(p), torch.zeros_like(v))
    if scale is not None:
        v = v * (scale.double() if torch.is_tensor(scale) else scale)
    s = residual.double() + v
    return _norm(s, 1, weight, bias, eps, kind), s


def philox(counter, key):
    """Philox4x32-10: counter [n, 4] and key of two 32-bit words -> [n, 4]."""
    c = [np.asarray(counter[:, i], dtype=np.uint64) for i in range(4)]
    k = [int(key[0]), int(key[1])]
    low = np.uint64(0xffffffff)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xffffffff, (k[1] + 0xBB67AE85) & 0xffffffff]
    return np.stack(c, 1).astype(np.uint32)


def dropout_scale(p):
    t = round(p * 65536)
    return 65536 / (65536 - t) if t < 65536 else 0.0


def dropout_keep(n, p, seed, subsequence=0, first=0):
    """Which of the elements first .. first + n of a tensor stay."""
    blocks = np.arange(first // 8, (first + n + 7) // 8, dtype=np.uint64)
    counter = np.stack([blocks & np.uint64(0xffffffff), blocks >> np.uint64(32), np.full_like(blocks, subsequence),
                        np.zeros_like(blocks)], 1)
    seed &= (1 << 64) - 1
    words = philox(counter, (seed & 0xffffffff, seed >> 32))
    bits = np.stack([words & 0xffff, words >> 16], 2).reshape(-1)[first % 8:][:n]
    return torch.from_numpy(bits >= round(p * 65536))
