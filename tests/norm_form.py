"""Group norm with an activation in 64 bits, forward and backward by hand, with a
hook wherever the kernels round (as tests/delta_chunk_form.py has it for the delta
rule) and places where a mistake of the kernels' joins can be put.

``hook(name, x, scale, n)``: a value, the size of its terms or partial sums, and the
number of roundings that it takes, each uniform in half a step either way:
sqrt(n / 3) 2^-24 of the scale in the root mean square."""
import torch

U = 2.0 ** -24


def exact(name, x, scale, n):
    return x


def roundings(seed):
    gen = torch.Generator().manual_seed(seed)
    return lambda name, x, scale, n: x + (n / 3) ** 0.5 * U * scale * torch.randn(x.shape, generator=gen, dtype=x.dtype)


def _mean(x, part=None):
    """Over positions and a group's channels, of all positions or of `part` of them."""
    return (x if part is None else x[:, part]).mean((1, 3), keepdim=True)


def run(x, G, w, b, eps, act, dy, hook=exact, lost=None):
    """y, dx, dw, db of x [N, L, C].  lost: None, ("moments", rows), the positions
    whose moments are not joined; "between", the slices' means' part of the
    variance, of slices of up to 128 positions; ("sums", rows), positions left out of the
    backward's two sums; ("columns", rows), of dw and db; "means", both sums."""
    N, L, C = x.shape
    keep = slice(None)
    kind = lost[0] if isinstance(lost, tuple) else lost
    if isinstance(lost, tuple):
        keep = torch.ones(L, dtype=torch.bool)
        keep[lost[1]] = False
    x, dy = (t.double().reshape(N, L, G, C // G) for t in (x, dy))
    w, b = (t.double().reshape(G, C // G) for t in (w, b))
    # sums of m values: 32 in a thread, then by pairs: at most 64 roundings of the
    # partial sums, whose mean is no larger than the values' root mean square
    size = _mean(x ** 2).sqrt()
    part = keep if kind == "moments" else None
    mean = hook("mean", _mean(x, part), size, 64)
    var = _mean((x - mean) ** 2, part)
    if kind == "between":
        var = torch.stack([((s - _mean(s)) ** 2).sum((1, 3), keepdim=True) for s in x.split(min(128, L // 2), 1)]).sum(0) / (L * (C // G))
    rstd = 1 / torch.sqrt(hook("var", var, var, 64) + eps)
    rstd = hook("rstd", rstd, rstd, 6)
    xh = (x - mean) * rstd
    xh = hook("x^", xh, xh.abs(), 3)
    z = hook("z", xh * w + b, (xh * w).abs() + b.abs(), 2)
    if act == "relu":
        y, slope = z.clamp(min=0), (z > 0).double()
    elif act == "silu":
        s = torch.sigmoid(z)
        y = hook("y", z * s, (z * s).abs() * (1 + z.abs()), 6)
        slope = hook("slope", s * (1 + z * (1 - s)), (1 + z.abs()) ** 2 * s, 8)
    else:
        y, slope = z, torch.ones_like(z)
    dz = hook("dz", dy * slope, (dy * slope).abs(), 1)
    h = hook("h", dz * w, (dz * w).abs(), 1)
    part = keep if kind == "sums" else None
    s0, s1 = _mean(h, part), _mean(h * xh, part)
    if part is not None:
        s0, s1 = (t * (keep.sum() / L) for t in (s0, s1))
    s0, s1 = hook("s0", s0, _mean(h ** 2).sqrt(), 64), hook("s1", s1, _mean((h * xh) ** 2).sqrt(), 64)
    if kind == "means":
        s0, s1 = 0 * s0, 0 * s1
    dx = hook("dx", rstd * (h - s0 - xh * s1), rstd * (h.abs() + s0.abs() + (xh * s1).abs()), 4)
    # columns: N L terms of no common sign; a rounding each, of partial sums that grow to the whole
    cols = slice(None) if kind != "columns" else keep

    def column(name, t):
        total, size = t[:, cols].sum((0, 1)), (t ** 2).sum((0, 1)).sqrt()
        return hook(name, total, (size + total.abs()) * 0.71, N * L).reshape(C)
    return y.reshape(N, L, C), dx.reshape(N, L, C), column("dw", dz * xh), column("db", dz)
