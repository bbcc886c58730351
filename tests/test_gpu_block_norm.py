"""The norms around a block and the counter-based dropout against their definitions in
64 bits.

Tolerance, with u = 2^-24 (half a step of fp32).  A row's sum adds up to 8 values in a
lane, then by pairs over 64 lanes and up to 16 in turn: at most 30 roundings, so a mean
of squares is off by 33 u of itself, 1 / its root by 20 u, and where a mean is taken out
first that is off by 31 u of the largest |x|.  Normalised values n are off by
OFF = 54 u (max |x| / deviation + 1).  A sigmoid is off by (8 + |z|) u.  Products and sums
of a few such factors: the sizes of the factors times the sum of their offs.  Sums
over rows add N terms one by one in a lane at worst.  Outputs are rounded once to
their types."""
import pytest
import torch

from oracle import block

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, B16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF = {F32: U, B16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {F32: 1e-37, B16: 1e-37, F16: 2.0 ** -25}
TYPES = [F32, B16, F16]
# rows, channels, groups: one value, odd ones, groups of one lane and of whole wavefronts, more groups
# than a workgroup has lane groups, rows of several wavefronts, the widest
GATED = [(1, 1, 1), (5, 8, 2), (77, 96, 3), (300, 512, 8), (3, 75, 5), (9, 1000, 1), (33, 2048, 16), (2, 8192, 1), (4, 50, 1),
         (1000, 24, 2), (6, 4096, 1024), (700, 768, 3), (13, 1536, 2), (4000, 64, 1)]
ROWS = [(1, 1), (5, 8), (77, 48), (300, 512), (3, 75), (9, 1000), (40, 2048), (2, 8192), (4, 50), (3000, 24), (600, 1024),
        (7, 4100), (5, 515)]


def rnd(gen, *shape):
    return torch.randn(*shape, generator=gen)


def near(name, got, want, tol, dtype):
    tol = tol + HALF[dtype] * (want.abs() + tol) + TINY[dtype]
    err = (got.double().cpu() - want).abs()
    assert got.dtype == dtype and got.shape == want.shape, name
    assert bool((err <= tol).all()), f"{name}: {float((err / tol).max()):.3g} of the bound, worst {float(err.max()):.3g}"


def norm_sizes(x, G, kind, eps=1e-5):
    """(how far normalised values may be off, the largest of them, the largest 1 / deviation)"""
    v = x.double().reshape(x.shape[0], G, -1)
    if kind == "layer":
        v = v - v.mean(2, keepdim=True)
    rstd = ((v * v).mean(2, keepdim=True) + eps).rsqrt()
    n = float((v * rstd).abs().max())
    return 54 * U * (float((x.abs().double().reshape(v.shape) * rstd).max()) + 1), n, float(rstd.max())


def big(t, other=1.0):
    return other if t is None else float(t.abs().max())


# -------------------------------------------------------------------- gated --
def gated_case(shape, dtype, seed):
    N, C, G = shape
    gen = torch.Generator().manual_seed(seed)
    x = (1.5 * rnd(gen, N, C) + rnd(gen, C)).to(dtype)
    return x, rnd(gen, N, C).to(dtype), 1 + 0.3 * rnd(gen, C), 0.3 * rnd(gen, C), rnd(gen, N, C).to(dtype)


def check_gated(dev, shape, dtype, kind, act, w, b, x, z, dy, lay=lambda t: t):
    from ssla_amd.norm import gated_norm
    G, eps = shape[2], 1e-5
    leaves64 = [None if t is None else t.double().requires_grad_() for t in (x, z, w, b)]
    ref = block.gated_norm(*leaves64[:2], G, *leaves64[2:], eps, act, kind)
    want = torch.autograd.grad(ref, [t for t in leaves64 if t is not None], dy.double())
    leaves = [None if t is None else lay(t.to(dev)).detach().requires_grad_() for t in (x, z, w, b)]
    with torch.no_grad():
        alone = gated_norm(*leaves[:2], G, *leaves[2:], eps=eps, activation=act, kind=kind)
    y = gated_norm(*leaves[:2], G, *leaves[2:], eps=eps, activation=act, kind=kind)
    assert torch.equal(y, alone)
    got = torch.autograd.grad(y, [t for t in leaves if t is not None], lay(dy.to(dev)))
    off, n, rstd = norm_sizes(x, G, kind)
    zmax = big(z)
    s_off, a_max = (8 + zmax) * U, max(zmax, 1.0) if act == "silu" else 1.0
    wm, bm = big(w), big(b, 0.0)
    v, v_off = n * wm + bm, off * wm + 3 * U * (n * wm + bm)
    a_off = a_max * (s_off + 2 * U)
    near("y", y.detach(), ref.detach(), v_off * a_max + v * (a_off + U * a_max), dtype)
    d = big(dy)
    slope, slope_off = 1.1, (zmax + 1) * (3 * s_off + 4 * U)   # (of g s (1 - s) + s)
    i = iter(zip(got, want))
    g, r = next(i)
    h, h_off = d * a_max * wm, d * wm * (a_off + 3 * U * a_max)
    # means of h and h n over the group, and n times the second: each at most h n, off by 33 U of that and the factors' offs
    near("dx", g, r, rstd * (1 + 20 * U) * (2 * h_off * (1 + n * n) + h * (1 + n) ** 2 * (60 * U) + 3 * h * (1 + n) * off), dtype)
    g, r = next(i)
    near("dz", g, r, d * (v_off * slope + v * slope_off + 3 * U * v * slope), dtype)
    N = shape[0]
    if w is not None:
        g, r = next(i)
        near("dw", g, r, torch.full_like(r, N * d * (a_max * off + n * (a_off + 3 * U * a_max) + a_max * n * (N + 64) * U)), F32)
    if b is not None:
        g, r = next(i)
        near("db", g, r, torch.full_like(r, N * d * (a_off + U * a_max + a_max * (N + 64) * U)), F32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", GATED)
def test_gated(dev, shape, dtype):
    x, z, w, b, dy = gated_case(shape, dtype, seed=shape[1])
    for kind in ("rms", "layer"):
        for act in ("silu", "sigmoid"):
            check_gated(dev, shape, dtype, kind, act, w, b, x, z, dy)
        check_gated(dev, shape, dtype, kind, "silu", None, b, x, z, dy)
        check_gated(dev, shape, dtype, kind, "silu", w, None, x, z, dy)
        check_gated(dev, shape, dtype, kind, "silu", None, None, x, z, dy)


def test_gated_slices(dev):
    """x and gate as columns of one matrix, off 16-byte borders too, and in another
    memory order; more dimensions; a gradient of one input alone."""
    from ssla_amd.norm import gated_norm
    shape = (50, 48, 4)
    for dtype in (F32, B16):
        x, z, w, b, dy = gated_case(shape, dtype, seed=4)
        for pad in (0, 3, 4):
            def lay(t, pad=pad):
                if t.dim() == 1:
                    return torch.cat([torch.zeros(pad, device=t.device), t])[pad:]
                wide = torch.zeros(50, 150, dtype=t.dtype, device=t.device)
                wide[:, 48 + pad:96 + pad] = t
                return wide[:, 48 + pad:96 + pad]
            check_gated(dev, shape, dtype, "rms", "silu", w, b, x, z, dy, lay)
        check_gated(dev, shape, dtype, "layer", "silu", w, b, x, z, dy, lambda t: t.t().contiguous().t() if t.dim() == 2 else t)
        full = [t.to(dev) for t in (x, z, w, b)]
        y = gated_norm(*full[:2], 4, *full[2:])
        assert torch.equal(gated_norm(full[0].view(5, 10, 48), full[1].view(5, 10, 48), 4, *full[2:]).view(50, 48), y)
        leaves = [t.clone().requires_grad_() for t in full]
        both = torch.autograd.grad(gated_norm(*leaves[:2], 4, *leaves[2:]), leaves, dy.to(dev))
        for i in range(4):
            args = [t.clone().requires_grad_(k == i) for k, t in enumerate(full)]
            (g,) = torch.autograd.grad(gated_norm(*args[:2], 4, *args[2:]), args[i], dy.to(dev))
            assert torch.equal(g, both[i])


# ----------------------------------------------------------------- residual --
def residual_case(shape, dtype, rdtype, seed):
    N, C = shape
    gen = torch.Generator().manual_seed(seed)
    x, r = (1.5 * rnd(gen, N, C) + 0.5 * rnd(gen, C)).to(dtype), (2 * rnd(gen, N, C)).to(rdtype)
    return (x, r, 1 + 0.3 * rnd(gen, C), 0.3 * rnd(gen, C), 0.5 + 0.2 * rnd(gen, C), 1 + 0.3 * rnd(gen, C),
            rnd(gen, N, C).to(dtype), rnd(gen, N, C).to(rdtype))


def check_residual(dev, case, kind, post, scale, affine, p, seed=77, sub=3, grads="both"):
    from ssla_amd.norm import residual_norm
    x, r, w, b, gamma, w2, dy, ds = case
    N, C = x.shape
    w, b, w2 = w if affine else None, b if affine else None, w2 if post and affine else None
    gamma = gamma if scale == "vector" else None
    alpha = 0.75 if scale == "number" else None
    keep = block.dropout_keep(N * C, p, seed, sub).view(N, C) if p else None
    names = ("x", "r", "w", "b", "gamma", "w2")
    l64 = {n: None if t is None else t.double().requires_grad_() for n, t in zip(names, (x, r, w, b, gamma, w2))}
    sc = alpha if gamma is None else l64["gamma"]
    ref = block.residual_norm(l64["x"], l64["r"], l64["w"], l64["b"], 1e-5, kind, sc, post, l64["w2"], keep, p)
    given = {"both": (dy, ds), "y": (dy, None), "sum": (None, ds)}[grads]
    outs = [o for o, g in zip(ref, given) if g is not None]
    gs = [g for g in given if g is not None]
    wanted = [n for n in names if l64[n] is not None and not (grads == "sum" and n in ("w", "b"))]
    want = torch.autograd.grad(outs, [l64[n] for n in wanted], [g.double() for g in gs])
    ld = {n: None if t is None else t.to(dev).requires_grad_() for n, t in zip(names, (x, r, w, b, gamma, w2))}

    def call():
        return residual_norm(ld["x"], ld["r"], ld["w"], ld["b"], kind=kind, scale=alpha if gamma is None else ld["gamma"],
                             post_norm=post, post_weight=ld["w2"], p=p, seed=seed, subsequence=sub)
    with torch.no_grad():
        alone = call()
    out = call()
    assert all(torch.equal(a, c) for a, c in zip(out, alone))
    got = torch.autograd.grad([o for o, g in zip(out, given) if g is not None], [ld[n] for n in wanted],
                              [g.to(dev) for g in gs])
    off2, n2, rstd2 = norm_sizes(x, 1, kind) if post else (0.0, big(x), 1.0)
    c = (alpha or 1.0) * big(gamma) * (block.dropout_scale(p) if p else 1.0)
    w2m = big(w2)
    branch, branch_off = c * n2 * w2m, c * w2m * (off2 + 5 * U * n2)
    s = float(ref[1].detach().abs().max())
    s_off = branch_off + U * (s + branch)
    near("sum", out[1].detach(), ref[1].detach(), s_off, r.dtype)
    off, n, rstd = norm_sizes(ref[1].detach(), 1, kind)
    off = off + s_off * rstd * (2 + n * n)   # (what the sum is off by, through the norm)
    wm, bm = big(w), big(b, 0.0)
    near("y", out[0].detach(), ref[0].detach(), off * wm + 3 * U * (n * wm + bm), x.dtype)
    d, dsm = (big(dy) if given[0] is not None else 0.0), (big(ds) if given[1] is not None else 0.0)
    h = d * wm
    dr = rstd * h * (1 + n) ** 2 + dsm
    dr_off = rstd * (1 + 20 * U) * (h * (1 + n) ** 2 * 70 * U + 3 * h * (1 + n) * off) + s_off * rstd * rstd * h * (2 + n) ** 3 + U * dr
    res = dict(zip(wanted, zip(got, want)))
    near("dr", *res["r"], dr_off, r.dtype)
    dp, dp_off = c * dr * w2m, c * w2m * (dr_off + 5 * U * dr)
    x_off = dp_off
    if post:
        x_off = rstd2 * (1 + 20 * U) * (2 * dp_off * (1 + n2 * n2) + dp * (1 + n2) ** 2 * 60 * U + 3 * dp * (1 + n2) * off2)
    near("dx", *res["x"], x_off, x.dtype)
    many = (N + 64) * U
    if "w" in res:
        near("dw", *res["w"], torch.full_like(w.double(), N * d * (off + n * 3 * U + n * many)), F32)
        near("db", *res["b"], torch.full_like(w.double(), N * d * (U + many)), F32)
    cs = c / big(gamma)
    if "gamma" in res:
        v, v_off = n2 * w2m, w2m * (off2 + 3 * U * n2)
        near("dgamma", *res["gamma"], torch.full_like(gamma.double(), N * cs * (dr_off * v + dr * v_off + dr * v * (4 * U + many))), F32)
    if "w2" in res:
        near("dw2", *res["w2"], torch.full_like(w2.double(), N * c * (dr_off * n2 + dr * off2 + dr * n2 * (6 * U + many))), F32)


@pytest.mark.parametrize("dtype,rdtype", [(F32, F32), (B16, B16), (B16, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("shape", ROWS)
def test_residual(dev, shape, dtype, rdtype):
    case = residual_case(shape, dtype, rdtype, seed=shape[1])
    for kind in ("rms", "layer"):
        check_residual(dev, case, kind, False, None, True, 0.0)
        check_residual(dev, case, kind, True, "vector", True, 0.25)
    check_residual(dev, case, "rms", True, "number", False, 0.0)
    check_residual(dev, case, "layer", False, "vector", False, 0.5)


@pytest.mark.parametrize("grads", ["y", "sum"])
def test_residual_one_gradient(dev, grads):
    case = residual_case((60, 96), B16, F32, seed=1)
    check_residual(dev, case, "rms", True, "vector", True, 0.1, grads=grads)
    check_residual(dev, case, "layer", False, None, True, 0.0, grads=grads)


def test_single_inputs_and_layouts(dev):
    """A gradient of one tensor alone is that of all; inputs in another memory order, off a
    16-byte border, of more dimensions."""
    from ssla_amd.norm import residual_norm
    x, r, w, b, gamma, w2, dy, ds = (t.to(dev) for t in residual_case((60, 40), F32, F32, seed=2))
    names = ("x", "r", "w", "b", "gamma", "w2")

    def run(t, lay=lambda t: t):
        return residual_norm(lay(t["x"]), lay(t["r"]), t["w"], t["b"], scale=t["gamma"], post_norm=True, post_weight=t["w2"],
                             p=0.3, seed=5)
    full = dict(zip(names, (x, r, w, b, gamma, w2)))
    leaves = {n: t.clone().requires_grad_() for n, t in full.items()}
    out = run(leaves)
    both = torch.autograd.grad(out, list(leaves.values()), (dy, ds))
    for i, n in enumerate(names):
        args = {m: t.clone().requires_grad_(m == n) for m, t in full.items()}
        assert torch.equal(torch.autograd.grad(run(args), args[n], (dy, ds))[0], both[i]), n
    for lay in (lambda t: t.t().contiguous().t(), lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(60, 40),
                lambda t: torch.cat([t, t], 1)[:, :40]):
        assert all(torch.equal(a, c) for a, c in zip(run(full, lay), out))
    for a, c in zip(run(full, lambda t: t.view(3, 4, 5, 40)), out):
        assert a.shape == (3, 4, 5, 40) and torch.equal(a.view(60, 40), c)


def test_edges(dev):
    """Rows of zeros; NaN and infinities stay in their row, and dropped ones nowhere;
    no rows; p of 1."""
    from ssla_amd.norm import gated_norm, residual_norm
    x, r, w, b, gamma, w2, dy, ds = (t.to(dev) for t in residual_case((30, 64), F32, F32, seed=3))
    y, s = residual_norm(torch.zeros_like(x), torch.zeros_like(r), w, b, kind="layer")
    assert torch.equal(y, b.expand_as(y)) and not s.any()
    assert not gated_norm(torch.zeros_like(x), r, 4).any()
    clean = residual_norm(x, r, w, b)
    cg = gated_norm(x, r, 4, w)
    for v in (torch.nan, torch.inf):
        bad = x.clone()
        bad[7, 5] = v
        y, s = residual_norm(bad, r, w, b)
        rest = torch.arange(30) != 7
        assert torch.equal(y[rest], clean[0][rest]) and not y[7].isfinite().all() and not s[7, 5].isfinite()
        y = gated_norm(bad, r, 4, w)
        assert torch.equal(y[rest], cg[rest]) and torch.equal(y[7, 16:], cg[7, 16:])
    keep = block.dropout_keep(30 * 64, 0.5, 9).view(30, 64).to(dev)
    holes = torch.where(keep, x, torch.nan)
    assert all(torch.equal(a, c) for a, c in zip(residual_norm(holes, r, w, p=0.5, seed=9), residual_norm(x, r, w, p=0.5, seed=9)))
    leaf, other = holes.clone().requires_grad_(), x.clone().requires_grad_()
    g = [torch.autograd.grad(residual_norm(t, r, w, p=0.5, seed=9), t, (dy, ds))[0] for t in (leaf, other)]
    assert torch.equal(*g)
    assert torch.equal(residual_norm(x, r, p=1.0, seed=1)[1], r)
    for shape in ((0, 64), (2, 0, 64)):
        e = torch.zeros(shape, device=dev, requires_grad=True)
        wl, gl = w.clone().requires_grad_(), gamma.clone().requires_grad_()
        y, s = residual_norm(e, e.detach(), wl, scale=gl)
        (y.sum() + s.sum() + gated_norm(e, e, 2, wl).sum()).backward()
        assert y.shape == shape and e.grad.shape == shape and not wl.grad.any() and not gl.grad.any()
    row = residual_norm(x[0], r[0], w, b)
    assert row[0].shape == (64,) and torch.equal(row[0], residual_norm(x[:1], r[:1], w, b)[0][0])


def test_the_same_every_time(dev):
    from ssla_amd.norm import gated_norm, residual_norm
    x, r, w, b, gamma, w2, dy, ds = (t.to(dev) for t in residual_case((5000, 200), B16, F32, seed=3))
    leaves = [t.requires_grad_() for t in (x, r, w, b, gamma, w2)]
    z = dy.clone().requires_grad_()
    runs = []
    for _ in range(3):
        out = residual_norm(x, r, w, b, scale=gamma, post_norm=True, post_weight=w2, p=0.1, seed=3)
        runs.append(torch.autograd.grad(out, leaves, (dy, ds)) +
                    torch.autograd.grad(gated_norm(x, z, 4, w, b), (x, z, w, b), dy))
    assert all(torch.equal(a, c) for q in runs[1:] for a, c in zip(runs[0], q))


def test_differences(dev):
    """A direction's slope against central differences in fp32: their distance bounds the
    third-order term, the loss's rounding is 1,500 sums of values that are off by 2^-19."""
    from ssla_amd.norm import gated_norm, residual_norm
    x, r, w, b, gamma, w2, dy, ds = residual_case((30, 24), F32, F32, seed=6)
    gen = torch.Generator().manual_seed(1)
    for kind in ("rms", "layer"):
        def res(*t):
            return residual_norm(*t[:4], kind=kind, scale=t[4], post_norm=True, post_weight=t[5], p=0.2, seed=8)

        def gat(*t):
            return (gated_norm(t[0], t[1], 3, t[2], t[3], kind=kind),)
        for f, ins, given in ((res, (x, r, w, b, gamma, w2), (dy, ds)), (gat, (x, r, w, b), (dy,))):
            d = [rnd(gen, *t.shape) for t in ins]
            leaves = [t.to(dev).requires_grad_() for t in ins]
            grads = torch.autograd.grad(f(*leaves), leaves, [g.to(dev) for g in given])
            slope = sum(float((g.double().cpu() * e).sum()) for g, e in zip(grads, d))

            def loss(h):
                out = f(*((t + h * e).to(dev) for t, e in zip(ins, d)))
                return sum(float((o.double().cpu() * g).sum()) for o, g in zip(out, given))
            h = 2.0 ** -7
            two = [(loss(h) - loss(-h)) / (2 * h), (loss(2 * h) - loss(-2 * h)) / (4 * h)]
            diff = (4 * two[0] - two[1]) / 3
            assert abs(diff - slope) <= abs(two[0] - two[1]) + 1500 * 2.0 ** -19 / h, (kind, f.__name__)


# ------------------------------------------------------------------ dropout --
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 7, 8, 9, 1000, 70001])
def test_dropout(dev, n, dtype):
    from ssla_amd.dropout import counter_dropout
    gen = torch.Generator().manual_seed(n)
    x, dy = rnd(gen, n).to(dtype), rnd(gen, n).to(dtype)
    for p, seed, sub in ((0.1, 0, 0), (0.5, -(1 << 63), 7), (0.999, (1 << 63) - 1, (1 << 32) - 1), (0.0, 5, 0), (1.0, 5, 0),
                         (2.0 ** -17 + 1e-9, 12, 0), (2.0 ** -18, 12, 0)):
        keep, f = block.dropout_keep(n, p, seed, sub), block.dropout_scale(p)
        for s in (seed, torch.tensor([seed], device=dev)):
            leaf = x.to(dev).requires_grad_()
            y = counter_dropout(leaf, p, s, sub)
            (g,) = torch.autograd.grad(y, leaf, dy.to(dev))
            for got, src in ((y.detach(), x), (g, dy)):
                # the factor is rounded once to fp32, the product once more
                near("y", got, torch.where(keep, src.double() * f, 0.0), 2 * U * src.double().abs() * f, dtype)
                assert torch.equal(got.cpu() == 0, ~keep | (src == 0) | (src.double().abs() * f < TINY[dtype]))


def test_dropout_layouts(dev):
    """Places go by the logical order; views off 16 bytes; what is dropped may be NaN; the
    seed may change between forward and backward."""
    from ssla_amd.dropout import counter_dropout
    x = rnd(torch.Generator().manual_seed(1), 40, 30).to(dev)
    y = counter_dropout(x, 0.4, 11)
    assert torch.equal(counter_dropout(x.t().contiguous().t(), 0.4, 11), y)
    assert torch.equal(counter_dropout(torch.cat([x.new_zeros(1), x.reshape(-1)])[1:].view(40, 30), 0.4, 11), y)
    assert torch.equal(counter_dropout(torch.where(y == 0, torch.nan, x), 0.4, 11), y)
    seed = torch.tensor([11], device=dev)
    leaf = x.clone().requires_grad_()
    out = counter_dropout(leaf, 0.4, seed)
    seed += 1
    (g,) = torch.autograd.grad(out, leaf, torch.ones_like(out))
    assert torch.equal(g == 0, y == 0) and not torch.equal(counter_dropout(x, 0.4, seed), y)
    assert counter_dropout(x[:0], 0.4, 1).shape == (0, 30)


def test_dropout_past_32_bits_of_bytes(dev):
    """Elements behind 2^32 bytes and 2^31 elements have bits of their own."""
    from ssla_amd.dropout import counter_dropout
    n = (1 << 31) + 4096
    y = counter_dropout(torch.ones(n, dtype=B16, device=dev), 0.5, 3)
    for first in (0, (1 << 31) - 2048, n - 4096):
        keep = block.dropout_keep(4096, 0.5, 3, first=first)
        assert torch.equal(y[first:first + 4096].cpu() != 0, keep)


def test_residual_drops_what_dropout_drops(dev):
    from ssla_amd.dropout import counter_dropout
    from ssla_amd.norm import residual_norm
    for dtype, C in ((F32, 96), (B16, 96), (F16, 75), (B16, 2048)):
        x, r, w, *_ = (t.to(dev) for t in residual_case((33, C), dtype, F32, seed=C))
        y, s = residual_norm(x, torch.zeros_like(r), w, p=0.35, seed=21, subsequence=4)
        assert torch.equal(s == 0, (counter_dropout(x, 0.35, 21, 4) == 0) | (x == 0))


# ------------------------------------------------------------ run together --
def test_a_block_in_a_graph(dev):
    """A linear-attention block as it is used (norm, projections, gated recurrence, gated norm
    by heads, projection, dropout, residual and the next norm): a training step captured once
    and replayed on changing inputs and seeds, with eager steps in between, and its
    gradients against the definitions in 64 bits."""
    from ssla_amd.norm import gated_norm, residual_norm
    from ssla_amd.scan import gated_scan
    gen = torch.Generator().manual_seed(0)
    T, C, G, lens = 700, 64, 4, [300, 1, 399]
    t64 = {"x": rnd(gen, T, C), "r": rnd(gen, T, C), "win": rnd(gen, 4 * C, C) / 8, "wout": rnd(gen, C, C) / 8,
           "nw": 1 + 0.1 * rnd(gen, C), "w": 1 + 0.1 * rnd(gen, C), "ls": 0.5 + 0.1 * rnd(gen, C)}
    dy, ds = rnd(gen, T, C), rnd(gen, T, C)
    names = list(t64)

    def forward(t, cu, seed):
        u, g, q, z = torch.nn.functional.linear(t["x"], t["win"]).split(C, 1)
        o, _ = gated_scan(u, g, cu, q=q, gate="sigmoid")
        a = gated_norm(o, z, G, t["nw"])
        return residual_norm(torch.nn.functional.linear(a, t["wout"]), t["r"], t["w"], scale=t["ls"], p=0.1, seed=seed)

    cu = torch.tensor([0, *lens]).cumsum(0).to(dev)
    gy, gs = dy.to(dev), ds.to(dev)

    def step(t, seed):
        out = forward(t, cu, seed)
        return *(o.detach() for o in out), *torch.autograd.grad(out, [t[n] for n in names], (gy, gs))

    static = {n: v.to(dev).requires_grad_() for n, v in t64.items()}
    seed = torch.tensor([5], device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static, seed)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(static, seed)
    for i in range(4):
        with torch.no_grad():
            static["x"].copy_(t64["x"] * (1 + 0.1 * i))
        seed.fill_(100 + i)
        graph.replay()
        want = step({n: v.detach().clone().requires_grad_() for n, v in static.items()}, seed)
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(got, want)), i

    d = {n: v.double().requires_grad_() for n, v in t64.items()}
    u, g, q, z = torch.nn.functional.linear(d["x"], d["win"]).split(C, 1)
    h, rows, t = [], torch.zeros(C, dtype=torch.float64), 0
    for n in lens:
        rows = torch.zeros(C, dtype=torch.float64)
        for _ in range(n):
            rows = torch.sigmoid(g[t]) * rows + u[t]
            h.append(rows)
            t += 1
    a = block.gated_norm(q * torch.stack(h), z, G, d["nw"])
    keep = block.dropout_keep(T * C, 0.1, 5).view(T, C)
    out = block.residual_norm(torch.nn.functional.linear(a, d["wout"]), d["r"], d["w"], scale=d["ls"], keep=keep, p=0.1)
    ref = *(o.detach() for o in out), *torch.autograd.grad(out, [d[n] for n in names], (dy.double(), ds.double()))
    seed.fill_(5)
    got = step({n: v.to(dev).requires_grad_() for n, v in t64.items()}, seed)
    for n, b, c in zip(["y", "sum", *names], got, ref):
        # products of 64 and up to 700 terms of fp32 lie between: 2^-14 of the largest value, some
        # 300 roundings of it, and a lost factor or term is far outside
        assert float((b.double().cpu() - c).abs().max()) <= 2.0 ** -14 * float(c.abs().max()), n


@pytest.mark.parametrize("dtype", [F32, B16])
@pytest.mark.parametrize("N,C,G", [(1, 8, 2), (2, 64, 1), (1023, 64, 4), (16411, 1024, 4), (5001, 75, 1), (5003, 75, 5), (3077, 2048, 16),
                                   (4099, 520, 1), (1537, 1032, 1), (70001, 24, 3), (2500, 4096, 1024), (777, 5000, 1)])
def test_sums_over_rows_count_every_row_once(dev, N, C, G, dtype):
    """Whole numbers whose sums over the rows are known: x is 1 or -1, so it is its own norm to
    8 U of itself (C ones times 1 / C, the root, a product), the gate is open and the
    gradients are integers up to 3 with signs at random.  A lane adds some hundred terms at
    most, so partial sums stay within 6 times 2.2 times 10 there and 13 N^0.5 behind: N
    roundings of at most 130 U and some hundred of 13 N^0.5 U, either way alike, are 0.003 in
    the root mean square for the longest.  A row lost or counted twice is a whole number off
    at every channel."""
    from ssla_amd.norm import gated_norm, residual_norm
    gen = torch.Generator().manual_seed(N + C)
    x = (torch.randint(0, 2, (N, C), generator=gen) * 2 - 1).to(dtype)
    d = (torch.randint(1, 4, (N, C), generator=gen) * (torch.randint(0, 2, (N, C), generator=gen) * 2 - 1)).to(dtype)
    one = torch.ones(C, device=dev)
    dw, db = (x.double() * d.double()).sum(0), d.double().sum(0)

    def same(name, got, want):
        err = (got.double().cpu() - want).abs()
        assert float(err.max()) <= 0.5, (name, float(err.max()))

    leaves = [t.clone().requires_grad_() for t in (one, 0 * one)]
    y = gated_norm(x.to(dev), torch.full((N, C), 60.0, dtype=dtype, device=dev), G, *leaves, eps=0.0, activation="sigmoid")
    for name, got, want in zip(("dw", "db"), torch.autograd.grad(y, leaves, d.to(dev)), (dw, db)):
        same(name, got, want)
    if G > 1:
        return
    leaves = [t.clone().requires_grad_() for t in (one, 0 * one)]
    y, s = residual_norm(torch.zeros(N, C, dtype=dtype, device=dev), x.to(dev), *leaves, eps=0.0)
    for name, got, want in zip(("dw", "db"), torch.autograd.grad(y, leaves, d.to(dev)), (dw, db)):
        same("residual " + name, got, want)
    leaves = [t.clone().requires_grad_() for t in (one, one)]
    y, s = residual_norm(x.to(dev), torch.zeros(N, C, dtype=dtype, device=dev), eps=0.0, scale=leaves[0], post_norm=True,
                         post_weight=leaves[1])
    for name, got in zip(("dgamma", "dw2"), torch.autograd.grad(s, leaves, d.to(dev))):
        same(name, got, dw)


def test_rows_past_32_bits(dev):
    """Behind 2^31 values a tensor rows are read, written, normalised and dropped at their own
    places: the last are those of a short call on them alone, in both directions."""
    from ssla_amd.norm import gated_norm, residual_norm
    N, C, last = (1 << 21) + 9, 1024, slice(-16, None)
    gen = torch.Generator(device=dev).manual_seed(0)
    x, r, d = (torch.randn(N, C, generator=gen, device=dev, dtype=B16) for _ in range(3))
    x.requires_grad_(), r.requires_grad_()
    for form in (lambda a, b: (gated_norm(a, b, 8),), lambda a, b: residual_norm(a, b, post_norm=True)):
        def run(*rows):
            out = form(*rows[:2])
            return *(o.detach() for o in out), *torch.autograd.grad(out, rows[:2], (rows[2],) * len(out))
        part = run(*(t.detach()[last].clone().requires_grad_() for t in (x, r)), d[last])
        for a, b in zip(run(x, r, d), part):
            assert torch.equal(a[last], b)
    _, s = residual_norm(x.detach(), torch.zeros_like(r), p=0.25, seed=11, subsequence=3)
    keep = block.dropout_keep(16 * C, 0.25, 11, 3, first=(N - 16) * C).view(16, C)
    assert torch.equal(s[last].cpu() != 0, keep & (x.detach()[last].cpu() != 0))


def test_tensors_at_odd_16_byte_borders(dev):
    """Inputs and outputs of the C entries at 16-byte borders that are no 32-byte ones: a row of
    8 values of an fp32 stream beside 16-bit ones is 32 bytes."""
    from ssla_amd import _lib
    N, C = 37, 96
    x, r, w, b, gamma, w2, dy, ds = (t.to(dev) for t in residual_case((N, C), B16, F32, seed=9))
    lib, P, st = _lib.load(), _lib.ptr, _lib.stream_of(x)
    ws = torch.empty(lib.ssla_residual_norm_bwd_workspace_size(N, C), dtype=torch.uint8, device=dev)

    def run(bytes_off):
        def lay(t):
            n = bytes_off // t.element_size()
            return torch.cat([t.new_zeros(n), t.reshape(-1)])[n:].view(t.shape)
        a, s, d, e, y, total, dx, dr = map(lay, (x, r, dy, ds, x, r, x, r))
        sums = [torch.empty_like(w) for _ in range(4)]
        assert all(t.data_ptr() % 32 == bytes_off for t in (a, s, d, e, y, total, dx, dr))
        _lib.check(lib.ssla_residual_norm_fwd(P(a), P(s), N, C, 0, P(w), P(b), 1e-5, 1.0, P(gamma), 1, P(w2), 0.0, None, 0,
                                              P(y), P(total), _lib.SSLA_BF16, _lib.SSLA_F32, st), "fwd")
        _lib.check(lib.ssla_residual_norm_bwd(P(d), P(e), P(a), P(s), N, C, 0, P(w), 1e-5, 1.0, P(gamma), 1, P(w2), 0.0, None,
                                              0, P(dx), P(dr), *map(P, sums), _lib.SSLA_BF16, _lib.SSLA_F32, P(ws), ws.numel(),
                                              st), "bwd")
        return y, total, dx, dr, *sums
    assert all(torch.equal(p, q) for p, q in zip(run(0), run(16)))


def test_probabilities_beside_the_middle_of_two_steps(dev):
    """t = round(p 2^16) of the given p, not of its fp32 value: elements whose bits are the step
    between them stay or go by it."""
    from ssla_amd.dropout import counter_dropout
    from ssla_amd.norm import residual_norm
    n = 1 << 20
    x = torch.ones(n // 1024, 1024, device=dev)
    for p in (19660.5 / 65536 + 1e-10, 19661.5 / 65536 - 1e-10):
        keep = block.dropout_keep(n, p, 6)
        assert not torch.equal(keep, block.dropout_keep(n, float(torch.tensor(p, dtype=torch.float32)), 6))
        assert torch.equal((counter_dropout(x, p, 6) != 0).cpu().view(-1), keep)
        assert torch.equal((residual_norm(x, 0 * x, p=p, seed=6)[1] != 0).cpu().view(-1), keep)
