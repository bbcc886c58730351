"""Group norm with an activation against its definition in 64 bits.

Tolerance of a forward value, with m values in a group and u = 2^-24 (half a
step of fp32): a mean of m values is off by at most (m / 64 + 16) u of the
largest |x| (at most m / 64 values follow each other in a sum, and 16 joins),
which the deviation divides; the rest are a few operations on values no larger
than x^ = (x - mean) / deviation.  So z is off by (m / 64 + 48) u (|x| / sigma +
1) of max |w| + |b|, the activations pass at most 1.1 of that on, and the output
is rounded once to its type.  The gradients are such sums again, each factor off
by as much."""
import pytest
import torch

from oracle.delta import group_norm

pytestmark = pytest.mark.gpu
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SHAPES = [((5, 8), 2), ((1, 1), 1), ((300, 512), 8), ((77, 96), 3), ((1, 4096), 1), ((3, 7, 12), 3), ((2, 60, 76, 64), 8),
          ((2, 33, 5), 5), ((9, 130, 20), 1), ((2, 5000, 48), 4), ((1, 3, 1000), 8), ((4, 18, 30), 6)]


def inputs(shape, dtype, seed, shift=1.0):
    gen = torch.Generator().manual_seed(seed)
    C = shape[-1]
    x = (torch.randn(shape, generator=gen) * 1.5 + shift * torch.randn(C, generator=gen)).to(dtype)
    w, b = 1 + 0.3 * torch.randn(C, generator=gen), 0.3 * torch.randn(C, generator=gen)
    return x, w, b, torch.randn(shape, generator=gen).to(dtype)


def unit(x, G, w, b):
    """(how far z may be off, 1 / sigma of the tightest group)"""
    z = x.double().reshape(x.shape[0], -1, G, x.shape[-1] // G)
    m = z.shape[1] * z.shape[3]
    rstd = float((z.var((1, 3), correction=0) + 1e-5).rsqrt().max())
    big = float(x.abs().max()) * rstd + 1
    return (m / 64 + 48) * 2.0 ** -24 * big * float(w.abs().max() + b.abs().max() + 1), rstd


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape,G", SHAPES)
def test_forward(dev, dtype, shape, G):
    from ssla_amd.norm import group_norm_act
    x, w, b, _ = inputs(shape, dtype, seed=shape[-1])
    for act in (None, "relu", "silu"):
        for ww, bb in ((w, b), (None, None), (w, None), (None, b)):
            ref = group_norm(x, G, ww, bb, activation=act)
            y = group_norm_act(x.to(dev), G, *(None if t is None else t.to(dev) for t in (ww, bb)), activation=act)
            tol = 1.1 * unit(x, G, w, b)[0] + HALF[dtype] * ref.abs()
            assert y.dtype == dtype and y.shape == x.shape
            err = (y.double().cpu() - ref).abs()
            assert bool((err <= tol).all()), (act, float(err.max()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape,G", SHAPES)
@pytest.mark.parametrize("act", [None, "relu", "silu"])
def test_gradients(dev, dtype, shape, G, act):
    from ssla_amd.norm import group_norm_act
    x, w, b, dy = inputs(shape, dtype, seed=shape[0] + 7)
    rx, rw, rb = (t.double().requires_grad_() for t in (x, w, b))
    ref = torch.autograd.grad(group_norm(rx, G, rw, rb, activation=act), (rx, rw, rb), dy.double())
    dx, dw, db = (t.to(dev).requires_grad_() for t in (x, w, b))
    got = torch.autograd.grad(group_norm_act(dx, G, dw, db, activation=act), (dx, dw, db), dy.to(dev))
    off, rstd = unit(x, G, w, b)
    xh = (group_norm(x, G).abs().max() + 1).item()
    dmax = float(dy.abs().max()) * 1.1
    # a border of relu: where z is off by more than its distance to 0 the
    # gradient there may be the other side's
    z = group_norm(x, G, w, b)
    near = (z.abs() <= off) if act == "relu" else torch.zeros_like(z, dtype=torch.bool)
    per = dmax * float(w.abs().max())
    tol = 4 * off * rstd * per * xh * xh + HALF[dtype] * ref[0].abs()
    if near.any():   # such a value moves its own gradient by dy w rstd and the group's means by its share
        z4 = near.reshape(x.shape[0], -1, G, x.shape[-1] // G).double()
        share = z4.mean((1, 3), keepdim=True).expand_as(z4).reshape(x.shape)
        tol = tol + per * rstd * (near.double() + 2 * xh * xh * share)
    err = (got[0].double().cpu() - ref[0]).abs()
    assert got[0].dtype == dtype and bool((err <= tol).all()), ("dx", float(err.max()))
    rows = x.numel() // x.shape[-1]
    for name, a, r, size in (("dw", got[1], ref[1], xh), ("db", got[2], ref[2], 1.0)):
        flips = near.reshape(rows, -1).sum(0).double() * dmax * size
        bound = rows * dmax * size * (4 * off + (rows / 64 + 64) * 2.0 ** -24) + flips
        assert a.dtype == torch.float32 and bool(((a.double().cpu() - r).abs() <= bound).all()), name


def test_sums_are_the_same_every_time(dev):
    from ssla_amd.norm import group_norm_act
    x, w, b, dy = (t.to(dev) for t in inputs((3, 4000, 64), torch.bfloat16, seed=3))
    x, w, b = (t.requires_grad_() for t in (x, w, b))
    runs = [torch.autograd.grad(group_norm_act(x, 8, w, b, activation="silu"), (x, w, b), dy) for _ in range(3)]
    assert all(torch.equal(a, c) for r in runs[1:] for a, c in zip(runs[0], r))


def test_differences(dev):
    """The gradient of a direction against a central difference of the loss in
    fp32: off by at most the fourth-order term and the loss's rounding."""
    from ssla_amd.norm import group_norm_act
    x, w, b, dy = inputs((3, 20, 16), torch.float32, seed=4)
    d = [torch.randn(t.shape, generator=torch.Generator().manual_seed(i)) for i, t in enumerate((x, w, b))]
    leaves = [t.to(dev).requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(group_norm_act(leaves[0], 4, *leaves[1:], activation="silu"), leaves, dy.to(dev))
    slope = sum(float((g.double().cpu() * e).sum()) for g, e in zip(grads, d))

    def loss(h):
        a = [(t + h * e).to(dev) for t, e in zip((x, w, b), d)]
        return float((group_norm_act(a[0], 4, *a[1:], activation="silu").double().cpu() * dy).sum())

    h = 2.0 ** -6
    four = [(loss(h) - loss(-h)) / (2 * h), (loss(2 * h) - loss(-2 * h)) / (4 * h)]
    diff = (4 * four[0] - four[1]) / 3
    # the two differences are h^2 c and 4 h^2 c off: their distance bounds what is left
    assert abs(diff - slope) <= abs(four[0] - four[1]) + 1e-4 * abs(slope) + 960 * 2.0 ** -20 / h


def test_values_at_the_edges(dev):
    """A constant group is normalised to its bias; a large common offset keeps the
    precision of the centred values; NaN and infinities stay in their group;
    empty inputs; a strided input; a view that starts off 16 bytes."""
    from ssla_amd.norm import group_norm_act
    w, b = torch.rand(16).to(dev) + 1, torch.rand(16).to(dev)
    y = group_norm_act(torch.full((2, 9, 16), 3.25, device=dev), 4, w, b)
    assert torch.equal(y, b.expand_as(y))
    x = torch.randn(2, 50, 16, generator=torch.Generator().manual_seed(1))
    far = x + 4096
    tol = (800 / 64 + 48) * 2.0 ** -24 * (4110 * 1.6 + 1)
    assert float((group_norm_act(far.to(dev), 4).double().cpu() - group_norm(far, 4)).abs().max()) <= tol
    clean = group_norm_act(x.to(dev), 4, w, b, activation="silu")
    for v in (torch.nan, torch.inf):
        bad = x.clone()
        bad[1, 7, 5] = v
        y = group_norm_act(bad.to(dev), 4, w, b, activation="silu")
        assert torch.equal(y[0], clean[0]) and torch.equal(y[1, :, :4], clean[1, :, :4])
        assert torch.equal(y[1, :, 8:], clean[1, :, 8:]) and y[1, :, 4:8].isnan().all()
    for shape in ((0, 16), (2, 0, 16)):
        e = torch.zeros(shape, device=dev, requires_grad=True)
        wl = w.clone().requires_grad_()
        y = group_norm_act(e, 4, wl, b)
        y.sum().backward()
        assert y.shape == shape and e.grad.shape == shape and not wl.grad.any()
    grid = torch.randn(2, 16, 5, 6, generator=torch.Generator().manual_seed(2)).to(dev)   # channels first
    y = group_norm_act(grid.permute(0, 2, 3, 1), 4, w, b)
    assert torch.equal(y, group_norm_act(grid.permute(0, 2, 3, 1).contiguous(), 4, w, b))
    flat = torch.randn(1 + 6 * 16, generator=torch.Generator().manual_seed(3)).to(dev)
    assert torch.equal(group_norm_act(flat[1:].view(6, 16), 4, w, b), group_norm_act(flat[1:].clone().view(6, 16), 4, w, b))


def test_captured_forward(dev):
    from ssla_amd.norm import group_norm_act
    x = torch.randn(4, 700, 64, generator=torch.Generator().manual_seed(5)).to(dev)
    cur = x.clone()
    group_norm_act(cur, 8, activation="silu")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = group_norm_act(cur, 8, activation="silu")
    for i in range(4):
        cur.copy_(x * (i + 1) + i)
        graph.replay()
        want = group_norm_act(cur, 8, activation="silu")
        torch.cuda.synchronize()
        assert torch.equal(y, want)
