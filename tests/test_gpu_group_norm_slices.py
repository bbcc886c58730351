"""Group norm on the samples that take every path of the slices: one, a few (joined
by the second pass), more than 64 (joined by a kernel of their own), groups that
span blocks of channels, single-value vectors; and small samples of many positions.

Bound: the root mean square of the error may be that of runs in 64 bits with a
model of fp32's roundings in them (tests/norm_form.py), plus half a step of a 16-bit
result.  test_norm_form shows on the CPU that lost slices, lost terms of the joins
and lost sums all pass these bounds.  The values drift along the positions, so that
slices have means of their own, dy goes with x^ and with its sign, so that the
backward's means are large, and dy is 0 where relu's border is near."""
import pytest
import torch

from tests import norm_form as form

HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
EPS = 1e-5
# N, L, C, G and which path fp32 takes
SLICES = [(2, 18240, 64, 8),    # 143 slices a sample, vectors of 4
          (1, 20000, 30, 6),    # 79 slices, single values (5 channels a group)
          (2, 500, 1200, 8),    # 16 x 5 slices, groups of 150 that span blocks of 256
          (3, 300, 2048, 2),    # 38 x 2 slices, groups of whole blocks
          (2, 4560, 64, 8),     # 36 slices
          (1, 700, 96, 3),      # a few slices
          (5, 90, 128, 1)]      # two slices
LANES = [(300, 40, 16, 2), (2000, 9, 24, 3), (64, 512, 4, 1), (700, 1, 512, 8), (1, 16, 64, 1)]   # groups of a wavefront


def inputs(shape, G, dtype, act, seed=0):
    N, L, C = shape
    gen = torch.Generator().manual_seed(seed + L + C)

    def randn(*s):
        return torch.randn(*s, generator=gen)

    drift = torch.linspace(-1, 1, L)[:, None] if L > 1 else torch.zeros(1, 1)
    x = (1.5 * randn(N, L, C) + randn(C) + 2 * drift).to(dtype)
    w, b = 1 + 0.3 * randn(C), 0.3 * randn(C)
    y = form.run(x, G, w, b, EPS, None, torch.zeros(N, L, C))[0]
    xh = (y - b) / w
    dy = randn(N, L, C) + 0.5 + 0.5 * xh
    if act == "relu":
        dy = torch.where(y.abs() < 1e-3, 0.0, dy)
    return x, w, b, dy.to(dtype)


def rms(t):
    return float(t.square().mean().sqrt())


def bounds(x, G, w, b, act, dy):
    """Results in 64 bits, and how far each may be off (root mean square)."""
    ref = form.run(x, G, w, b, EPS, act, dy)
    noisy = [form.run(x, G, w, b, EPS, act, dy, form.roundings(seed)) for seed in range(2)]
    return ref, [(sum(rms(n[i] - r) ** 2 for n in noisy) / len(noisy)) ** 0.5 for i, r in enumerate(ref)]


def compare(dev, shape, G, dtype, act):
    from ssla_amd.norm import group_norm_act
    x, w, b, dy = inputs(shape, G, dtype, act)
    ref, tol = bounds(x, G, w, b, act, dy)
    leaves = [t.to(dev).requires_grad_() for t in (x, w, b)]
    y = group_norm_act(leaves[0], G, *leaves[1:], eps=EPS, activation=act)
    got = (y.detach(), *torch.autograd.grad(y, leaves, dy.to(dev)))
    with torch.no_grad():   # (keeps no statistics: the joined moments lie in the workspace)
        alone = group_norm_act(leaves[0], G, *leaves[1:], eps=EPS, activation=act)
    assert torch.equal(alone, got[0])
    for i, name in ((1, "dx"), (2, "dw"), (3, "db")):   # one gradient wanted
        only = leaves[i - 1]
        args = [t if t is only else t.detach() for t in leaves]
        (g,) = torch.autograd.grad(group_norm_act(args[0], G, *args[1:], eps=EPS, activation=act), only, dy.to(dev))
        assert torch.equal(g, got[i]), name
    for name, a, r, t in zip(("y", "dx", "dw", "db"), got, ref, tol):
        half = HALF[a.dtype] * rms(r)
        off = rms(a.double().cpu() - r)
        assert off <= t + half, f"{name}: {off:.3g}, bound {t + half:.3g}, of {rms(r):.3g}"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", [None, "relu", "silu"])
@pytest.mark.parametrize("shape", SLICES)
def test_slices(dev, shape, act, dtype):
    compare(dev, shape[:3], shape[3], dtype, act)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", [None, "relu", "silu"])
@pytest.mark.parametrize("shape", LANES)
def test_lanes(dev, shape, act, dtype):
    compare(dev, shape[:3], shape[3], dtype, act)


@pytest.mark.gpu
def test_many_slices_in_a_graph(dev):
    """Forward and backward through the join kernels, captured once and replayed on
    changing inputs with eager steps in between."""
    from ssla_amd.norm import group_norm_act
    x, w, b, dy = (t.to(dev) for t in inputs((2, 18240, 64), 8, torch.float32, "silu"))
    static = [t.clone().requires_grad_() for t in (x, w, b)]

    def step(leaves):
        y = group_norm_act(leaves[0], 8, *leaves[1:], activation="silu")
        return y.detach(), *torch.autograd.grad(y, leaves, dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(static)
    for i in range(4):
        with torch.no_grad():
            static[0].copy_(x * (1 + i) + i)
        graph.replay()
        want = step([t.detach().clone().requires_grad_() for t in static])
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(got, want)), i
