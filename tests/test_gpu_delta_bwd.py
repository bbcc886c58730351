"""Gradients of the chunked gated delta rule against autograd through its
definition in 64 bits, and against differences.

Tolerance, as for the forward (a contraction carries on what a token's roundings
add, now in both directions): a token's gradients are sums of at most K + V
products and of 64 rows with about 192 further operations, so after T tokens a
gradient is off by at most (K + V + 256) T half steps of fp32 (2^-24) of the
largest value, and in the root mean square by the square root of that number.  A
gate's gradient adds the 64 rows of its chunk, each as large as the gradient
itself: 64 and 8 times as much.  Gradients of 16 bits are rounded once more."""
import pytest
import torch

from oracle.delta import gated_delta
from tests.test_gpu_delta import HALF, inputs

pytestmark = pytest.mark.gpu
NAMES = ("dq", "dk", "dv", "dg", "dbeta", "dh0")


def reference(x, s0, lens, scale, do, dht):
    leaves = [t.double().requires_grad_() for t in x]
    h0 = None if s0 is None else s0.double().requires_grad_()
    o, ht = gated_delta(*leaves, lens, scale, h0)
    outs, given = ([o, ht], [do.double(), dht.double()]) if dht is not None else ([o], [do.double()])
    return torch.autograd.grad(outs, leaves + ([] if h0 is None else [h0]), given)


def gradients(dev, x, s0, cu, scale, do, dht):
    from ssla_amd.delta import chunk_gated_delta
    leaves = [t.to(dev).requires_grad_() for t in x]
    h0 = None if s0 is None else s0.to(dev).requires_grad_()
    o, ht = chunk_gated_delta(*leaves, cu.to(dev), scale=scale, initial_state=h0, output_final_state=dht is not None)
    outs, given = ([o, ht], [do.to(dev), dht.to(dev)]) if dht is not None else ([o], [do.to(dev)])
    return torch.autograd.grad(outs, leaves + ([] if h0 is None else [h0]), given)


def check(got, ref, K, V, T, dtype):
    u = 2.0 ** -24
    for name, a, r in zip(NAMES, got, ref):
        a, r = a.double().cpu(), r.cpu()
        assert a.shape == r.shape and torch.isfinite(a).all(), name
        if not r.numel():
            continue
        n, more = (K + V + 256) * T, (64, 8) if name == "dg" else (1, 1)
        half = HALF[dtype] if dtype != torch.float32 and name in ("dq", "dk", "dv") else 0.0
        big, rms, err = float(r.abs().max()), float(r.square().mean().sqrt()), (a - r).abs()
        assert bool((err <= more[0] * n * u * big + half * r.abs()).all()), f"{name}: {float(err.max()):.3g} of {big:.3g}"
        off = float(err.square().mean().sqrt())
        assert off <= more[1] * n ** 0.5 * u * max(rms, big / 8) + half * rms, f"{name}: rms {off:.3g} of {rms:.3g}"


def both(dev, lens, Hk, H, K, V, dtype, seed, h0=True, change=None, scale=None):
    x, cu, s0 = inputs(lens, Hk, H, K, V, dtype, seed, h0=h0)
    if change:
        change(*x)
    gen = torch.Generator().manual_seed(seed + 1)
    do = torch.randn(sum(lens), H, V, generator=gen).to(dtype)
    dht = torch.randn(len(lens), H, K, V, generator=gen) if h0 else None
    scale = K ** -0.5 if scale is None else scale
    check(gradients(dev, x, s0, cu, scale, do, dht), reference(x, s0, lens, scale, do, dht), K, V, max(lens), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hk,H,K,V", [(2, 2, 64, 64), (1, 2, 32, 16), (1, 3, 128, 40), (2, 4, 16, 17), (1, 1, 1, 1),
                                      (1, 1, 100, 130), (1, 2, 36, 64)])
def test_ragged(dev, dtype, Hk, H, K, V):
    for h0 in (True, False):
        both(dev, [0, 1, 63, 64, 65, 130, 7, 0], Hk, H, K, V, dtype, seed=K + V, h0=h0)


@pytest.mark.parametrize("dtype,K,V", [(torch.float32, 64, 64), (torch.bfloat16, 128, 96), (torch.float16, 32, 64),
                                       (torch.bfloat16, 64, 20)])
def test_segments(dev, dtype, K, V):
    def slow(q, k, v, g, beta):
        g /= 8
    both(dev, [700, 3, 0, 512, 256, 257, 90], 1, 2, K, V, dtype, seed=3, change=slow)


@pytest.mark.parametrize("kind", ["equal keys", "no decay", "strong", "resets", "beta 0", "beta 1", "scale 0"])
def test_regimes(dev, kind):
    def change(q, k, v, g, beta):
        if kind == "equal keys":
            k[:] = k[:1]
            g[:] = 0
            beta[:] = 1
        elif kind == "no decay":
            g[:] = 0
        elif kind == "strong":
            g[:] = -30 * torch.rand(g.shape, generator=torch.Generator().manual_seed(1))
        elif kind == "resets":
            # (autograd of exp gives 0 at a gate of -150 as at -inf, where it would meet 0 inf)
            g[torch.rand(g.shape, generator=torch.Generator().manual_seed(2)) < 0.1] = -150.0
        elif kind.startswith("beta"):
            beta[:] = float(kind[-1])
    both(dev, [200, 70], 1, 2, 64, 32, torch.float32, seed=8, change=change, scale=0.0 if kind == "scale 0" else 0.5)


def test_gates_of_minus_infinity(dev):
    """They give the gradients of a very strong gate, bit for bit."""
    x, cu, s0 = inputs([150], 1, 2, 32, 32, torch.float32, seed=5)
    do, dht = torch.randn(150, 2, 32), torch.randn(1, 2, 32, 32)
    x[3][[0, 40, 100]] = -torch.inf
    got = gradients(dev, x, s0, cu, 1.0, do, dht)
    x[3][[0, 40, 100]] = -1e30
    assert all(torch.equal(a, b) for a, b in zip(got, gradients(dev, x, s0, cu, 1.0, do, dht)))
    assert all(torch.isfinite(t).all() for t in got)


def test_long_batches_are_their_sequences(dev):
    """Sequences packed with others and cut into segments of another length have
    the gradients of the sequence alone (up to the order of sums); rows in no
    sequence get zeros."""
    lens = [4096, 1000, 3, 2049]
    x, cu, s0 = inputs(lens, 2, 4, 64, 64, torch.float32, seed=6)
    x[3] /= 16
    gen = torch.Generator().manual_seed(7)
    pad = 5
    x = [torch.cat([torch.randn(pad, *t.shape[1:], generator=gen), t, torch.randn(9, *t.shape[1:], generator=gen)]) for t in x]
    do, dht = torch.randn(sum(lens) + 14, 4, 64, generator=gen), torch.randn(4, 4, 64, 64, generator=gen)
    whole = gradients(dev, x, s0, cu + pad, 0.125, do, dht)
    for t in whole[:5]:
        assert not t[:pad].any() and not t[-9:].any()
    for n, rows in enumerate(lens):
        a = pad + sum(lens[:n])
        alone = gradients(dev, [t[a:a + rows] for t in x], s0[n:n + 1], torch.tensor([0, rows]), 0.125, do[a:a + rows],
                          dht[n:n + 1])
        got = [t[a:a + rows] for t in whole[:5]] + [whole[5][n:n + 1]]
        check(got, [t.double() for t in alone], 64, 64, rows, torch.float32)


def test_differences(dev):
    """The slope along a direction of all inputs against central differences of
    the fp32 forward, whose two step sizes bound what they leave out."""
    from ssla_amd.delta import chunk_gated_delta
    lens = [150, 33]
    x, cu, s0 = inputs(lens, 1, 2, 32, 32, torch.float32, seed=11)
    gen = torch.Generator().manual_seed(12)
    d = [torch.randn(t.shape, generator=gen) * (0.1 if i < 3 else 0.02) for i, t in enumerate((*x, s0))]
    do, dht = torch.randn(183, 2, 32, generator=gen), torch.randn(2, 2, 32, 32, generator=gen)
    grads = gradients(dev, x, s0, cu, 1.0, do, dht)
    slope = sum(float((g.double().cpu() * e).sum()) for g, e in zip(grads, d))

    def loss(h):
        y = [(t + h * e).to(dev) for t, e in zip((*x, s0), d)]
        o, ht = chunk_gated_delta(*y[:5], cu.to(dev), scale=1.0, initial_state=y[5], output_final_state=True)
        return float((o.double().cpu() * do).sum() + (ht.double().cpu() * dht).sum())

    h = 2.0 ** -5
    two = [(loss(h) - loss(-h)) / (2 * h), (loss(2 * h) - loss(-2 * h)) / (4 * h)]
    diff = (4 * two[0] - two[1]) / 3
    # 11,712 + 4,096 outputs, each off by at most (32 + 256) 150 2^-24 in the worst case and by its root in the mean
    noise = (15808 * 288 * 150) ** 0.5 * 2.0 ** -24 * 4 / h
    assert abs(diff - slope) <= abs(two[0] - two[1]) + noise, (diff, slope, two)


def test_gradients_through_casts_and_unused_outputs(dev):
    """16-bit gates and weights get 16-bit gradients; a final state alone, or a
    loss that leaves it out, has its gradient; no second derivative; keys wider
    than the chunk kernels take are refused under autograd."""
    from ssla_amd.delta import chunk_gated_delta
    x, cu, s0 = inputs([70], 1, 2, 32, 16, torch.bfloat16, seed=13)
    x[3], x[4] = x[3].bfloat16(), x[4].bfloat16()
    ref = reference(x, s0, [70], 32 ** -0.5, torch.zeros(70, 2, 16), torch.ones(1, 2, 32, 16))
    leaves = [t.to(dev).requires_grad_() for t in (*x, s0)]
    o, ht = chunk_gated_delta(*leaves[:5], cu.to(dev), initial_state=leaves[5], output_final_state=True)
    got = torch.autograd.grad(ht.sum(), leaves, retain_graph=True, allow_unused=True)
    for name, a, r, t in zip(NAMES, got, ref, leaves):
        assert a.dtype == t.dtype
        tol = HALF[a.dtype] * r.abs() + (32 + 16 + 256) * 70 * 2.0 ** -24 * max(float(r.abs().max()), 1e-3) * 64
        assert bool(((a.double().cpu() - r).abs() <= tol).all()), name
    only = torch.autograd.grad(o.float().sum(), leaves)
    assert all(torch.isfinite(t).all() for t in only)
    with pytest.raises(RuntimeError):
        o, _ = chunk_gated_delta(*leaves[:5], cu.to(dev))
        g1 = torch.autograd.grad(o.float().sum(), leaves[:5], create_graph=True)
        torch.autograd.grad(sum(t.float().sum() for t in g1), leaves[:5])
    x, cu, _ = inputs([4], 1, 1, 130, 8, torch.float32, seed=14)
    with pytest.raises(NotImplementedError):
        chunk_gated_delta(*(t.to(dev).requires_grad_() for t in x), cu.to(dev))
    y = [t[:0].to(dev).requires_grad_() for t in inputs([1], 1, 2, 32, 16, torch.float32, seed=15)[0]]
    h0 = torch.ones(2, 2, 32, 16, device=dev, requires_grad=True)
    o, ht = chunk_gated_delta(*y, torch.zeros(3, dtype=torch.int64, device=dev), initial_state=h0, output_final_state=True)
    (dh0,) = torch.autograd.grad(ht.sum(), h0)
    assert o.shape == (0, 2, 16) and bool((dh0 == 1).all())
    y = [t.to(dev).requires_grad_() for t in inputs([3], 1, 2, 32, 16, torch.float32, seed=15)[0]]
    o, _ = chunk_gated_delta(*y, torch.zeros(1, dtype=torch.int64, device=dev))   # rows, but no sequence
    assert not any(t.any() for t in torch.autograd.grad(o, y, torch.ones_like(o)))


def test_same_bits_every_time(dev):
    x, cu, s0 = inputs([900, 300, 70], 1, 4, 64, 64, torch.bfloat16, seed=16)
    do, dht = torch.randn(1270, 4, 64).bfloat16(), torch.randn(3, 4, 64, 64)
    first = gradients(dev, x, s0, cu, 0.125, do, dht)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, gradients(dev, x, s0, cu, 0.125, do, dht)))


def test_training_step_in_a_graph(dev):
    """Forward and backward of the rule and of the head-wise norm behind it,
    captured once and replayed on changing inputs with eager steps in between:
    every replay equals its eager step."""
    from ssla_amd.delta import chunk_gated_delta
    from ssla_amd.norm import group_norm_act
    x, cu, s0 = inputs([500, 90], 1, 2, 64, 32, torch.bfloat16, seed=17)
    cu, do = cu.to(dev), torch.randn(590, 64).bfloat16().to(dev)

    def step(leaves):
        o, ht = chunk_gated_delta(*leaves[:5], cu, initial_state=leaves[5], output_final_state=True)
        y = group_norm_act(o.flatten(1), 2, activation="silu")
        return y, *torch.autograd.grad((y, ht.sum()), leaves, (do, torch.ones((), device=dev)))

    static = [t.to(dev).requires_grad_() for t in (*x, s0)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(static)
    for i in range(4):
        with torch.no_grad():
            static[2].copy_(x[2] * (1 + i))
            static[5].copy_(s0 * (1 - i))
        graph.replay()
        want = step([t.detach().clone().requires_grad_() for t in static])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


@pytest.mark.parametrize("dtype,K,V", [(torch.bfloat16, 64, 64), (torch.float32, 24, 40)])
def test_long_among_many_short(dev, dtype, K, V):
    def slow(q, k, v, g, beta):
        g.div_(8)
    both(dev, [5, 0, 3, 800, 2, 1, 0, 7, 1100] + [1, 0, 2] * 8 + [513, 9, 300], 1, 2, K, V, dtype, seed=K, change=slow)
