"""The gated delta rule token by token against its definition in 64 bits.

Tolerance: with |k| = 1, 0 <= beta <= 1 and g <= 0 the state's map is a
contraction, so what a token's roundings add to a state stays at most that
large.  A token rounds each of its sums of K terms and about 16 more operations
once, each by at most half a step of fp32 (2^-24) of the values in them, so
after T tokens a state or output is off by at most (K + 16) T 2^-24 of the
largest value, and an output by half a step of its own type more."""
import pytest
import torch
import torch.nn.functional as F

from oracle.delta import gated_delta

pytestmark = pytest.mark.gpu
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def inputs(lens, Hk, H, K, V, dtype, seed, h0=True):
    gen = torch.Generator().manual_seed(seed)
    T = sum(lens)
    q, k = (F.normalize(torch.randn(T, Hk, K, generator=gen), dim=-1).to(dtype) for _ in range(2))
    v = torch.randn(T, H, V, generator=gen).to(dtype)
    g = F.logsigmoid(torch.randn(T, H, generator=gen) + 1)
    beta = torch.sigmoid(2 * torch.randn(T, H, generator=gen))
    s0 = 0.5 * torch.randn(len(lens), H, K, V, generator=gen) if h0 else None
    cu = torch.tensor([0] + lens).cumsum(0)
    return [q, k, v, g, beta], cu, s0


def close(a, ref, K, T, dtype, name):
    big = float(ref.abs().max()) if ref.numel() else 0.0
    err = (a.double().cpu() - ref).abs()
    tol = (K + 16) * max(T, 1) * 2.0 ** -24 * big + HALF[dtype] * ref.abs()
    assert a.shape == ref.shape and torch.isfinite(a).all(), name
    assert bool((err <= tol).all()), f"{name}: off by {float(err.max()):.3g}, largest value {big:.3g}"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hk,H,K,V", [(2, 2, 32, 32), (1, 3, 16, 16), (2, 4, 64, 40), (1, 1, 1, 1), (1, 2, 100, 17),
                                      (2, 2, 128, 64), (1, 2, 256, 20), (1, 1, 200, 130)])
def test_recurrent(dev, dtype, Hk, H, K, V):
    from ssla_amd.delta import fused_recurrent_gated_delta
    lens = [0, 1, 2, 17, 40, 0]
    for h0 in (True, False):
        x, cu, s0 = inputs(lens, Hk, H, K, V, dtype, seed=K + V, h0=h0)
        o, ht = fused_recurrent_gated_delta(*(t.to(dev) for t in x), cu.to(dev),
                                            initial_state=None if s0 is None else s0.to(dev), output_final_state=True)
        ro, rs = gated_delta(*x, lens, K ** -0.5, s0)
        assert o.dtype == dtype and ht.dtype == torch.float32
        close(o, ro, K, max(lens), dtype, "o")
        close(ht, rs, K, max(lens), torch.float32, "ht")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("Hk,H,K,V", [(2, 2, 16, 32), (1, 2, 32, 24), (2, 2, 64, 40), (1, 2, 100, 17), (2, 2, 256, 32)])
def test_many_sequences(dev, dtype, Hk, H, K, V):
    """Batches with more than a wavefront of 16 columns for each SIMD (the small
    ones run 8 columns a wavefront)."""
    from ssla_amd.delta import fused_recurrent_gated_delta
    lens = [(7 * n) % 5 for n in range(300)]
    x, cu, s0 = inputs(lens, Hk, H, K, V, dtype, seed=K)
    o, ht = fused_recurrent_gated_delta(*(t.to(dev) for t in x), cu.to(dev), initial_state=s0.to(dev),
                                        output_final_state=True)
    ro, rs = gated_delta(*x, lens, K ** -0.5, s0)
    close(o, ro, K, 4, dtype, "o")
    close(ht, rs, K, 4, torch.float32, "ht")


def test_recurrent_edges_of_the_gates(dev):
    """Gates of -inf and 0, writes of weight 0 and 1, 16-bit gates, strided
    inputs, offsets on the host and a scale of its own."""
    from ssla_amd.delta import fused_recurrent_gated_delta
    lens = [30, 7]
    (q, k, v, g, beta), cu, s0 = inputs(lens, 2, 2, 32, 24, torch.float32, seed=5)
    g[3], g[20], g[31] = -torch.inf, 0.0, -200.0
    beta[4], beta[5] = 0.0, 1.0
    g, beta = g.bfloat16(), beta.bfloat16()
    ro, rs = gated_delta(q, k, v, g, beta, lens, 0.7, s0)
    wide = torch.stack([q, k], 1).to(dev)
    o, ht = fused_recurrent_gated_delta(wide[:, 0], wide[:, 1], v.to(dev).transpose(1, 2).contiguous().transpose(1, 2),
                                        g.to(dev), beta.to(dev), cu, scale=0.7, initial_state=s0.to(dev),
                                        output_final_state=True)
    close(o, ro, 32, 30, torch.float32, "o")
    close(ht, rs, 32, 30, torch.float32, "ht")


def test_rows_outside_and_nonfinite_rows(dev):
    """Rows in no sequence are not written; a row that is not finite leaves the
    rows before it, its sequence's other columns and the other sequences bit
    for bit as they are."""
    from ssla_amd import _lib
    from ssla_amd.delta import fused_recurrent_gated_delta
    (q, k, v, g, beta), _, _ = inputs([50], 1, 2, 16, 16, torch.float32, seed=6)
    x = [t.to(dev) for t in (q, k, v, g, beta)]
    cu = torch.tensor([3, 20, 20, 41], device=dev)
    o = torch.full((50, 2, 16), 7.0, device=dev)
    P = _lib.ptr
    _lib.check(_lib.load().ssla_gated_delta_recurrent(*(P(t) for t in x), P(cu), 3, 50, 1, 2, 16, 16, 1.0, None, P(o),
                                                      None, None, 0, None, _lib.SSLA_F32, _lib.stream_of(o)), "rec")
    assert bool((o[:3] == 7).all()) and bool((o[41:] == 7).all()) and not bool((o[3:41] == 7).any())
    clean, _ = fused_recurrent_gated_delta(*x, cu, scale=1.0)
    assert torch.equal(clean[3:41], o[3:41])
    bad = [t.clone() for t in x]
    bad[2][10, 1, 4] = torch.inf
    got, _ = fused_recurrent_gated_delta(*bad, cu, scale=1.0)
    hit = torch.zeros(50, 2, 16, dtype=torch.bool, device=dev)
    hit[10:20, 1, 4] = True
    assert torch.equal(got[3:41][~hit[3:41]], clean[3:41][~hit[3:41]]) and not torch.isfinite(got[hit]).any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K,V", [(32, 32), (64, 128), (20, 24)])
def test_sites_and_steps(dev, dtype, K, V):
    """A scan over histories equals its tokens run as steps and the definition;
    sites that are not named keep their states bit for bit."""
    from ssla_amd.delta import sparse_delta_scan, sparse_delta_step
    lens, sites = [3, 1, 0, 6], [1, 2, 5, 8]
    (q, k, v, g, beta), cu, _ = inputs(lens, 1, 2, K, V, dtype, seed=K, h0=False)
    table = torch.randn(10, 2, K, V, generator=torch.Generator().manual_seed(1))
    x = [t.to(dev) for t in (q, k, v, g, beta)]
    s1, s2 = table.to(dev), table.to(dev)
    at = torch.tensor(sites, device=dev)
    o = sparse_delta_scan(*x, cu.to(dev), at, s1, check=True)
    ro, rs = gated_delta(q, k, v, g, beta, lens, K ** -0.5, table[sites])
    close(o, ro, K, 6, dtype, "o")
    close(s1[at], rs, K, 6, torch.float32, "state")
    rest = [i for i in range(10) if i not in sites]
    assert torch.equal(s1[rest].cpu(), table[rest]) and torch.equal(s1[5].cpu(), table[5])
    steps = torch.empty_like(o)
    for t in range(max(lens)):
        on = [n for n in range(4) if t < lens[n]]
        rows = torch.tensor([int(cu[n]) + t for n in on], device=dev)
        steps[rows] = sparse_delta_step(torch.tensor([sites[n] for n in on], device=dev), *(a[rows] for a in x), s2,
                                        check=True)
    close(steps, ro, K, 6, dtype, "steps")
    close(s2[at], rs, K, 6, torch.float32, "state of steps")
    assert torch.equal(s2[rest].cpu(), table[rest])


def test_bad_site_lists(dev):
    from ssla_amd.delta import sparse_delta_scan, sparse_delta_step
    (q, k, v, g, beta), _, _ = inputs([4], 2, 2, 16, 16, torch.float32, seed=9)
    x = [t.to(dev) for t in (q, k, v, g, beta)]
    table = torch.randn(6, 2, 16, 16, generator=torch.Generator().manual_seed(2)).to(dev)
    for bad, skipped in (([0, 2, 2, 5], [2]), ([-1, 0, 1, 2], [0]), ([0, 1, 2, 6], [3]), ([3, 1, 4, 5], [1]),
                         ([0, 1, 2, 1 << 40], [3])):
        at = torch.tensor(bad, device=dev)
        for form in (lambda s, **a: sparse_delta_step(at, *x, s, **a),
                     lambda s, **a: sparse_delta_scan(*x, torch.arange(5, device=dev), at, s, **a)):
            with pytest.raises(ValueError, match="strictly increasing"):
                form(table.clone(), check=True)
            s = table.clone()
            o = form(s)
            named = [b for i, b in enumerate(bad) if i not in skipped]
            rest = [i for i in range(6) if i not in named]
            assert not o[skipped].any() and torch.equal(s[rest], table[rest])
            assert bool((s[named] != table[named]).flatten(1).any(1).all())
    s = table.clone()
    empty = [t[:0] for t in x]
    assert sparse_delta_step(torch.zeros(0, dtype=torch.int32, device=dev), *empty, s).shape == (0, 2, 16)
    assert torch.equal(s, table)
    with pytest.raises(NotImplementedError):
        sparse_delta_step(torch.arange(4, device=dev), x[0].requires_grad_(), *x[1:], s)


def test_step_in_a_graph_and_on_a_stream(dev):
    """A captured step replayed on changing inputs equals eager steps, every
    time; a step on another stream equals them too."""
    from ssla_amd.delta import sparse_delta_step
    (q, k, v, g, beta), _, _ = inputs([40], 1, 2, 32, 32, torch.float32, seed=11)
    x = [t.to(dev) for t in (q, k, v, g, beta)]
    at = torch.tensor([0, 3, 4, 9], dtype=torch.int32, device=dev)
    cur = [t[:4].clone() for t in x]
    state = torch.randn(10, 2, 32, 32, generator=torch.Generator().manual_seed(3)).to(dev)
    eager = state.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = state.clone()
        first = sparse_delta_step(at, *cur, other)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, sparse_delta_step(at, *cur, state.clone()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sparse_delta_step(at, *cur, state)
    for t in range(6):
        for c, a in zip(cur, x):
            c.copy_(a[4 * t:4 * t + 4])
        graph.replay()
        want = sparse_delta_step(at, *cur, eager)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(state, eager)


@pytest.mark.parametrize("dtype", [torch.int64, torch.int16, torch.uint8])
def test_site_lists_of_other_integers(dev, dtype):
    """Site lists of any integer type name the same sites as 32-bit ones."""
    from ssla_amd.delta import sparse_delta_scan, sparse_delta_step
    (q, k, v, g, beta), cu, _ = inputs([3, 0, 5], 1, 2, 16, 20, torch.float32, seed=21)
    x = [t.to(dev) for t in (q, k, v, g, beta)]
    state = torch.randn(6, 2, 16, 20, generator=torch.Generator().manual_seed(4)).to(dev)
    at = torch.tensor([0, 2, 5], device=dev)
    outs = []
    for t in (torch.int32, dtype):
        s = state.clone()
        o = sparse_delta_scan(*x, cu.to(dev), at.to(t), s, check=True)
        outs.append((o, sparse_delta_step(at.to(t), *(a[:3] for a in x), s, check=True), s))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    assert not torch.equal(outs[0][2], state)
