"""The chunked gated delta rule against its definition in 64 bits, and on long
batches against the token-by-token kernel.

Tolerance: with |k| = 1, 0 <= beta <= 1 and g <= 0 the state's map is a
contraction, so what a token's roundings add to the state stays at most that
large.  A token's u is a sum of 64 values (its row of Tm), each a sum of K
products, Tm's own entries are sums of 64, and about 64 more operations round
once: at most K + 256 half steps of fp32 (2^-24) a token, of the largest value.
That bounds every value linearly in the tokens T; the roundings do not know of
each other, so their root mean square grows with sqrt((K + 256) T), which is the
second bound.  Outputs of 16 bits are rounded once more (half a step)."""
import pytest
import torch

from oracle.delta import gated_delta
from tests.test_gpu_delta import HALF, inputs

pytestmark = pytest.mark.gpu


def close(a, ref, K, T, dtype, name):
    a, ref = a.double().cpu(), ref.double().cpu()
    assert a.shape == ref.shape and torch.isfinite(a).all(), name
    if not ref.numel():
        return
    big, rms = float(ref.abs().max()), float(ref.square().mean().sqrt())
    err, u, n = (a - ref).abs(), 2.0 ** -24, (K + 256) * max(T, 1)
    half = 0.0 if dtype == torch.float32 else HALF[dtype]
    assert bool((err <= n * u * big + half * ref.abs()).all()), f"{name}: off by {float(err.max()):.3g} of {big:.3g}"
    got = float(err.square().mean().sqrt())
    assert got <= n ** 0.5 * u * max(rms, big / 8) + half * rms, f"{name}: rms {got:.3g} of {rms:.3g}"


def run(dev, x, cu, s0, **kw):
    from ssla_amd.delta import chunk_gated_delta
    return chunk_gated_delta(*(t.to(dev) for t in x), cu.to(dev), initial_state=None if s0 is None else s0.to(dev),
                             output_final_state=True, **kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hk,H,K,V", [(2, 2, 64, 64), (1, 2, 32, 16), (1, 3, 128, 40), (2, 4, 16, 17), (1, 1, 1, 1),
                                      (1, 1, 100, 130), (1, 2, 36, 64)])
def test_ragged(dev, dtype, Hk, H, K, V):
    """Sequences that are empty, of one row, one less, as many and one more than
    a chunk, and longer; with and without an initial state."""
    lens = [0, 1, 63, 64, 65, 130, 7, 0]
    for h0 in (True, False):
        x, cu, s0 = inputs(lens, Hk, H, K, V, dtype, seed=K + V, h0=h0)
        o, ht = run(dev, x, cu, s0)
        ro, rs = gated_delta(*x, lens, K ** -0.5, s0)
        assert o.dtype == dtype and ht.dtype == torch.float32
        close(o, ro, K, max(lens), dtype, "o")
        close(ht, rs, K, max(lens), torch.float32, "ht")


@pytest.mark.parametrize("dtype,K,V", [(torch.float32, 64, 64), (torch.bfloat16, 128, 96), (torch.float16, 32, 64),
                                       (torch.bfloat16, 64, 20)])
def test_segments(dev, dtype, K, V):
    """Sequences longer than a segment, one of whole segments, and short ones
    between them."""
    lens = [700, 3, 0, 512, 256, 257, 90]
    x, cu, s0 = inputs(lens, 1, 2, K, V, dtype, seed=3)
    x[3] = x[3] / 8   # a memory of many chunks
    o, ht = run(dev, x, cu, s0)
    ro, rs = gated_delta(*x, lens, K ** -0.5, s0)
    close(o, ro, K, max(lens), dtype, "o")
    close(ht, rs, K, max(lens), torch.float32, "ht")


@pytest.mark.parametrize("dtype,Hk,H,K,V,lens", [
    (torch.bfloat16, 8, 8, 64, 64, [4096] * 8), (torch.float32, 2, 4, 64, 64, [9000, 17, 4000, 0, 1283]),
    (torch.bfloat16, 2, 4, 128, 128, [5000, 11000]), (torch.float16, 1, 1, 32, 32, [30000]),
    (torch.bfloat16, 2, 2, 64, 64, [40] * 700)])
def test_long_batches(dev, dtype, Hk, H, K, V, lens):
    from ssla_amd.delta import fused_recurrent_gated_delta
    x, cu, s0 = inputs(lens, Hk, H, K, V, torch.float32, seed=4)
    x[3] = x[3] / 16
    x = [t.to(dtype) if i < 3 else t for i, t in enumerate(x)]
    o, ht = run(dev, x, cu, s0)
    x = [t.float() if i < 3 else t for i, t in enumerate(x)]
    ro, rs = fused_recurrent_gated_delta(*(t.to(dev) for t in x), cu.to(dev), initial_state=s0.to(dev),
                                         output_final_state=True)
    close(o, ro, K, max(lens), dtype, "o")
    close(ht, rs, K, max(lens), torch.float32, "ht")


@pytest.mark.parametrize("kind", ["equal keys", "no decay", "strong", "resets", "beta 0", "beta 1"])
def test_regimes(dev, kind):
    """Where a chunk's system is hardest: equal keys written with full weight (A
    is all ones), no decay, decays of e^-30 a token, gates of -inf, weights of 0
    and 1."""
    lens = [200, 70]
    x, cu, s0 = inputs(lens, 1, 2, 64, 32, torch.float32, seed=8)
    q, k, v, g, beta = x
    if kind == "equal keys":
        k[:] = k[:1]
        g[:] = 0
        beta[:] = 1
    elif kind == "no decay":
        g[:] = 0
    elif kind == "strong":
        g[:] = -30 * torch.rand(g.shape, generator=torch.Generator().manual_seed(1))
    elif kind == "resets":
        g[torch.rand(g.shape, generator=torch.Generator().manual_seed(2)) < 0.1] = -torch.inf
    else:
        beta[:] = float(kind[-1])
    o, ht = run(dev, x, cu, s0, scale=0.5)
    ro, rs = gated_delta(*x, lens, 0.5, s0)
    close(o, ro, 64, 200, torch.float32, "o")
    close(ht, rs, 64, 200, torch.float32, "ht")


def test_layouts(dev):
    """Strided inputs, views that start off 16 bytes, offsets on the host, 16-bit
    gates and weights, rows in no sequence."""
    from ssla_amd import _lib
    from ssla_amd.delta import chunk_gated_delta
    for dtype in (torch.float32, torch.bfloat16):
        (q, k, v, g, beta), _, _ = inputs([150], 1, 2, 32, 16, dtype, seed=9)
        g, beta = g.bfloat16(), beta.bfloat16()
        ro, _ = gated_delta(q[5:140], k[5:140], v[5:140], g[5:140], beta[5:140], [135], 1.0)
        both = torch.cat([q, k], -1).to(dev)
        flat = torch.empty(1 + k.numel(), dtype=dtype, device=dev)
        flat[1:] = k.to(dev).flatten()
        o, _ = chunk_gated_delta(both[..., :32], flat[1:].view_as(k), v.to(dev), g.to(dev), beta.to(dev),
                                 torch.tensor([5, 140]), scale=1.0)
        close(o[5:140], ro, 32, 135, dtype, "o")
    x = [t.to(dev) for t in (q.float(), k.float(), v.float(), g.float(), beta.float())]
    cu = torch.tensor([5, 140], device=dev)
    o = torch.full((150, 2, 16), 7.0, device=dev)
    P, lib = _lib.ptr, _lib.load()
    ws = torch.empty(lib.ssla_gated_delta_chunk_workspace_size(1, 150, 2, 32, 16), dtype=torch.uint8, device=dev)
    _lib.check(lib.ssla_gated_delta_chunk_fwd(*(P(t) for t in x), P(cu), 1, 150, 1, 2, 32, 16, 1.0, None, P(o), None, None,
                                              0, P(ws), ws.numel(), _lib.stream_of(o)), "chunk")
    assert bool((o[:5] == 7).all()) and bool((o[140:] == 7).all()) and not bool((o[5:140] == 7).any())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("row", [3, 64, 100, 299])
def test_nonfinite_rows_stay_causal(dev, dtype, row):
    """A value that is not finite changes no earlier row, no other head or
    sequence, and in v no other column, bit for bit; what it reaches is not
    finite either.  q reaches its own row only."""
    x, cu, s0 = inputs([300, 80], 2, 2, 64, 32, dtype, seed=10)
    clean_o, clean_s = run(dev, x, cu, s0)
    for which, value in ((0, torch.nan), (1, torch.inf), (1, torch.nan), (2, -torch.inf), (3, torch.nan),
                         (3, torch.inf), (4, torch.inf)):
        bad = [t.clone() for t in x]
        bad[which][(row, 1, 5) if which < 3 else (row, 1)] = value
        o, ht = run(dev, bad, cu, s0)
        hit = torch.zeros_like(o, dtype=torch.bool)
        state = torch.zeros_like(ht, dtype=torch.bool)
        if which == 0:
            hit[row, 1] = True
        elif which == 2:
            hit[row:300, 1, 5] = True
            state[0, 1, :, 5] = True
        else:
            hit[row:300, 1] = True
            state[0, 1] = True
        assert torch.equal(o[~hit], clean_o[~hit]) and torch.equal(ht[~state], clean_s[~state]), (which, value)
        assert not torch.isfinite(o[hit]).any() and not torch.isfinite(ht[state]).any(), (which, value)
    s0[0, 1, 3, 7] = torch.inf
    o, ht = run(dev, x, cu, s0)
    assert not torch.isfinite(o[:300, 1, 7]).any() and torch.equal(o[300:], clean_o[300:])
    assert torch.equal(o[:, :, 8:], clean_o[:, :, 8:]) and torch.equal(ht[..., :7], clean_s[..., :7])


def test_empty_batches(dev):
    from ssla_amd.delta import chunk_gated_delta
    x, _, _ = inputs([1], 1, 2, 32, 16, torch.float32, seed=1)
    none = [t[:0].to(dev) for t in x]
    s0 = torch.randn(3, 2, 32, 16, generator=torch.Generator().manual_seed(1)).to(dev)
    o, ht = chunk_gated_delta(*none, torch.zeros(4, dtype=torch.int64, device=dev), initial_state=s0,
                              output_final_state=True)
    assert o.shape == (0, 2, 16) and torch.equal(ht, s0)
    o, ht = chunk_gated_delta(*none, torch.zeros(1, dtype=torch.int64, device=dev), output_final_state=True)
    assert ht.shape == (0, 2, 32, 16)
    o, ht = chunk_gated_delta(*(t.to(dev) for t in x), torch.tensor([0, 0, 1, 1], device=dev), output_final_state=True)
    assert not ht[0].any() and not ht[2].any() and ht[1].any()


def test_two_streams_and_a_graph(dev):
    """Calls in flight on two streams at once, and a captured call replayed on
    changing inputs, give what a call alone gives."""
    from ssla_amd.delta import chunk_gated_delta
    x, cu, s0 = inputs([900, 300], 1, 2, 64, 64, torch.bfloat16, seed=12)
    y, cy, _ = inputs([100] * 9, 1, 2, 64, 64, torch.bfloat16, seed=13)
    x, y, cu, cy, s0 = [t.to(dev) for t in x], [t.to(dev) for t in y], cu.to(dev), cy.to(dev), s0.to(dev)
    want, other = chunk_gated_delta(*x, cu, initial_state=s0)[0], chunk_gated_delta(*y, cy)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(4):
        got.append(chunk_gated_delta(*x, cu, initial_state=s0)[0])
        with torch.cuda.stream(side):
            mine = chunk_gated_delta(*y, cy)[0]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in got) and torch.equal(mine, other)
    cur = [t.clone() for t in x]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, ht = chunk_gated_delta(*cur, cu, initial_state=s0, output_final_state=True)
    for i in range(4):
        cur[2].copy_(x[2] * (i + 1))
        graph.replay()
        eo, eh = chunk_gated_delta(*cur, cu, initial_state=s0, output_final_state=True)
        torch.cuda.synchronize()
        assert torch.equal(o, eo) and torch.equal(ht, eh)


def test_wide_keys_run_token_by_token(dev):
    from ssla_amd.delta import chunk_gated_delta
    x, cu, s0 = inputs([20, 3], 1, 1, 160, 24, torch.float32, seed=14)
    o, ht = run(dev, x, cu, s0)
    ro, rs = gated_delta(*x, [20, 3], 160 ** -0.5, s0)
    close(o, ro, 160, 20, torch.float32, "o")
    close(ht, rs, 160, 20, torch.float32, "ht")
    x, cu, _ = inputs([4], 1, 1, 257, 8, torch.float32, seed=15)
    with pytest.raises(NotImplementedError):
        chunk_gated_delta(*(t.to(dev) for t in x), cu.to(dev))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hk,H,K,V", [(1, 2, 32, 16), (2, 4, 16, 17), (1, 1, 1, 1), (2, 2, 24, 40)])
def test_chunk_kernels_on_short_sequences(dev, dtype, Hk, H, K, V):
    """The chunk kernels on batches that chunk_gated_delta gives to the other
    kernel, and both of them on either side of the rule."""
    from ssla_amd.delta import _chunk_fwd, _token_rows, chunk_gated_delta
    lens = [0, 1, 63, 64, 65, 30, 7, 0]
    assert sum(lens) <= len(lens) * _token_rows(K)
    x, cu, s0 = inputs(lens, Hk, H, K, V, dtype, seed=K + V)
    d = [t.to(dev) for t in x]
    o, ht, _ = _chunk_fwd(*d, cu.to(dev), 0.5, s0.to(dev), True)
    ro, rs = gated_delta(*x, lens, 0.5, s0)
    close(o, ro, K, max(lens), dtype, "o")
    close(ht, rs, K, max(lens), torch.float32, "ht")
    for n in (1, 2):   # T = n rows: token by token; 1 sequence of more: chunks
        few = [t[:n * _token_rows(K) // 2 + 1] for t in x]
        T = few[0].shape[0]
        o, ht = run(dev, few, torch.tensor([0, T]), s0[:1], scale=0.5)
        ro, rs = gated_delta(*few, [T], 0.5, s0[:1])
        close(o, ro, K, T, dtype, "o")
        close(ht, rs, K, T, torch.float32, "ht")


MANY = [5, 0, 3, 800, 2, 1, 0, 7, 1100] + [1, 0, 2] * 8 + [513, 9, 300]   # more sequences than inner segments


@pytest.mark.parametrize("dtype,K,V", [(torch.bfloat16, 64, 64), (torch.float32, 24, 40)])
def test_long_among_many_short(dev, dtype, K, V):
    """Long sequences that start in a unit of rows where short ones lie too, with
    a gradient recorded (the chunk kernels whatever the average length is)."""
    x, cu, s0 = inputs(MANY, 1, 2, K, V, dtype, seed=K)
    x[3] = x[3] / 8
    x[4].requires_grad_()
    o, ht = run(dev, x, cu, s0)
    assert o.requires_grad
    ro, rs = gated_delta(*(t.detach() for t in x), MANY, K ** -0.5, s0)
    close(o.detach(), ro, K, max(MANY), dtype, "o")
    close(ht.detach(), rs, K, max(MANY), torch.float32, "ht")
