"""chunk_gated_delta without a gradient on batches whose sequences are short on
average: every sequence by the kernel for its own length (up to 64 rows token by
token, longer ones by chunks), whatever lies beside it.

A sequence's values do not depend on the batch where it is cut into the same
segments, so the two kernels' own results on the batch are compared bit for bit;
against the definition in 64 bits the bounds are test_gpu_delta_chunk's."""
import pytest
import torch

from oracle.delta import gated_delta
from tests.test_gpu_delta import inputs
from tests.test_gpu_delta_chunk import close

pytestmark = pytest.mark.gpu
BATCHES = {
    "prompt among single rows": [1] * 40 + [700] + [1] * 23,
    "prompt first": [600] + [1, 2] * 30,
    "prompt last, empty sequences before": [0] * 50 + [3, 0, 900],
    "padded by empty sequences": [1, 0, 300, 64, 65, 63] + [0] * 60,
    "several of each": [5, 0, 130, 2, 257, 64, 1, 128, 66, 33, 512] + [1, 9, 0] * 30 + [70],
    "no long one": [20, 1, 0, 64, 40] * 8,
}


def batch(lens, dtype, K, V, seed, Hk=1, H=2):
    x, cu, s0 = inputs(lens, Hk, H, K, V, dtype, seed=seed)
    x[3] = x[3] / 8   # a memory of many chunks
    return x, cu, s0


@pytest.mark.parametrize("dtype,Hk,H,K,V", [(torch.bfloat16, 1, 2, 64, 64), (torch.float32, 1, 2, 24, 40),
                                            (torch.float16, 3, 3, 32, 20), (torch.bfloat16, 1, 2, 16, 130)])
@pytest.mark.parametrize("name", BATCHES)
def test_every_sequence_by_its_own_length(dev, name, dtype, Hk, H, K, V):
    from ssla_amd.delta import _chunk_fwd, _token_rows, chunk_gated_delta, fused_recurrent_gated_delta
    lens = BATCHES[name]
    N, T = len(lens), sum(lens)
    assert 128 < T <= N * _token_rows(K)
    x, cu, s0 = batch(lens, dtype, K, V, K + V, Hk, H)
    d, cud, s0d = [t.to(dev) for t in x], cu.to(dev), s0.to(dev)
    o, ht = chunk_gated_delta(*d, cud, initial_state=s0d, output_final_state=True)
    to, ts = fused_recurrent_gated_delta(*d, cud, initial_state=s0d, output_final_state=True)
    co, cs, _ = _chunk_fwd(*d, cud, K ** -0.5, s0d, True)
    for n, rows in enumerate(lens):
        a, (wo, ws) = int(cu[n]), (to, ts) if rows <= 64 else (co, cs)
        assert torch.equal(o[a:a + rows], wo[a:a + rows]) and torch.equal(ht[n], ws[n]), (n, rows)
    long = [n for n in range(N) if lens[n] > 64]
    assert not long or not torch.equal(to[int(cu[long[0]]):], co[int(cu[long[0]]):])   # (the two can be told apart)
    ro, rs = gated_delta(*x, lens, K ** -0.5, s0)
    close(o, ro, K, max(lens), dtype, "o")
    close(ht, rs, K, max(lens), torch.float32, "ht")


def test_rows_outside_and_no_states(dev):
    """Rows in no sequence are not written; no initial state, no final one."""
    from ssla_amd import _lib
    from ssla_amd.delta import chunk_gated_delta
    lens = [2, 200, 0, 1, 64, 30] + [0] * 8
    x, _, _ = batch([4 + sum(lens) + 7], torch.float32, 32, 16, 3)
    cu = torch.tensor([4] + lens).cumsum(0)
    d, cud = [t.to(dev) for t in x], cu.to(dev)
    T, P, lib = d[0].shape[0], _lib.ptr, _lib.load()
    o = torch.full((T, 2, 16), 7.0, device=dev)
    ws = torch.empty(lib.ssla_gated_delta_mixed_workspace_size(T, 2, 32, 16), dtype=torch.uint8, device=dev)
    _lib.check(lib.ssla_gated_delta_mixed_fwd(*(P(t) for t in d), P(cud), len(lens), T, 1, 2, 32, 16, 0.5, None, P(o), None,
                                              _lib.SSLA_F32, P(ws), ws.numel(), _lib.stream_of(o)), "mixed")
    assert bool((o[:4] == 7).all()) and bool((o[-7:] == 7).all()) and not bool((o[4:-7] == 7).any())
    got, none = chunk_gated_delta(*d, cud, scale=0.5)
    assert none is None and torch.equal(got[4:-7], o[4:-7])
    ro, _ = gated_delta(*(t[4:-7] for t in x), lens, 0.5)
    close(got[4:-7], ro, 32, 200, torch.float32, "o")


def test_nonfinite_rows_stay_with_their_sequence(dev):
    from ssla_amd.delta import chunk_gated_delta
    lens = [3, 200, 5, 300] + [1] * 12
    x, cu, _ = batch(lens, torch.bfloat16, 32, 32, 5)
    clean, _ = chunk_gated_delta(*(t.to(dev) for t in x), cu.to(dev))
    for n in (0, 1, 2, 3):
        bad = [t.clone() for t in x]
        row = int(cu[n]) + 1
        bad[2][row, 1, 7] = torch.nan
        o, _ = chunk_gated_delta(*(t.to(dev) for t in bad), cu.to(dev))
        hit = torch.zeros_like(o, dtype=torch.bool)
        hit[row:int(cu[n + 1]), 1, 7] = True
        assert torch.equal(o[~hit], clean[~hit]) and not torch.isfinite(o[hit]).any(), n


def test_captured_with_offsets_that_change(dev):
    """One captured call, replayed on other lengths of the same rows (padded by
    empty sequences) with eager calls in between: every replay equals them."""
    from ssla_amd.delta import chunk_gated_delta
    N, T = 48, 900
    x, _, s0 = batch([T], torch.bfloat16, 64, 64, 6)
    s0 = s0.repeat(N, 1, 1, 1).to(dev)
    d = [t.to(dev) for t in x]
    cuts = [[T], [1] * 30 + [870], [400, 400, 100], [20] * 45, [64] * 14 + [4], [65] * 13 + [55]]
    cu = torch.zeros(N + 1, dtype=torch.int64, device=dev)

    def offsets(lens):
        return torch.tensor([0] + lens + [0] * (N - len(lens))).cumsum(0).to(dev)

    cu.copy_(offsets(cuts[0]))
    chunk_gated_delta(*d, cu, initial_state=s0, output_final_state=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, ht = chunk_gated_delta(*d, cu, initial_state=s0, output_final_state=True)
    for lens in cuts + cuts[:2]:
        cu.copy_(offsets(lens))
        graph.replay()
        eo, eh = chunk_gated_delta(*d, offsets(lens), initial_state=s0, output_final_state=True)
        torch.cuda.synchronize()
        assert torch.equal(o, eo) and torch.equal(ht, eh), lens[:3]


def test_rows_too_wide_for_chunks(dev):
    """Rows that only the token kernel's offsets reach run token by token, whatever
    their lengths (ssla_gated_delta_mixed_fwd takes no workspace then)."""
    from ssla_amd import _lib
    from ssla_amd.delta import chunk_gated_delta, fused_recurrent_gated_delta
    H, K, V, lens = 1 << 17, 64, 1, [1, 120, 1, 2, 9]
    assert _lib.load().ssla_gated_delta_mixed_workspace_size(sum(lens), H, K, V) == 0
    gen = torch.Generator(device=dev).manual_seed(1)
    T = sum(lens)
    q, k = (torch.nn.functional.normalize(torch.randn(T, 1, K, generator=gen, device=dev), dim=-1) for _ in range(2))
    v = torch.randn(T, H, V, generator=gen, device=dev)
    g, beta = -torch.rand(T, H, generator=gen, device=dev), torch.rand(T, H, generator=gen, device=dev)
    cu = torch.tensor([0] + lens, device=dev).cumsum(0)
    o, ht = chunk_gated_delta(q, k, v, g, beta, cu, output_final_state=True)
    to, ts = fused_recurrent_gated_delta(q, k, v, g, beta, cu, output_final_state=True)
    assert torch.equal(o, to) and torch.equal(ht, ts)
    at = [0, 77, H - 1]
    ro, _ = gated_delta(*(t.cpu() for t in (q.expand(-1, 3, -1), k.expand(-1, 3, -1), v[:, at], g[:, at], beta[:, at])), lens,
                        K ** -0.5)
    close(o[:, at], ro, K, max(lens), torch.float32, "o")
