"""The gated recurrence over packed sequences and its single tokens against the
definition in 64 bits.

Tolerance, with u = 2^-24 (half a step of fp32).  A gate is off by at most 10 u of
its value: e^x by 4 (the unit's 2, and two roundings of its correction), sigmoid by
4 + 1 for 1 + e^-|g|, 2 for the reciprocal, and for negative logits 4 + 1 of the
product with e^-|g|.  A step adds 1 for its own rounding, and where pieces of the
time axis are joined 1 for the product of the gates and 1 for the join.  So every
step is off by at most 13 u of its terms' sizes: EPS = 16 u, carried through the
recurrence as oracle.block says.  A 16-bit output is rounded once: half a step of its
type, and values below its normal range by half of its smallest step."""
import pytest
import torch

from oracle.block import gated_scan as ref_scan

pytestmark = pytest.mark.gpu
EPS = 16 * 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}
F32, B16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [(F32, F32), (B16, B16), (B16, F32), (F16, F16), (F16, F32)]
# lengths: one row, odd ones, empty ones at either end and between, starts on every kind of border, long ones
LENS = [[1], [77], [0, 3, 0, 0, 130, 1, 1, 0], [64, 64, 128, 256, 512], [5] * 300, [2049, 1, 63, 4096, 65], [0, 0], [20000]]


def inputs(lens, C, dt, dtg, gate, seed, T=None):
    gen = torch.Generator().manual_seed(seed)
    T, N = sum(lens) if T is None else T, len(lens)
    g = torch.randn(T, C, generator=gen) * 2 + 2
    g = {"sigmoid": g, "log": torch.nn.functional.logsigmoid(g), "value": torch.sigmoid(g) * (1 - 2 * (g < 0).float())}[gate]
    x = {"u": torch.randn(T, C, generator=gen).to(dt), "g": g.to(dtg), "q": torch.randn(T, C, generator=gen).to(dt),
         "h0": torch.randn(N, C, generator=gen), "do": torch.randn(T, C, generator=gen).to(dt),
         "dht": torch.randn(N, C, generator=gen)}
    return x


def offsets(lens, first=0):
    return torch.tensor([first, *lens]).cumsum(0)


def compare(name, got, want, off, dtype):
    tol = off + HALF[dtype] * (want.abs() + off) + TINY[dtype]
    err = (got.double().cpu() - want).abs()
    assert got.dtype == dtype and got.shape == want.shape, name
    assert bool((err <= tol).all()), f"{name}: {float((err - tol).max()):.3g} over, worst {float(err.max()):.3g}"


def check(dev, lens, x, gate, read=True, state=True, first=0, total=None, cu_dtype=torch.int64, lay=lambda t: t):
    """Forward, with and without a gradient, and backward."""
    from ssla_amd.scan import gated_scan
    T = sum(lens)
    total = T if total is None else total
    dt, dtg = x["u"].dtype, x["g"].dtype
    ref = ref_scan(*(x[n][first:first + T] for n in ("u", "g")), lens, x["q"][first:first + T] if read else None, gate,
                   x["h0"] if state else None, x["do"][first:first + T], x["dht"] if state else None, EPS)
    d = {n: lay(t.to(dev)) for n, t in x.items()}
    leaves = [d[n].detach().requires_grad_() for n in ("u", "g", "q", "h0")]
    u, g, q, h0 = leaves[0], leaves[1], leaves[2] if read else None, leaves[3] if state else None
    cu = offsets(lens, first).to(cu_dtype).to(dev)
    with torch.no_grad():
        alone = gated_scan(u, g, cu, q=q, gate=gate, initial_state=h0, output_final_state=True)
        bare, none = gated_scan(u, g, cu, q=q, gate=gate, initial_state=h0)
    assert none is None and torch.equal(bare, alone[0])
    o, ht = gated_scan(u, g, cu, q=q, gate=gate, initial_state=h0, output_final_state=True)
    assert torch.equal(o, alone[0]) and torch.equal(ht, alone[1])
    wanted = [t for t in (u, g, q, h0) if t is not None]
    got = torch.autograd.grad((o, ht) if state else (o,), wanted, (d["do"], d["dht"]) if state else (d["do"],))
    grads = dict(zip([n for n, t in zip(("du", "dg", "dq", "dh0"), (u, g, q, h0)) if t is not None], got))

    def whole(t):
        out = torch.zeros(total, t.shape[1], dtype=torch.float64)
        out[first:first + T] = t
        return out

    compare("o", o.detach(), whole(ref["o"][0]), whole(ref["o"][1]), dt)
    compare("ht", ht.detach(), *ref["ht"], F32)
    for n, t in grads.items():
        if n == "dh0":
            compare(n, t, *ref[n], F32)
        else:
            compare(n, t, *map(whole, ref[n]), dtg if n == "dg" else dt)


@pytest.mark.parametrize("dt,dtg", TYPES)
@pytest.mark.parametrize("lens", LENS, ids=lambda x: f"{len(x)}x{max(x)}")
def test_lengths(dev, lens, dt, dtg):
    C = 8 if max(lens) > 5000 else 40
    check(dev, lens, inputs(lens, C, dt, dtg, "sigmoid", seed=len(lens)), "sigmoid")


@pytest.mark.parametrize("dt,dtg", TYPES)
@pytest.mark.parametrize("gate", ["value", "log", "sigmoid"])
@pytest.mark.parametrize("C", [1, 3, 12, 24, 75, 136, 264, 1000])
def test_channels_and_gates(dev, C, gate, dt, dtg):
    lens = [70, 0, 201, 9, 300]
    x = inputs(lens, C, dt, dtg, gate, seed=C)
    check(dev, lens, x, gate)
    check(dev, lens, x, gate, read=False, state=False)


@pytest.mark.parametrize("read", [True, False])
@pytest.mark.parametrize("state", [True, False])
def test_rows_in_no_sequence(dev, read, state):
    """Rows before the first and behind the last sequence: zeros, also where they
    hold NaN and infinities, and the sequences do not see them."""
    lens, first, total = [100, 0, 700, 33], 131, 131 + 833 + 300
    for dt, C in ((F32, 20), (B16, 64)):
        x = inputs(lens, C, dt, dt, "sigmoid", seed=5, T=total)
        for n in ("u", "g", "q", "do"):
            x[n][:first], x[n][first + 833:] = torch.nan, torch.inf
        check(dev, lens, x, "sigmoid", read, state, first, total, torch.int32)


def test_slices_of_a_projection(dev):
    """u, g and q as columns of one matrix, off 16-byte borders too; rows in another
    memory order; a gradient that is a transposed view."""
    lens, C = [150, 220], 48
    for dt in (F32, F16):
        x = inputs(lens, C, dt, dt, "log", seed=8)
        for pad in (0, 3, 5):
            def lay(t, pad=pad):
                if t.shape[0] != 370:
                    return t
                wide = torch.zeros(370, 3 * C + pad, dtype=t.dtype, device=t.device)
                wide[:, C + pad:2 * C + pad] = t
                return wide[:, C + pad:2 * C + pad]
            check(dev, lens, x, "log", lay=lay)
        check(dev, lens, x, "log", lay=lambda t: t.t().contiguous().t())


def test_broadcast_inputs(dev):
    """Rows that are one row expanded: the gradient is summed over them."""
    from ssla_amd.scan import gated_scan
    lens, C = [90, 40], 16
    x = inputs(lens, C, F32, F32, "sigmoid", seed=2)
    cu = offsets(lens).to(dev)
    full = [x[n].to(dev) for n in ("u", "q")]
    row = x["g"][:1].to(dev).requires_grad_()
    o, _ = gated_scan(full[0], row.expand(130, C), cu, q=full[1], gate="sigmoid")
    got, = torch.autograd.grad(o, row, x["do"].to(dev))
    many = row.detach().expand(130, C).contiguous().requires_grad_()
    o2, _ = gated_scan(full[0], many, cu, q=full[1], gate="sigmoid")
    want, = torch.autograd.grad(o2, many, x["do"].to(dev))
    assert torch.equal(o, o2) and torch.equal(got, want.sum(0, keepdim=True))


@pytest.mark.parametrize("C", [8, 96])
def test_gates_at_the_edges(dev, C):
    """Closed gates cut the sequence, open ones keep it, resets in log form; a state
    of NaN or infinity stays in its sequence and channel."""
    from ssla_amd.scan import gated_scan
    lens = [400, 300, 50]
    cu = offsets(lens).to(dev)
    x = inputs(lens, C, F32, F32, "log", seed=3)
    x["g"][::7] = -torch.inf
    x["g"][3::11] = 0
    check(dev, lens, x, "log")
    y = inputs(lens, C, F32, F32, "sigmoid", seed=3)
    y["g"][::7] = -torch.inf
    y["g"][3::11] = torch.inf
    y["g"][5::13] = -200
    y["g"][6::13] = 200
    check(dev, lens, y, "sigmoid")
    u, g = x["u"].to(dev), x["g"].clamp(min=-3).to(dev)
    clean, ct = gated_scan(u, g, cu, gate="log", output_final_state=True)
    for v in (torch.nan, torch.inf):
        bad = u.clone()
        bad[420, 2] = v
        o, ht = gated_scan(bad, g, cu, gate="log", output_final_state=True)
        same = torch.ones_like(o, dtype=torch.bool)
        same[420:700, 2] = False
        assert torch.equal(o[same], clean[same]) and not o[420, 2].isfinite()
        assert torch.equal(ht[[0, 2]], ct[[0, 2]]) and torch.equal(ht[1, 3:], ct[1, 3:])
        h0 = torch.zeros(3, C, device=dev)
        h0[1, 2] = v
        o, _ = gated_scan(u, g, cu, gate="log", initial_state=h0)
        same[400:700, 2] = False
        assert torch.equal(o[same], clean[same])


def test_differences(dev):
    """A direction's slope against central differences of the loss in fp32: their
    distance bounds the third-order term, the loss's rounding is 2000 sums of values
    that are off by 2^-20."""
    from ssla_amd.scan import gated_scan
    lens, C = [100, 30], 12
    cu = offsets(lens).to(dev)
    for gate in ("value", "log", "sigmoid"):
        x = inputs(lens, C, F32, F32, gate, seed=6)
        names = ("u", "g", "q", "h0")
        d = {n: torch.randn(x[n].shape, generator=torch.Generator().manual_seed(i)) for i, n in enumerate(names)}

        def loss(h):
            u, g, q, h0 = ((x[n] + h * d[n]).to(dev) for n in names)
            o, ht = gated_scan(u, g, cu, q=q, gate=gate, initial_state=h0, output_final_state=True)
            return float((o.double().cpu() * x["do"]).sum() + (ht.double().cpu() * x["dht"]).sum())

        leaves = [x[n].to(dev).requires_grad_() for n in names]
        out = gated_scan(leaves[0], leaves[1], cu, q=leaves[2], gate=gate, initial_state=leaves[3], output_final_state=True)
        grads = torch.autograd.grad(out, leaves, (x["do"].to(dev), x["dht"].to(dev)))
        slope = sum(float((gr.double().cpu() * d[n]).sum()) for n, gr in zip(names, grads))
        h = 2.0 ** -8
        two = [(loss(h) - loss(-h)) / (2 * h), (loss(2 * h) - loss(-2 * h)) / (4 * h)]
        diff = (4 * two[0] - two[1]) / 3
        assert abs(diff - slope) <= abs(two[0] - two[1]) + 2000 * 2.0 ** -20 / h, gate


def test_one_gradient_of_several(dev):
    """Gradients of o alone, of ht alone, and of one input are those of the whole."""
    from ssla_amd.scan import gated_scan
    lens, C = [300, 200], 24
    cu = offsets(lens).to(dev)
    x = {n: t.to(dev) for n, t in inputs(lens, C, F32, F32, "sigmoid", seed=1).items()}

    def run(grads, *names):
        leaves = {n: x[n].clone().requires_grad_(n in names) for n in ("u", "g", "q", "h0")}
        o, ht = gated_scan(leaves["u"], leaves["g"], cu, q=leaves["q"], gate="sigmoid", initial_state=leaves["h0"],
                           output_final_state=True)
        out = {"o": (o, x["do"]), "ht": (ht, x["dht"])}
        return torch.autograd.grad([out[n][0] for n in grads], [leaves[n] for n in names], [out[n][1] for n in grads])

    all_of = run(("o", "ht"), "u", "g", "q", "h0")
    for i, n in enumerate(("u", "g", "q", "h0")):
        assert torch.equal(run(("o", "ht"), n)[0], all_of[i])
    ref = ref_scan(*(x[n].cpu() for n in ("u", "g")), lens, x["q"].cpu(), "sigmoid", x["h0"].cpu(), 0 * x["do"].cpu(),
                   x["dht"].cpu(), EPS)
    for n, t in zip(("du", "dg", "dq", "dh0"), run(("ht",), "u", "g", "q", "h0")):
        compare(n, t, *ref[n], F32)


def test_the_same_every_time(dev):
    from ssla_amd.scan import gated_scan
    for lens, C in (([30000], 64), ([3000] * 12, 256), ([17] * 2000, 40)):
        x = {n: t.to(dev) for n, t in inputs(lens, C, B16, F32, "sigmoid", seed=9).items()}
        cu = offsets(lens).to(dev)
        leaves = [x[n].requires_grad_() for n in ("u", "g", "q", "h0")]
        runs = []
        for _ in range(6):
            out = gated_scan(*leaves[:2], cu, q=leaves[2], gate="sigmoid", initial_state=leaves[3], output_final_state=True)
            runs.append([t.detach() for t in out] + list(torch.autograd.grad(out, leaves, (x["do"], x["dht"]))))
        assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(runs[0], r)), lens


def test_no_rows(dev):
    from ssla_amd.scan import gated_scan
    h0 = torch.randn(2, 8, generator=torch.Generator().manual_seed(1)).to(dev).requires_grad_()
    e = torch.zeros(0, 8, device=dev, requires_grad=True)
    o, ht = gated_scan(e, e, torch.zeros(3, dtype=torch.int64, device=dev), q=e, initial_state=h0, output_final_state=True)
    assert o.shape == (0, 8) and torch.equal(ht, h0)
    ht.square().sum().backward()
    assert torch.equal(h0.grad, 2 * h0.detach()) and e.grad.shape == (0, 8)
    x = torch.ones(5, 8, device=dev)
    o, ht = gated_scan(x, x, torch.zeros(1, dtype=torch.int64, device=dev), output_final_state=True)
    assert not o.any() and ht.shape == (0, 8)


@pytest.mark.parametrize("lens", [[9000, 0, 40], [30] * 50])
def test_a_training_step_in_a_graph(dev, lens):
    """Captured once, replayed on changing inputs with eager steps in between."""
    from ssla_amd.scan import gated_scan
    C = 72
    x = {n: t.to(dev) for n, t in inputs(lens, C, B16, B16, "sigmoid", seed=4).items()}
    cu = offsets(lens).to(dev)
    names = ("u", "g", "q", "h0")

    def step(leaves):
        out = gated_scan(*leaves[:2], cu, q=leaves[2], gate="sigmoid", initial_state=leaves[3], output_final_state=True)
        return *(t.detach() for t in out), *torch.autograd.grad(out, leaves, (x["do"], x["dht"]))

    static = [x[n].clone().requires_grad_() for n in names]
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
            for s, n in zip(static, names):
                s.copy_(x[n] * (1 + 0.25 * i))
        graph.replay()
        want = step([s.detach().clone().requires_grad_() for s in static])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_two_streams_at_once(dev):
    from ssla_amd.scan import gated_scan
    work = []
    for i, (lens, C) in enumerate((([40000], 128), ([5000] * 7, 200))):
        x = {n: t.to(dev) for n, t in inputs(lens, C, B16, F32, "log", seed=i).items()}
        work.append((x, offsets(lens).to(dev)))
    want = [gated_scan(x["u"], x["g"], cu, q=x["q"], gate="log", initial_state=x["h0"], output_final_state=True)
            for x, cu in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    got = [[], []]
    for _ in range(5):
        for i, (s, (x, cu)) in enumerate(zip(streams, work)):
            with torch.cuda.stream(s):
                got[i].append(gated_scan(x["u"], x["g"], cu, q=x["q"], gate="log", initial_state=x["h0"],
                                         output_final_state=True))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for g in got[i] for a, b in zip(g, want[i]))


# ---------------------------------------------------------- single tokens --
@pytest.mark.parametrize("dt,dtg", TYPES)
@pytest.mark.parametrize("gate", ["value", "log", "sigmoid"])
@pytest.mark.parametrize("rows,n,C", [(1, 1, 1), (300, 77, 30), (50, 50, 96), (4560, 912, 200), (9, 4, 1000)])
def test_step(dev, rows, n, C, gate, dt, dtg):
    from ssla_amd.scan import sparse_gated_step
    x = inputs([1] * n, C, dt, dtg, gate, seed=rows)
    gen = torch.Generator().manual_seed(n)
    table = torch.randn(rows, C, generator=gen)
    at = torch.randperm(rows, generator=gen)[:n].sort().values
    for read in (True, False):
        ref = ref_scan(x["u"], x["g"], [1] * n, x["q"] if read else None, gate, table[at], eps=EPS)
        state = table.to(dev)
        o = sparse_gated_step(at.to(dev), x["u"].to(dev), x["g"].to(dev), state, q=x["q"].to(dev) if read else None,
                              gate=gate, check=True)
        compare("o", o, *ref["o"], dt)
        want, off = table.double(), torch.zeros(rows, C, dtype=torch.float64)
        want[at], off[at] = ref["ht"]
        compare("state", state, want, off, F32)
        rest = torch.ones(rows, dtype=torch.bool)
        rest[at] = False
        assert torch.equal(state.cpu()[rest], table[rest])


def test_steps_are_a_scan(dev):
    """Tokens one by one through a table and one call over them agree."""
    from ssla_amd.scan import gated_scan, sparse_gated_step
    C, n, steps = 40, 6, 5
    x = {k: t.to(dev) for k, t in inputs([steps] * n, C, F32, F32, "sigmoid", seed=0).items()}
    at = torch.tensor([1, 2, 5, 7, 8, 11], device=dev)
    state = torch.zeros(12, C, device=dev)
    state[at] = x["h0"]
    o, ht = gated_scan(x["u"], x["g"], offsets([steps] * n).to(dev), q=x["q"], gate="sigmoid", initial_state=x["h0"],
                       output_final_state=True)
    for t in range(steps):
        rows = torch.arange(n, device=dev) * steps + t
        assert torch.allclose(sparse_gated_step(at, x["u"][rows], x["g"][rows], state, q=x["q"][rows], gate="sigmoid"), o[rows],
                              rtol=0, atol=64 * EPS)
    assert torch.allclose(state[at], ht, rtol=0, atol=64 * EPS)


def test_step_skips_bad_entries(dev):
    from ssla_amd.scan import sparse_gated_step
    C = 24
    x = {k: t.to(dev) for k, t in inputs([1] * 6, C, F32, F32, "value", seed=0).items()}
    table = torch.randn(10, C, generator=torch.Generator().manual_seed(1)).to(dev)
    good = table.clone()
    sparse_gated_step(torch.tensor([0, 9], device=dev), x["u"][[0, 5]], x["g"][[0, 5]], good)   # (the first 4 is not above 10)
    for idx in (torch.tensor([0, -1, 10, 4, 4, 9]), torch.tensor([0, -(1 << 40), 1 << 40, 4, 4, 9])):
        state = table.clone()
        o = sparse_gated_step(idx.to(dev), x["u"], x["g"], state)
        assert torch.equal(state, good) and not o[1:5].any() and o[[0, 5]].all()
        with pytest.raises(ValueError, match="strictly increasing"):
            sparse_gated_step(idx.to(dev), x["u"], x["g"], table.clone(), check=True)
    e = torch.zeros(0, C, device=dev)
    assert sparse_gated_step(torch.zeros(0, dtype=torch.int32, device=dev), e, e, table).shape == (0, C)


def test_past_32_bits(dev):
    """2^31 values a tensor: the last rows are those of a short call on the end alone
    (gates of about a half forget 200 rows to nothing), in both directions."""
    from ssla_amd.scan import gated_scan
    T, C = (1 << 21) + 1000, 1024
    gen = torch.Generator(device=dev).manual_seed(0)
    u, g, do = (torch.randn(T, C, generator=gen, device=dev, dtype=B16) for _ in range(3))
    u.requires_grad_(), g.requires_grad_()
    o, ht = gated_scan(u, g, torch.tensor([0, T], device=dev), gate="sigmoid", output_final_state=True)
    du, dg = torch.autograd.grad(o, (u, g), do)
    for rows in (slice(T - 2000, T), slice(0, 2000)):
        a, b = (t.detach()[rows].clone().requires_grad_() for t in (u, g))
        p, pt = gated_scan(a, b, torch.tensor([0, 2000], device=dev), gate="sigmoid", output_final_state=True)
        da, db = torch.autograd.grad(p, (a, b), do[rows])
        mid = slice(1000, 1500)   # (1,000 rows from one end, 500 from the other)
        for whole, part in ((o, p), (du, da), (dg, db)):
            w, q = whole[rows][mid].detach().double(), part[mid].detach().double()
            assert bool(((w - q).abs() <= 2.0 ** -7 * q.abs() + 1e-4).all())   # (one rounding either side of a border)
        if rows.start:
            assert torch.allclose(ht, pt, rtol=0, atol=64 * EPS)


def test_offsets_that_decrease_end(dev):
    """Offsets that are not in order leave their rows unspecified; the call ends, and a good
    one after it is right."""
    from ssla_amd.scan import gated_scan
    x = {n: t.to(dev) for n, t in inputs([900], 40, F32, F32, "sigmoid", seed=1).items()}
    good = torch.tensor([0, 900], device=dev)
    want = gated_scan(x["u"], x["g"], good, gate="sigmoid")[0]
    for cu in ([0, 500, 200, 900], [900, 0, 900], [-5, 2000, 3], [700, 700, 100]):
        u = x["u"].clone().requires_grad_()
        n = len(cu) - 1
        o, ht = gated_scan(u, x["g"], torch.tensor(cu, device=dev), gate="sigmoid",
                           initial_state=torch.zeros(n, 40, device=dev), output_final_state=True)
        torch.autograd.grad((o, ht), u, (torch.ones_like(o), torch.ones_like(ht)))
        torch.cuda.synchronize()
        assert torch.equal(gated_scan(x["u"], x["g"], good, gate="sigmoid")[0], want)


def test_two_graphs_of_one_pool(dev):
    """Two captured calls whose workspaces may share memory, replayed in turn."""
    from ssla_amd.scan import gated_scan
    sets = [{n: t.to(dev) for n, t in inputs([6000, 50], C, B16, B16, "sigmoid", seed=C).items()} for C in (64, 136)]
    cu = offsets([6000, 50]).to(dev)

    def call(x):
        return gated_scan(x["u"], x["g"], cu, q=x["q"], gate="sigmoid", initial_state=x["h0"], output_final_state=True)

    want = [call(x) for x in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        [call(x) for x in sets]
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs, pool = [], [], None
    for x in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outs.append(call(x))
        pool = graph.pool()
        graphs.append(graph)
    for i in range(4):
        for graph, out, w in zip(graphs, outs, want):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, w)), i


def test_many_sequences(dev):
    """More sequences than a workgroup has threads, of one row and of none."""
    gen = torch.Generator().manual_seed(0)
    lens = torch.randint(0, 3, (3000,), generator=gen).tolist()
    check(dev, lens, inputs(lens, 12, F32, F32, "sigmoid", seed=0), "sigmoid")
    check(dev, [1] * 1500, inputs([1] * 1500, 8, B16, F32, "log", seed=1), "log")
    lens = [0] * 2000 + [700] + [0] * 2000
    check(dev, lens, inputs(lens, 8, F32, F32, "value", seed=2), "value")


def test_states_off_16_bytes(dev):
    """Tables, initial states and gradients of final ones that begin at any 4-byte border."""
    from ssla_amd.scan import gated_scan, sparse_gated_step
    lens, C = [3, 0, 70, 1], 16
    x = {n: t.to(dev) for n, t in inputs(lens, C, F32, F32, "sigmoid", seed=7).items()}
    cu = offsets(lens).to(dev)

    def off(t):
        return torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)

    def run(lay):
        leaves = [x[n].clone().requires_grad_() for n in ("u", "g")] + [lay(x["h0"]).requires_grad_()]
        out = gated_scan(leaves[0], leaves[1], cu, gate="sigmoid", initial_state=leaves[2], output_final_state=True)
        return *out, *torch.autograd.grad(out, leaves, (x["do"], lay(x["dht"])))

    assert all(torch.equal(a, b) for a, b in zip(run(off), run(torch.clone)))
    at, tables = torch.tensor([0, 2], device=dev), [off(x["h0"]), x["h0"].clone()]
    outs = [sparse_gated_step(at, x["u"][:2], x["g"][:2], t, gate="sigmoid") for t in tables]
    assert torch.equal(*outs) and torch.equal(*tables)


@pytest.mark.parametrize("dt", [F32, B16])
def test_steps_in_a_graph(dev, dt):
    """A single token's step captured once and replayed: the table goes on from replay to
    replay, with other tokens and other rows, as in eager steps."""
    from ssla_amd.scan import sparse_gated_step
    rows, n, C = 50, 9, 40
    gen = torch.Generator().manual_seed(2)
    tokens = [[torch.randn(n, C, generator=gen).to(dev, dt) for _ in range(3)] for _ in range(5)]
    sites = [torch.randperm(rows, generator=gen)[:n].sort().values.int().to(dev) for _ in range(5)]
    u, g, q = (t.clone() for t in tokens[0])
    at, state = sites[0].clone(), torch.zeros(rows, C, device=dev)
    sparse_gated_step(at, u, g, state, q=q, gate="sigmoid")
    state.zero_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = sparse_gated_step(at, u, g, state, q=q, gate="sigmoid")
    table = torch.zeros_like(state)
    for i, (x, idx) in enumerate(zip(tokens, sites)):
        for to, t in zip((u, g, q, at), (*x, idx)):
            to.copy_(t)
        graph.replay()
        want = sparse_gated_step(idx, x[0], x[1], table, q=x[2], gate="sigmoid")
        torch.cuda.synchronize()
        assert torch.equal(o, want) and torch.equal(state, table), i


# sequences over many tiles of narrow rows: one, ends on and beside powers of two, short ones between
@pytest.mark.parametrize("dt,dtg", [(F32, F32), (B16, F32)])
@pytest.mark.parametrize("lens,C", [([70000], 4), ([8192, 8191, 16385, 1, 0, 20000], 20), ([3, 30000, 0, 2], 7),
                                    ([1000, 12000], 200)], ids=lambda x: str(x).replace(" ", ""))
def test_long_narrow(dev, lens, C, dt, dtg):
    check(dev, lens, inputs(lens, C, dt, dtg, "sigmoid", seed=C), "sigmoid")


def test_long_narrow_the_same_every_time(dev):
    """Gates near 1, so that every state reaches far: repeated calls give the same bits, and
    offsets that are not in order still end."""
    from ssla_amd.scan import gated_scan
    T, C = 200000, 24
    gen = torch.Generator().manual_seed(8)
    u, do = (torch.randn(T, C, generator=gen).to(dev) for _ in range(2))
    u.requires_grad_()
    g = (torch.randn(T, C, generator=gen) + 9).to(dev).requires_grad_()
    bad = torch.tensor([0, 150000, 20, 199999, 100000, 7, T], device=dev)
    want = None
    for i in range(6):
        o, ht = gated_scan(u, g, torch.tensor([0, T], device=dev), gate="sigmoid", output_final_state=True)
        got = o.detach(), ht.detach(), *torch.autograd.grad(o, (u, g), do)
        if want is not None:
            assert all(torch.equal(a, b) for a, b in zip(got, want)), i
        want = got
        gated_scan(u.detach(), g.detach(), bad, gate="sigmoid", output_final_state=True)
    torch.cuda.synchronize()


def compare_all(name, got, want, off, dtype):
    """As compare(), with the same NaN and infinities in the same places."""
    have = got.double().cpu()
    assert torch.equal(have.isnan(), want.isnan()), name
    infinite, finite = want.isinf(), want.isfinite()
    assert torch.equal(have[infinite], want[infinite]), name
    compare(name, got.cpu()[finite], want[finite], off[finite], dtype)


# tiles of 256 rows (128 in the backward) without spans, of 512 with spans, single channels
@pytest.mark.parametrize("gate", ["value", "log", "sigmoid"])
@pytest.mark.parametrize("C,n", [(300, 2500), (8, 20000), (7, 9000)])
def test_infinite_states_go_on(dev, C, n, gate):
    """An infinite state, or gradient, stays so through rows whose gates multiply to less
    than fp32 holds, with the gates' signs, until a gate of exactly 0 makes it NaN; as row by row."""
    from ssla_amd.scan import gated_scan
    lens = [400, n, 50]
    x = inputs(lens, C, F32, F32, gate, seed=11)
    x["g"] = x["g"] * 0.5 if gate == "value" else x["g"] - 2
    x["u"][420, 2], x["u"][430, 5], x["h0"][1, 3] = torch.inf, -torch.inf, torch.inf
    x["u"][1000, 6] = torch.nan
    x["do"][n + 300, 1], x["dht"][1, 0] = torch.inf, -torch.inf
    if gate != "sigmoid":
        x["g"][2000, 2] = x["g"][600, 4] = 0 if gate == "value" else -torch.inf
    ref = ref_scan(x["u"], x["g"], lens, x["q"], gate, x["h0"], x["do"], x["dht"], EPS)
    leaves = [x[k].to(dev).requires_grad_() for k in ("u", "g", "q", "h0")]
    o, ht = gated_scan(*leaves[:2], offsets(lens).to(dev), q=leaves[2], gate=gate, initial_state=leaves[3], output_final_state=True)
    grads = torch.autograd.grad((o, ht), leaves, (x["do"].to(dev), x["dht"].to(dev)))
    for k, t in zip(("o", "ht", "du", "dg", "dq", "dh0"), (o.detach(), ht.detach(), *grads)):
        compare_all(k, t, *ref[k], F32)
    assert ref["o"][0][420:1900, 2].isinf().all() and ref["du"][0][500:n, 0].isinf().all()


# two channel blocks or more without spans, with spans, single channels
@pytest.mark.parametrize("gate", ["value", "log"])
@pytest.mark.parametrize("C,n", [(300, 2500), (8, 20000), (7, 9000)])
def test_gates_above_one(dev, C, n, gate):
    """Gates around 1, whose products grow and fall by up to some powers of ten over a piece
    of the time axis, in both directions."""
    lens = [400, n, 50]
    x = inputs(lens, C, F32, F32, "value", seed=12)
    g = torch.randn(x["g"].shape, generator=torch.Generator().manual_seed(1)) * 0.02 + 0.0005
    x["g"] = g if gate == "log" else torch.exp(g) * (1 - 2 * (x["g"] < 0.5).float())
    assert float((g if gate == "log" else x["g"].abs().log()).cumsum(0).abs().max()) > 5
    check(dev, lens, x, gate)
    check(dev, lens, x, gate, read=False, state=False)


def row_by_row(x, gate):
    """One sequence in fp32, for where it passes fp32."""
    a, slope = (x["g"], 1.0) if gate == "value" else (x["g"].exp(), x["g"].exp())
    h, states = x["h0"][0], []
    for t in range(x["u"].shape[0]):
        states.append(h)
        h = a[t] * h + x["u"][t]
    states.append(h)
    e, grads = x["dht"][0], []
    for t in range(x["u"].shape[0] - 1, -1, -1):
        grads.append(x["q"][t] * x["do"][t] + e)
        e = a[t] * grads[-1]
    h, s = torch.stack(states), torch.stack(grads[::-1])
    return {"o": x["q"] * h[1:], "ht": h[-1:], "du": s, "dg": s * h[:-1] * slope, "dq": x["do"] * h[1:], "dh0": e[None]}


@pytest.mark.parametrize("gate", ["value", "log"])
@pytest.mark.parametrize("C,n", [(300, 2500), (8, 20000), (7, 9000)])
def test_products_past_fp32(dev, C, n, gate):
    """Gates whose product over a piece of the time axis passes fp32: a state, or gradient, of 0
    stays 0, and a gate of 0 behind them (before them for gradients) empties any finite
    state as it does row by row."""
    from ssla_amd.scan import gated_scan
    lens = [n]
    x = inputs(lens, C, F32, F32, "value", seed=13)
    x["g"] = x["g"].abs()
    # forward: 1e-30 from row 500 on, times 8^64 over rows 640 .. 703, emptied at row 704
    x["g"][500] = x["g"][704] = 0
    x["g"][501:640], x["g"][640:704] = 1, 8
    x["u"][500], x["u"][501:704] = 1e-30, 0
    # backward: 1e-30 from row 1299 down, times 8^64 over rows 1164 .. 1101, emptied at row 1100
    x["g"][1100] = x["g"][1300] = 0
    x["g"][1101:1165], x["g"][1165:1300] = 8, 1
    x["u"][1100:1300], x["do"][1100:1299], x["do"][1299] = 0, 0, 1e-30
    # 0 in either direction through 8^200
    x["g"][1500] = x["g"][1701] = 0
    x["g"][1501:1701] = 8
    x["u"][1500:1701], x["do"][1500:1701] = 0, 0
    if gate == "log":
        x["g"] = x["g"].log()
    ref = ref_scan(x["u"], x["g"], lens, x["q"], gate, x["h0"], x["do"], x["dht"], EPS)
    rows = row_by_row(x, gate)
    leaves = [x[k].to(dev).requires_grad_() for k in ("u", "g", "q", "h0")]
    o, ht = gated_scan(*leaves[:2], offsets(lens).to(dev), q=leaves[2], gate=gate, initial_state=leaves[3], output_final_state=True)
    grads = torch.autograd.grad((o, ht), leaves, (x["do"].to(dev), x["dht"].to(dev)))
    for k, t in zip(("o", "ht", "du", "dg", "dq", "dh0"), (o.detach(), ht.detach(), *grads)):
        compare_all(k, t, torch.where(rows[k].isfinite(), ref[k][0], rows[k].double()), ref[k][1], F32)
    # (the gradients of rows 639 to 500 are 8^64 = 6e57 of row 703's: infinite in fp32, NaN behind the gate of 0)
    assert rows["o"].isfinite().all() and rows["du"][704:].isfinite().all() and rows["du"][500:640].isinf().all()


def test_log_gates_to_the_ends_of_fp32(dev):
    """e^g, and the gate's gradient, wherever e^g is a normal number: off by 4 U of itself (the
    unit's 2, and two roundings of the correction), the gradient's products of 1 exact."""
    from ssla_amd.scan import gated_scan, sparse_gated_step
    g = torch.cat([torch.linspace(lo, hi, 4096) for lo, hi in ((-87.33654, -87), (-87, 87), (87, 88.72283), (-1, 1))])
    g = g.clamp(min=-87.33654, max=88.72283).view(64, 256).to(dev)
    want = g.double().exp()
    assert float(want.min()) >= torch.finfo(F32).tiny and float(want.max()) <= torch.finfo(F32).max
    none, one = torch.zeros_like(g), torch.ones_like(g)
    leaf = g.clone().requires_grad_()
    o, _ = gated_scan(none, leaf, torch.arange(65, device=dev), gate="log", initial_state=one)
    (dg,) = torch.autograd.grad(o, leaf, one)
    step = sparse_gated_step(torch.arange(64, device=dev), none, g, one.clone(), gate="log")
    for name, got in (("scan", o.detach()), ("gradient", dg), ("step", step)):
        off = (got.double() - want).abs() / want * 2 ** 24
        assert float(off.max()) <= 4, (name, float(off.max()), float(g.flatten()[off.argmax()]))


def test_logits_to_the_end_of_fp32(dev):
    """The sigmoid of a logit, wherever it is a normal number, by the 10 U of the bound above."""
    from ssla_amd.scan import gated_scan, sparse_gated_step
    g = torch.cat([torch.linspace(lo, hi, 4096) for lo, hi in ((-87.33654, -87), (-87, -1), (-1, 1), (1, 120))])
    g = g.clamp(min=-87.33654).view(64, 256).to(dev)
    want = 1 / (1 + torch.exp(-g.double()))
    assert float(want.min()) >= torch.finfo(F32).tiny
    none, one = torch.zeros_like(g), torch.ones_like(g)
    o, _ = gated_scan(none, g, torch.arange(65, device=dev), gate="sigmoid", initial_state=one)
    step = sparse_gated_step(torch.arange(64, device=dev), none, g, one.clone(), gate="sigmoid")
    for name, got in (("scan", o), ("step", step)):
        off = (got.double() - want).abs() / want * 2 ** 24
        assert float(off.max()) <= 10, (name, float(off.max()), float(g.flatten()[off.argmax()]))
