"""The precision that the chunked gated delta rule promises: states, gradients and
the o of fp32 inputs are as good as fp32 arithmetic.

Bound: the root mean square of the error may be that of runs of the chunk form in 64
bits with a model of fp32's roundings in it, one for every term of a sum (the
matrix instructions add 32 terms of up to six pairs of parts at a time).  Results of
16 bits are rounded once more, by half a step at most.  On the CPU
test_delta_chunk_form shows that an operand that loses its third part passes these
bounds.  Maps of segments are not in the model: a long sequence's bounds hold for
them too.

Keys are normalised or not (|beta k^2| < 2 keeps the state's map from growing by
itself), gates fade fast, hardly, or grow."""
import pytest
import torch

from tests import delta_chunk_form as form
from tests.test_gpu_delta import HALF

NAMES = ("dq", "dk", "dv", "dg", "dbeta", "dh0")
CASES = ["fading", "long memory", "long keys", "like keys", "growing"]
SIZES = [(64, 64), (128, 40), (32, 32)]
H, T = 2, 300


def case(kind, dtype, K, V, T=T):
    gen = torch.Generator().manual_seed(K + V)

    def randn(*shape):
        return torch.randn(*shape, generator=gen)

    q, k = randn(T, H, K) * K ** -0.5, torch.nn.functional.normalize(randn(T, H, K), dim=-1)
    g = torch.nn.functional.logsigmoid(randn(T, H) + 1)
    beta = torch.sigmoid(2 * randn(T, H))
    if kind == "long memory":
        g = g / 64
    elif kind == "long keys":
        k = k * (0.2 + 1.2 * torch.rand(T, H, 1, generator=gen))   # |k|^2 up to 1.96
        g = g / 16
    elif kind == "like keys":   # along one direction either way: rows of Tm far from the identity's
        k = torch.nn.functional.normalize(k + 2 * randn(1, H, K) * K ** -0.5 * randn(T, H, 1).sign(), dim=-1)
        g, beta = g / 256, 0.5 + 0.4 * beta
    elif kind == "growing":   # up and down, by about e over 300 rows
        g = 0.3 * randn(T, H)
        g = g - g.mean(0) + 0.004
    x = [q.to(dtype), k.to(dtype), randn(T, H, V).to(dtype), g, beta]
    return x, 0.5 * randn(H, K, V), randn(T, H, V).to(dtype), randn(H, K, V), K ** -0.5


def rms(x):
    return float(x.square().mean().sqrt())


def bounds(x, s0, do, dht, scale):
    """Results in 64 bits, and how far each may be off (root mean square)."""
    def run(hook):
        o, ht, saved = form.forward(*x, scale, s0, hook=hook)
        return (o, ht, *form.backward(saved, scale, do, dht, hook=hook))
    ref = run(form.exact)
    noisy = [run(form.roundings(seed)) for seed in range(3)]
    return ref, [(sum(rms(n[i] - r) ** 2 for n in noisy) / len(noisy)) ** 0.5 for i, r in enumerate(ref)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("K,V", SIZES)
@pytest.mark.parametrize("kind", CASES)
def test_as_good_as_fp32(dev, kind, dtype, K, V):
    compare(dev, dtype, *case(kind, dtype, K, V))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,K,V", [(torch.float32, 64, 64), (torch.bfloat16, 128, 32), (torch.float16, 32, 64)])
@pytest.mark.parametrize("kind", ["long memory", "growing"])
def test_segments_are_as_good(dev, kind, dtype, K, V):
    """Five segments, three of them carried over by their maps."""
    compare(dev, dtype, *case(kind, dtype, K, V, T=1200))


def compare(dev, dtype, x, s0, do, dht, scale):
    from ssla_amd.delta import chunk_gated_delta
    ref, tol = bounds(x, s0, do, dht, scale)
    leaves = [t.to(dev).requires_grad_() for t in (*x, s0[None])]
    o, ht = chunk_gated_delta(*leaves[:5], torch.tensor([0, do.shape[0]], device=dev), scale=scale, initial_state=leaves[5],
                              output_final_state=True)
    grads = torch.autograd.grad((o, ht), leaves, (do.to(dev), dht[None].to(dev)))
    got = (o.detach(), ht.detach()[0], *grads[:5], grads[5][0])
    for name, a, r, t in zip(("o", "ht", *NAMES), got, ref, tol):
        if a.dtype != torch.float32:
            t = t + HALF[dtype] * rms(r) + (2.0 ** -15 * rms(r) if name == "o" else 0.0)
        off = rms(a.double().cpu() - r)
        assert off <= t, f"{name}: {off:.3g}, bound {t:.3g}, of {rms(r):.3g}"


@pytest.mark.gpu
@pytest.mark.parametrize("total", [63.0, 87.0])
def test_gates_up_to_the_stated_sum(dev, total):
    """Consecutive positive gates from a state of zeros, and back again.  Up to 64 in
    sum every token is as near as its state's size allows (its o is scale S^T q: off
    by at most the bound of test_gpu_delta_chunk, (K + 256) T half steps, of scale sum
    |q| max |S|); up to 88 values are finite.  (A decay of e^-64 = 2^-92.3 has a third
    part of 2^-108 or more, of e^-87 = 2^-125.5 one below 2^-126, the smallest normal
    number, which counts as 0 in the products.)"""
    from ssla_amd.delta import _chunk_fwd, fused_recurrent_gated_delta
    K = V = 32
    x, _, _, _, scale = case("fading", torch.float32, K, V, T=90)
    q, k, v, g, beta = x
    g[:] = -0.01
    g[2:8], g[20:26] = total / 6, -total / 6
    g[64:70], g[75:81] = total / 6, -total / 6
    S, ref, tol = torch.zeros(H, K, V, dtype=torch.float64), [], []
    for t in range(90):
        o, S, _ = form.forward(*(a[t:t + 1] for a in x), scale, S)
        ref.append(o)
        tol.append((K + 256) * 90 * 2.0 ** -24 * scale * q[t].double().abs().sum(-1) * S.abs().amax((1, 2)))
    ref, tol = torch.cat(ref), torch.stack(tol)[..., None]
    d, cu = [t.to(dev) for t in x], torch.tensor([0, 90], device=dev)
    chunks, tokens = _chunk_fwd(*d, cu, scale, None, False)[0], fused_recurrent_gated_delta(*d, cu, scale=scale)[0]
    assert torch.isfinite(chunks).all()
    for o in (tokens, chunks) if total <= 64 else (tokens,):
        err = (o.double().cpu() - ref).abs()
        assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.gpu
@pytest.mark.parametrize("power", [-90, 90])
@pytest.mark.parametrize("K,V", [(64, 64), (32, 20)])
def test_small_and_large_values(dev, power, K, V):
    """The rule is linear in v: values 2^power times as large give results that are,
    bit for bit (dv apart, which v does not enter)."""
    from ssla_amd.delta import chunk_gated_delta
    x, _, do, _, scale = case("long memory", torch.float32, K, V, T=600)

    def run(v):
        leaves = [t.to(dev).requires_grad_() for t in (x[0], x[1], v, x[3], x[4])]
        o, ht = chunk_gated_delta(*leaves, torch.tensor([0, 600], device=dev), scale=scale, output_final_state=True)
        dq, dk, dv, dg, db = torch.autograd.grad(o, leaves, do.to(dev))
        return [t.detach() for t in (o, ht, dq, dk, dg, db)], dv

    (one, dv1), (other, dv2) = run(x[2]), run(x[2] * 2.0 ** power)
    assert torch.equal(dv1, dv2)
    for name, a, b in zip(("o", "ht", "dq", "dk", "dg", "dbeta"), one, other):
        assert torch.equal(a * 2.0 ** power, b), name
