"""The chunk form that the precision tests model roundings in: it is the definition,
and its model of the kernels' roundings is well below what a lost part of an operand
does (no GPU needed)."""
import pytest
import torch

from oracle.delta import gated_delta
from tests import delta_chunk_form as form
from tests.test_gpu_delta_precision import CASES, NAMES, SIZES, bounds, case, rms


@pytest.mark.parametrize("kind", CASES)
def test_is_the_definition(kind):
    x, s0, do, dht, scale = case(kind, torch.float32, 24, 16)
    T = do.shape[0]
    leaves = [t.double().requires_grad_() for t in (*x, s0)]
    o, ht = gated_delta(*leaves[:5], [T], scale, leaves[5][None])
    want = (o, ht[0], *torch.autograd.grad([o, ht], leaves, [do.double(), dht.double()[None]]))
    fo, fs, saved = form.forward(*x, scale, s0)
    for name, a, r in zip(("o", "ht", *NAMES), (fo, fs, *form.backward(saved, scale, do, dht)), want):
        assert float((a - r).abs().max()) <= 1e-9 * max(1.0, float(r.abs().max())), name


def test_bounds_would_notice_a_lost_part():
    """Leaving out the third part of any operand of the walks passes the bound of
    some result in some case."""
    most = {}
    for K, V in SIZES:
        for kind in CASES:
            x, s0, do, dht, scale = case(kind, torch.float32, K, V)
            ref, tol = bounds(x, s0, do, dht, scale)
            for which in ("S operand", "X operand", "Tm operand", "u operand", "D operand", "dX operand"):
                lose = form.losing(which)
                o, ht, saved = form.forward(*x, scale, s0, hook=lose)
                bad = (o, ht, *form.backward(saved, scale, do, dht, hook=lose))
                most[which] = max(most.get(which, 0), *(rms(a - r) / t for a, r, t in zip(bad, ref, tol)))
    assert min(most.values()) > 2.8, most
