"""The form that the group norm's bounds come from is the definition, and mistakes of
the joins and sums are far outside the bounds (no GPU needed)."""
import pytest
import torch

from oracle.delta import group_norm
from tests import norm_form as form
from tests.test_gpu_group_norm_slices import EPS, SLICES, bounds, inputs, rms


@pytest.mark.parametrize("act", [None, "relu", "silu"])
def test_is_the_definition(act):
    x, w, b, dy = inputs((3, 50, 24), 4, torch.float32, act)
    leaves = [t.double().requires_grad_() for t in (x, w, b)]
    y = group_norm(leaves[0], 4, *leaves[1:], EPS, act)
    want = (y.detach(), *torch.autograd.grad(y, leaves, dy.double()))
    for a, r in zip(form.run(x, 4, w, b, EPS, act, dy), want):
        assert float((a - r).abs().max()) <= 1e-10 * float(r.abs().max())


@pytest.mark.parametrize("act", [None, "relu", "silu"])
@pytest.mark.parametrize("shape", [s for s in SLICES if s[1] * s[2] < 400000 or s[2] == 64])
def test_bounds_would_notice(shape, act):
    """Per mistake, the result that must be out of its bound."""
    x, w, b, dy = inputs(shape[:3], shape[3], torch.float32, act)
    G, L = shape[3], shape[1]
    ref, tol = bounds(x, G, w, b, act, dy)
    last = slice(L - min(L // 4, 128), L)   # a slice
    for lost, where in ((("moments", last), (0, 1)), ("between", (0, 1)), (("sums", last), (1,)), ("means", (1,)),
                        (("columns", last), (2, 3))):
        bad = form.run(x, G, w, b, EPS, act, dy, lost=lost)
        for i in where:
            assert rms(bad[i] - ref[i]) > 8 * tol[i], (lost, i)
    for i in (1, 2, 3):
        assert rms(ref[i]) > 1000 * tol[i]
