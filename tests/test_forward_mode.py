"""Forward-mode differentiation is refused: a kernel that is handed the primal's
pointer would drop the tangent without a word.  (Before any device work: no GPU
needed.)"""
import pytest
import torch
from torch.autograd import forward_ad

T, H, K, V = 4, 2, 16, 8


def _calls():
    from ssla_amd import delta, norm
    cu, at, state = torch.tensor([0, T]), torch.arange(T), torch.zeros(5, H, K, V)
    rule = [torch.zeros(T, 1, K), torch.zeros(T, 1, K), torch.zeros(T, H, V), torch.zeros(T, H), torch.zeros(T, H)]
    h0 = torch.zeros(1, H, K, V)
    return {
        "chunk": (lambda *x: delta.chunk_gated_delta(*x[:5], cu, initial_state=x[5]), [*rule, h0]),
        "recurrent": (lambda *x: delta.fused_recurrent_gated_delta(*x[:5], cu, initial_state=x[5]), [*rule, h0]),
        "scan": (lambda *x: delta.sparse_delta_scan(*x[:5], cu, torch.tensor([1]), x[5]), [*rule, state]),
        "step": (lambda *x: delta.sparse_delta_step(at, *x[:5], x[5]), [*rule, state]),
        "norm": (lambda x, w, b: norm.group_norm_act(x, 2, w, b), [torch.zeros(3, 8), torch.ones(8), torch.zeros(8)]),
    }


@pytest.mark.parametrize("name", ["chunk", "recurrent", "scan", "step", "norm"])
def test_tangents_are_refused(name):
    f, args = _calls()[name]
    for i in range(len(args)):
        with forward_ad.dual_level():
            x = list(args)
            x[i] = forward_ad.make_dual(x[i], torch.ones_like(x[i]))
            for off in (False, True):
                with torch.set_grad_enabled(not off), pytest.raises(NotImplementedError, match="forward-mode"):
                    f(*x)
    with forward_ad.dual_level(), pytest.raises(ValueError, match="device tensors"):   # (no tangent: the next check)
        f(*args)


@pytest.mark.parametrize("name", ["chunk", "step", "norm"])
def test_jvp_is_refused(name):
    f, args = _calls()[name]
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(f, tuple(args), tuple(torch.ones_like(a) for a in args))
