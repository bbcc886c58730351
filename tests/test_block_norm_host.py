"""Refusals of the norms around a block and the counter-based dropout, before any device
work (no GPU needed)."""
import pytest
import torch
from torch.autograd import forward_ad

from ssla_amd import _lib


def test_gated_entries_refuse():
    lib = _lib.load()

    def fwd(N=2, C=8, G=2, kind=0, act=2, ld=8, dt=0):
        return lib.ssla_gated_norm_fwd(None, ld, None, ld, N, C, G, kind, None, None, 1e-5, act, None, dt, None)

    def bwd(N=2, C=8, G=2, kind=0, act=2, ld=8, dt=0):
        return lib.ssla_gated_norm_bwd(None, None, ld, None, ld, N, C, G, kind, None, None, 1e-5, act, None, None, None, None,
                                       dt, None, 0, None)

    for f in (fwd, bwd):
        for bad in (dict(N=-1), dict(C=0), dict(G=0), dict(G=3), dict(kind=2), dict(kind=-1), dict(act=0), dict(act=4), dict(ld=7)):
            assert f(**bad) == _lib.SSLA_ERR_ARG, (f, bad)
        assert f(dt=3) == _lib.SSLA_ERR_DTYPE
        assert f() == _lib.SSLA_ERR_ARG                       # null tensors
        assert f(C=8193, G=1, ld=8193) == _lib.SSLA_ERR_UNSUPPORTED
        assert f(N=1 << 38, C=8192, G=1, ld=8192) == _lib.SSLA_ERR_UNSUPPORTED
        assert f(N=0) == _lib.SSLA_OK
    size = lib.ssla_gated_norm_bwd_workspace_size
    assert size(0, 8, 2) == 0 and size(8, 8, 3) == 0 and 0 < size(100, 64, 2) <= size(100000, 64, 2)
    st = lib.ssla_gated_norm_bwd(16, 16, 8, 16, 8, 100, 8, 2, 0, None, None, 1e-5, 2, None, None, 16, None, 0, 16,
                                 size(100, 8, 2) - 1, None)
    assert st == _lib.SSLA_ERR_WORKSPACE


def test_residual_entries_refuse():
    lib = _lib.load()

    def fwd(N=2, C=8, kind=0, post=0, w2=None, p=0.0, seed=None, dt=0, dtr=0):
        return lib.ssla_residual_norm_fwd(None, None, N, C, kind, None, None, 1e-5, 1.0, None, post, w2, p, seed, 0, None, None,
                                          dt, dtr, None)

    def bwd(N=2, C=8, kind=0, post=0, w2=None, p=0.0, seed=None, dt=0, dtr=0):
        return lib.ssla_residual_norm_bwd(None, None, None, None, N, C, kind, None, 1e-5, 1.0, None, post, w2, p, seed, 0, None,
                                          None, None, None, None, None, dt, dtr, None, 0, None)

    for f in (fwd, bwd):
        for bad in (dict(N=-1), dict(C=0), dict(kind=2), dict(w2=16), dict(p=-0.1), dict(p=1.1), dict(p=float("nan")), dict(p=0.5)):
            assert f(**bad) == _lib.SSLA_ERR_ARG, (f, bad)
        for bad in (dict(dt=3, dtr=3), dict(dt=0, dtr=1), dict(dt=1, dtr=2)):
            assert f(**bad) == _lib.SSLA_ERR_DTYPE, (f, bad)
        assert f() == _lib.SSLA_ERR_ARG                       # null tensors
        assert f(C=8193) == _lib.SSLA_ERR_UNSUPPORTED
        assert f(N=0) == _lib.SSLA_OK
    size = lib.ssla_residual_norm_bwd_workspace_size
    assert size(0, 8) == 0 and 0 < size(100, 64) <= size(100000, 64)
    st = lib.ssla_residual_norm_bwd(16, None, 16, 16, 100, 8, 0, None, 1e-5, 1.0, None, 0, None, 0.0, None, 0, None, None, 16, None,
                                    None, None, 0, 0, None, 0, None)
    assert st == _lib.SSLA_ERR_WORKSPACE


def test_dropout_entry_refuses():
    f = _lib.load().ssla_counter_dropout
    for n, p in ((-1, 0.5), (4, -0.5), (4, 1.5), (4, float("nan"))):
        assert f(None, n, p, None, 0, None, 0, None) == _lib.SSLA_ERR_ARG
    assert f(None, 4, 0.5, None, 0, None, 3, None) == _lib.SSLA_ERR_DTYPE
    assert f(None, 4, 0.5, None, 0, None, 0, None) == _lib.SSLA_ERR_ARG
    assert f(None, 0, 0.5, None, 0, None, 0, None) == _lib.SSLA_OK


def test_gated_refuses():
    from ssla_amd.norm import gated_norm
    x = torch.zeros(3, 8)
    with pytest.raises(ValueError, match="device tensors"):
        gated_norm(x, x, 2)
    for args, kw in (((x, x[:2]), {}), ((x, x[:, :4]), {}), ((torch.tensor(1.0),) * 2, {}), ((x[:, :0], x[:, :0]), {}),
                     ((x, x, 3), {}), ((x, x, 0), {}), ((x, x), dict(activation="relu")), ((x, x), dict(kind="batch")),
                     ((x, x), dict(eps=-1.0)), ((x, x), dict(eps=float("nan"))), ((x, x), dict(weight=torch.zeros(7))),
                     ((x, x), dict(bias=torch.zeros(8, dtype=torch.int32)))):
        with pytest.raises(ValueError):
            gated_norm(*args, **kw)
    for a, b in ((x.double(), x.double()), (x, x.half())):
        with pytest.raises(TypeError):
            gated_norm(a, b)
    with pytest.raises(NotImplementedError, match="8192"):
        gated_norm(torch.zeros(1, 8193), torch.zeros(1, 8193))


def test_residual_refuses():
    from ssla_amd.norm import residual_norm
    x = torch.zeros(3, 8)
    with pytest.raises(ValueError, match="device tensors"):
        residual_norm(x, x)
    for kw in (dict(residual=x[:2]), dict(weight=torch.zeros(7)), dict(bias=torch.zeros(9)), dict(scale=torch.zeros(1)),
               dict(post_weight=torch.zeros(8)), dict(kind="batch"), dict(eps=-1.0), dict(p=1.5), dict(p="x")):
        with pytest.raises(ValueError):
            residual_norm(x, kw.pop("residual", x), **kw)
    for a, b in ((x.double(), x.double()), (x, x.half()), (x.half(), x.bfloat16())):
        with pytest.raises(TypeError):
            residual_norm(a, b)
    with pytest.raises(NotImplementedError, match="8192"):
        residual_norm(torch.zeros(1, 8193), torch.zeros(1, 8193))


def test_dropout_refuses():
    from ssla_amd.dropout import counter_dropout
    x = torch.zeros(3, 8)
    with pytest.raises(ValueError, match="device tensors"):
        counter_dropout(x, 0.5, 1)
    for p in (-0.1, 1.1, float("nan"), None):
        with pytest.raises(ValueError, match="p must"):
            counter_dropout(x, p, 1)
    with pytest.raises(TypeError):
        counter_dropout(x.double(), 0.5, 1)


def test_seeds_refuse():
    from ssla_amd.dropout import _seed
    cpu = torch.device("cpu")
    for seed, sub in ((torch.zeros(2, dtype=torch.int64), 0), (torch.zeros(1, dtype=torch.int32), 0), (1.5, 0), (None, 0), (1 << 63, 0),
                      (1, -1), (1, 1 << 32), (1, 1.0)):
        with pytest.raises(ValueError):
            _seed("f", seed, sub, cpu)
    with pytest.raises(ValueError, match="must lie on"):
        _seed("f", torch.zeros(1, dtype=torch.int64), 0, torch.device("cuda:0"))
    assert int(_seed("f", -5, 0, cpu)) == -5


def test_tangents_are_refused():
    from ssla_amd.dropout import counter_dropout
    from ssla_amd.norm import gated_norm, residual_norm
    x, v = torch.zeros(3, 8), torch.zeros(8)
    forms = [(lambda *t: gated_norm(t[0], t[1], 2, t[2], t[3]), [x, x, v, v]),
             (lambda *t: residual_norm(*t[:4], scale=t[4], post_norm=True, post_weight=t[5]), [x, x, v, v, v, v]),
             (lambda t: counter_dropout(t, 0.5, 1), [x])]
    for f, args in forms:
        for i in range(len(args)):
            with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
                t = list(args)
                t[i] = forward_ad.make_dual(t[i], torch.ones_like(t[i]))
                f(*t)


def test_probabilities_are_rounded_once():
    """p counts in steps of 2^-16, t = round(p 2^16): one beside the middle of two steps is not
    rounded to fp32, which holds the middle, before."""
    from ssla_amd.dropout import _p
    for p in (19660.5 / 65536 + 1e-10, 19661.5 / 65536 - 1e-10, 0.1, 0.0, 1.0, 2.0 ** -17 + 1e-12, 2.0 ** -18, 1 - 1e-9):
        t = round(p * 65536)
        assert torch.tensor(_p("f", p), dtype=torch.float32).double().item() * 65536 == t, p
