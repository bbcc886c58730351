"""Refusals of the gated delta rule and the group norm, before any device work
(no GPU needed): the C entry points' argument checks and the Python functions'
shape and type checks."""
import pytest
import torch

from ssla_amd import _lib


def test_recurrent_entry_refuses():
    f = _lib.load().ssla_gated_delta_recurrent

    def call(n=1, T=4, Hk=1, H=1, K=16, V=16, cu=None, idx=None, rows=0, dtype=0):
        return f(None, None, None, None, None, cu, n, T, Hk, H, K, V, 1.0, None, None, None, idx, rows, None, dtype, None)

    for bad in (dict(n=-1), dict(T=-1), dict(Hk=0), dict(H=0), dict(Hk=2, H=3), dict(K=0), dict(V=0)):
        assert call(**bad) == _lib.SSLA_ERR_ARG, bad
        assert b"bad sizes" in _lib.load().ssla_last_error()
    assert call(K=257) == _lib.SSLA_ERR_UNSUPPORTED
    assert call() == _lib.SSLA_ERR_ARG                      # no offsets and T != n
    assert call(T=1) == _lib.SSLA_ERR_ARG                   # null tensors
    assert call(T=0, cu=8, idx=8) == _lib.SSLA_ERR_ARG      # a site list without a table
    assert call(n=0) == _lib.SSLA_OK
    assert call(T=0, cu=8, dtype=7) == _lib.SSLA_ERR_DTYPE


def test_norm_entry_refuses():
    lib = _lib.load()

    def fwd(N=2, L=3, C=8, G=2, act=0, dtype=0):
        return lib.ssla_group_norm_fwd(None, N, L, C, G, None, None, 1e-5, act, None, None, dtype, None, 0, None)

    for bad in (dict(N=-1), dict(L=-1), dict(C=0), dict(G=0), dict(G=3), dict(act=3), dict(act=-1)):
        assert fwd(**bad) == _lib.SSLA_ERR_ARG, bad
    assert fwd() == _lib.SSLA_ERR_ARG                       # null tensors
    assert fwd(N=0) == _lib.SSLA_OK and fwd(L=0) == _lib.SSLA_OK
    assert fwd(N=1 << 31) == _lib.SSLA_ERR_UNSUPPORTED
    bwd = lib.ssla_group_norm_bwd
    assert bwd(None, None, None, 2, 3, 8, 3, None, None, 0, None, None, None, 0, None, 0, None) == _lib.SSLA_ERR_ARG
    assert bwd(None, None, None, 2, 3, 8, 2, None, None, 0, None, None, None, 0, None, 0, None) == _lib.SSLA_ERR_ARG


def _args(T=4, Hk=1, H=2, K=16, V=8, dt=torch.float32):
    return [torch.zeros(T, Hk, K, dtype=dt), torch.zeros(T, Hk, K, dtype=dt), torch.zeros(T, H, V, dtype=dt),
            torch.zeros(T, H), torch.zeros(T, H)]


def _forms():
    from ssla_amd import delta
    cu = torch.tensor([0, 4])
    state = torch.zeros(5, 2, 16, 8)
    return [lambda *x: delta.fused_recurrent_gated_delta(*x, cu),
            lambda *x: delta.sparse_delta_scan(*x, cu, torch.tensor([1]), state),
            lambda *x: delta.sparse_delta_step(torch.arange(4), *x, state)]


@pytest.mark.parametrize("form", range(3))
def test_rule_refuses(form):
    f = _forms()[form]
    with pytest.raises(ValueError, match="device tensors"):
        f(*_args())
    for at, shape in ((0, (4, 16)), (1, (4, 1, 12)), (2, (3, 2, 8)), (3, (4, 1)), (4, (4, 2, 1)), (2, (4, 0, 8))):
        x = _args()
        x[at] = torch.zeros(shape)
        with pytest.raises(ValueError):
            f(*x)
    x = _args(Hk=2)
    x[2] = torch.zeros(4, 3, 8)
    x[3] = x[4] = torch.zeros(4, 3)
    with pytest.raises(ValueError, match="share"):
        f(*x)
    x = _args()
    x[1] = x[1].half()
    with pytest.raises(TypeError):
        f(*x)
    with pytest.raises(TypeError):
        f(*_args(dt=torch.float64))
    x = _args()
    x[3] = x[3].int()
    with pytest.raises(TypeError):
        f(*x)


def test_tables_refuse():
    from ssla_amd.delta import sparse_delta_step
    for state in (torch.zeros(5, 2, 16, 9), torch.zeros(5, 2, 16, 8).half(), torch.zeros(5, 2, 8, 16).transpose(2, 3)):
        with pytest.raises(ValueError, match="contiguous fp32"):
            sparse_delta_step(torch.arange(4), *_args(), state)


def test_norm_refuses():
    from ssla_amd.norm import group_norm_act
    x = torch.zeros(2, 3, 8)
    with pytest.raises(ValueError, match="device tensors"):
        group_norm_act(x, 2)
    for bad in (dict(num_groups=3), dict(num_groups=0), dict(num_groups=2, activation="tanh"),
                dict(num_groups=2, weight=torch.zeros(7)), dict(num_groups=2, bias=torch.zeros(8, dtype=torch.int32)),
                dict(num_groups=2, eps=-1.0), dict(num_groups=2, eps=float("nan"))):
        with pytest.raises(ValueError):
            group_norm_act(x, **bad)
    with pytest.raises(ValueError):
        group_norm_act(torch.zeros(8), 2)
    with pytest.raises(TypeError):
        group_norm_act(x.double(), 2)


def test_chunk_entry_refuses():
    lib = _lib.load()

    def call(n=1, T=4, Hk=1, H=1, K=16, V=16, cu=8, dtype=0, ws=None, nbytes=0):
        return lib.ssla_gated_delta_chunk_fwd(None, None, None, None, None, cu, n, T, Hk, H, K, V, 1.0, None, None, None,
                                              None, dtype, ws, nbytes, None)

    for bad in (dict(n=-1), dict(T=-1), dict(Hk=0), dict(H=0), dict(Hk=2, H=3), dict(K=0), dict(V=0)):
        assert call(**bad) == _lib.SSLA_ERR_ARG, bad
    assert call(K=129) == _lib.SSLA_ERR_UNSUPPORTED
    assert call(cu=None) == _lib.SSLA_ERR_ARG and call() == _lib.SSLA_ERR_ARG
    assert call(n=0) == _lib.SSLA_OK
    size = lib.ssla_gated_delta_chunk_workspace_size
    assert call(T=0) == _lib.SSLA_ERR_WORKSPACE
    assert call(T=0, ws=16, nbytes=size(1, 0, 1, 16, 16) - 1) == _lib.SSLA_ERR_WORKSPACE
    assert call(T=0, ws=8, nbytes=size(1, 0, 1, 16, 16)) == _lib.SSLA_ERR_WORKSPACE
    assert call(T=0, ws=16, nbytes=size(1, 0, 1, 16, 16), dtype=9) == _lib.SSLA_ERR_DTYPE
    assert size(1, 64, 1, 129, 16) == 0 and size(-1, 64, 1, 16, 16) == 0
    assert 0 < size(1, 64, 1, 16, 16) < size(2, 64, 1, 16, 16) < size(2, 640, 1, 16, 16) < size(2, 640, 2, 16, 16)


def test_chunk_backward_entry_refuses():
    lib = _lib.load()

    def call(n=1, T=4, Hk=1, H=1, K=16, V=16, cu=8, dtype=0, ws=None, nbytes=0):
        return lib.ssla_gated_delta_chunk_bwd(None, None, None, None, None, cu, n, T, Hk, H, K, V, 1.0, None, None, None,
                                              None, None, None, None, None, None, None, dtype, ws, nbytes, None)

    for bad in (dict(n=-1), dict(T=-1), dict(Hk=0), dict(H=0), dict(Hk=2, H=3), dict(K=0), dict(V=0)):
        assert call(**bad) == _lib.SSLA_ERR_ARG, bad
    assert call(K=129) == _lib.SSLA_ERR_UNSUPPORTED
    assert call(cu=None) == _lib.SSLA_ERR_ARG and call() == _lib.SSLA_ERR_ARG
    assert call(T=0, dtype=9) == _lib.SSLA_ERR_DTYPE
    size = lib.ssla_gated_delta_chunk_bwd_workspace_size
    assert call(T=0) == _lib.SSLA_ERR_WORKSPACE
    assert call(T=0, ws=16, nbytes=size(1, 0, 1, 1, 16, 16) - 1) == _lib.SSLA_ERR_WORKSPACE
    assert size(1, 64, 1, 1, 129, 16) == 0 and size(1, 64, 2, 3, 16, 16) == 0
    assert size(1, 64, 2, 2, 16, 16) < size(1, 64, 1, 2, 16, 16)


def test_rows_too_wide_are_refused():
    """Offsets inside a block of rows, or inside a state, are 32 bits."""
    lib = _lib.load()
    for H, K, V in ((1 << 17, 64, 128), (1, 128, 1 << 22), (1, 1, (1 << 20) + 1)):
        assert lib.ssla_gated_delta_chunk_fwd(None, None, None, None, None, 8, 1, 0, 1, H, K, V, 1.0, None, None, None,
                                              None, 0, None, 0, None) == _lib.SSLA_ERR_UNSUPPORTED
        assert lib.ssla_gated_delta_chunk_bwd(None, None, None, None, None, 8, 1, 0, 1, H, K, V, 1.0, None, None, None, None,
                                              None, None, None, None, None, None, 0, None, 0, None) == _lib.SSLA_ERR_UNSUPPORTED
    for H, K, V in ((1 << 18, 64, 128), (1, 1, (1 << 20) + 1)):
        assert lib.ssla_gated_delta_recurrent(None, None, None, None, None, 8, 1, 0, 1, H, K, V, 1.0, None, None, None, None,
                                              0, None, 0, None) == _lib.SSLA_ERR_UNSUPPORTED
