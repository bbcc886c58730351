"""Refusals of the gated recurrence and its single tokens, before any device work (no
GPU needed)."""
import pytest
import torch
from torch.autograd import forward_ad

from ssla_amd import _lib


def test_scan_entries_refuse():
    lib = _lib.load()

    def fwd(n=1, T=4, C=8, gate=0, cu=8, ld=8, dt=0, dtg=0):
        return lib.ssla_gated_scan_fwd(None, ld, None, ld, None, 0, cu, n, T, C, gate, None, None, None, None, dt, dtg, None,
                                       0, None)

    def bwd(n=1, T=4, C=8, gate=0, cu=8, ld=8, dt=0, dtg=0):
        return lib.ssla_gated_scan_bwd(None, ld, None, ld, None, 0, cu, n, T, C, gate, None, None, None, None, None, None,
                                       None, None, dt, dtg, None, 0, None)

    def step(n=1, T=4, C=8, gate=0, cu=8, ld=8, dt=0, dtg=0):
        return lib.ssla_sparse_gated_step(cu, T if n >= 0 else n, None, ld, None, ld, None, 0, None, 5, C, gate, None, None,
                                          dt, dtg, None)

    for f in (fwd, bwd, step):
        for bad in (dict(n=-1), dict(T=-1), dict(C=0), dict(gate=3), dict(gate=-1), dict(ld=7)):
            assert f(**bad) == _lib.SSLA_ERR_ARG, (f, bad)
        for bad in (dict(dt=3, dtg=3), dict(dt=0, dtg=1), dict(dt=1, dtg=2), dict(dt=2, dtg=1)):
            assert f(**bad) == _lib.SSLA_ERR_DTYPE, (f, bad)
        assert f() == _lib.SSLA_ERR_ARG                       # null tensors
    for f in (fwd, bwd):
        assert f(cu=None) == _lib.SSLA_ERR_ARG
        assert f(T=1 << 34, C=1 << 10, ld=1 << 10) == _lib.SSLA_ERR_UNSUPPORTED
        assert f(ld=(1 << 20) + 1) == _lib.SSLA_ERR_UNSUPPORTED      # (offsets in a tile of rows are 32 bits)
        assert f(C=(1 << 20) + 1, ld=1 << 21) == _lib.SSLA_ERR_UNSUPPORTED
    size = lib.ssla_gated_scan_workspace_size(100000, 64)
    for f in (lib.ssla_gated_scan_fwd, lib.ssla_gated_scan_bwd):      # a long sequence needs its workspace (checked before any launch)
        for ws, n in ((None, size), (16, 1000), (8, size)):
            if f is lib.ssla_gated_scan_fwd:
                st = f(16, 64, 16, 64, None, 0, 16, 1, 100000, 64, 0, None, 16, None, None, 0, 0, ws, n, None)
            else:
                st = f(16, 64, 16, 64, None, 0, 16, 1, 100000, 64, 0, None, 16, 16, None, 16, 16, None, None, 0, 0, ws, n, None)
            assert st == _lib.SSLA_ERR_WORKSPACE, (ws, n)
    assert step(T=0) == _lib.SSLA_OK
    assert lib.ssla_sparse_gated_step(8, 1, None, 8, None, 8, None, 0, None, -1, 8, 0, None, None, 0, 0, None) == _lib.SSLA_ERR_ARG
    for size in (lib.ssla_gated_scan_workspace_size, lib.ssla_gated_scan_keep_size):
        assert size(-1, 8) == 0 and size(0, 8) == 0 and size(100, 0) == 0
    assert 0 < lib.ssla_gated_scan_keep_size(100, 8) < lib.ssla_gated_scan_keep_size(1000, 8)


def _forms():
    from ssla_amd.scan import gated_scan, sparse_gated_step
    return [lambda u, g, **k: gated_scan(u, g, torch.tensor([0, 4]), **k),
            lambda u, g, **k: sparse_gated_step(torch.arange(4), u, g, torch.zeros(9, 6), **k)]


@pytest.mark.parametrize("form", range(2))
def test_functions_refuse(form):
    f = _forms()[form]
    x = torch.zeros(4, 6)
    with pytest.raises(ValueError, match="device tensors"):
        f(x, x)
    for u, g, q in ((x, x[:3], None), (x, x[:, :5], None), (x[None], x[None], None), (x, x, x[:, :5]), (x[:, :0], x[:, :0], None)):
        with pytest.raises(ValueError):
            f(u, g, q=q)
    with pytest.raises(ValueError, match="gate"):
        f(x, x, gate="tanh")
    for u, g, q in ((x.double(), x, None), (x, x.int(), None), (x, x, x.half())):
        with pytest.raises(TypeError):
            f(u, g, q=q)
    wide = torch.zeros(1, 1).expand(4, (1 << 20) + 1)
    with pytest.raises(NotImplementedError, match="channels"):
        f(wide, wide)
    for i in range(3):
        with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
            args = [x, x, x]
            args[i] = forward_ad.make_dual(x, torch.ones_like(x))
            f(args[0], args[1], q=args[2])


def test_scan_refuses():
    from ssla_amd.scan import gated_scan
    x = torch.zeros(4, 6)
    with pytest.raises(ValueError, match="device tensors"):
        gated_scan(x, x, torch.tensor([0, 4]), initial_state=torch.zeros(1, 6))
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        gated_scan(x, x, torch.tensor([0, 4]), initial_state=forward_ad.make_dual(torch.zeros(1, 6), torch.ones(1, 6)))


def test_tables_refuse():
    from ssla_amd.scan import sparse_gated_step
    x = torch.zeros(4, 6)
    for state in (torch.zeros(9, 7), torch.zeros(9, 6).half(), torch.zeros(6, 9).t(), torch.zeros(9, 6, 1)):
        with pytest.raises(ValueError, match="contiguous fp32"):
            sparse_gated_step(torch.arange(4), x, x, state)


def test_entries_refuse_more_sequences_than_they_count():
    lib = _lib.load()
    n = (1 << 30) + 1
    assert lib.ssla_gated_scan_fwd(16, 8, 16, 8, None, 0, 16, n, 4, 8, 0, None, 16, None, None, 0, 0, None, 0,
                                   None) == _lib.SSLA_ERR_UNSUPPORTED
    assert lib.ssla_gated_scan_bwd(16, 8, 16, 8, None, 0, 16, n, 4, 8, 0, None, 16, 16, None, 16, 16, None, None, 0, 0, None, 0,
                                   None) == _lib.SSLA_ERR_UNSUPPORTED
    assert lib.ssla_sparse_gated_step(16, n, 16, 8, 16, 8, None, 0, 16, 5, 8, 0, 16, None, 0, 0, None) == _lib.SSLA_ERR_UNSUPPORTED


def test_entries_refuse_more_workgroups_than_a_launch_holds():
    """A launch's threads are counted in 32 bits: 2^32 rows of one channel are 2^23 tiles of
    512 rows and 512 threads (twice that in the backward), one more than it holds."""
    lib = _lib.load()
    T = 1 << 32
    size = lib.ssla_gated_scan_workspace_size(T, 1)
    assert lib.ssla_gated_scan_fwd(16, 1, 16, 1, None, 0, 16, 1, T, 1, 0, None, 16, None, None, 1, 1, 16, size,
                                   None) == _lib.SSLA_ERR_UNSUPPORTED
    assert b"workgroups" in lib.ssla_last_error()
    assert lib.ssla_gated_scan_bwd(16, 1, 16, 1, None, 0, 16, 1, T // 2, 1, 0, None, 16, 16, None, 16, 16, None, None, 1, 1, 16, size,
                                   None) == _lib.SSLA_ERR_UNSUPPORTED
    assert b"workgroups" in lib.ssla_last_error()
    n = 1 << 30   # single tokens, a thread a channel of 5: 5 2^30 threads
    assert lib.ssla_sparse_gated_step(16, n, 16, 5, 16, 5, None, 0, 16, 5, 5, 0, 16, None, 0, 0,
                                      None) == _lib.SSLA_ERR_UNSUPPORTED
    assert b"workgroups" in lib.ssla_last_error()
