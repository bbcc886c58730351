"""Refusals of ssla_gated_delta_mixed_fwd, before any device work (no GPU needed),
and the slots of its workspace."""
from ssla_amd import _lib


def test_entry_refuses():
    lib = _lib.load()
    size = lib.ssla_gated_delta_mixed_workspace_size

    def call(n=1, T=4, Hk=1, H=1, K=16, V=16, cu=8, dtype=0, ws=None, nbytes=0):
        return lib.ssla_gated_delta_mixed_fwd(None, None, None, None, None, cu, n, T, Hk, H, K, V, 1.0, None, None, None,
                                              dtype, ws, nbytes, None)

    for bad in (dict(n=-1), dict(T=-1), dict(Hk=0), dict(H=0), dict(Hk=2, H=3), dict(K=0), dict(V=0)):
        assert call(**bad) == _lib.SSLA_ERR_ARG, bad
        assert b"gated_delta_mixed_fwd: bad sizes" in lib.ssla_last_error()
    assert call(K=129) == _lib.SSLA_ERR_UNSUPPORTED
    assert call(cu=None) == _lib.SSLA_ERR_ARG and call() == _lib.SSLA_ERR_ARG
    assert call(n=0) == _lib.SSLA_OK
    assert call(T=0) == _lib.SSLA_ERR_WORKSPACE
    assert call(T=0, ws=16, nbytes=size(0, 1, 16, 16) - 1) == _lib.SSLA_ERR_WORKSPACE
    assert call(T=0, ws=8, nbytes=size(0, 1, 16, 16)) == _lib.SSLA_ERR_WORKSPACE
    assert call(T=0, ws=16, nbytes=size(0, 1, 16, 16), dtype=9) == _lib.SSLA_ERR_DTYPE
    assert call(T=0, V=(1 << 20) + 1, ws=16) == _lib.SSLA_ERR_UNSUPPORTED
    assert size(64, 1, 129, 16) == 0 and size(-1, 1, 16, 16) == 0
    assert 0 < size(0, 1, 16, 16) < size(640, 1, 16, 16) < size(640, 2, 16, 16)


def test_slots_of_long_sequences_are_apart():
    """Where only sequences of more than m rows own slots (start // m + piece, pieces
    of 2 m rows or more), no two pieces share one, the sequence that the search
    finds for a slot (the last that starts at or before it) is its owner, and no
    slot lies past T // m."""
    import random
    rng = random.Random(1)
    for m, piece in ((32, 64), (64, 256), (64, 704)):
        for _ in range(300):
            lens = [rng.choice((0, 1, m - 1, m, rng.randrange(m), 65, m + 1, 2 * m, rng.randrange(65, 2000)))
                    for _ in range(rng.randrange(1, 40))]
            bos = [sum(lens[:n]) for n in range(len(lens))]
            T, owner = sum(lens), {}
            for n, rows in enumerate(lens):
                if rows > 64:
                    for j in range(-(-rows // piece)):
                        slot = bos[n] // m + j
                        assert slot not in owner and slot <= T // m
                        owner[slot] = n
            for slot, n in owner.items():
                assert max(i for i in range(len(lens)) if bos[i] // m <= slot) == n
