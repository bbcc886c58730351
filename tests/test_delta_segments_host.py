"""How the chunked delta rule cuts a batch, seen through the size of what its
forward leaves to its backward (no GPU needed)."""
import pytest

from ssla_amd import _lib

ROWS = 64


def inner_segments(n, T, H=1, K=64, V=64):
    """The segments with a successor that a batch of these sizes can have."""
    size = _lib.load().ssla_gated_delta_chunk_segments_size(n, T, H, K, V)
    one = K * V * 4 * H + 3 * K * K * 2 * H   # (K a power of two from 32 on, H K V of whole 256 bytes)
    assert size % one == 0
    return size // one


@pytest.mark.parametrize("H,K,V", [(1, 64, 64), (2, 64, 64), (1, 128, 128), (4, 32, 16)])
@pytest.mark.parametrize("T", [16384, 65536, 262144, 1 << 20])
def test_many_sequences_do_not_cut_one_finer(T, H, K, V):
    """However many short or empty sequences lie beside it, a long one is cut into
    at most 128 segments, or into what it would be cut into alone, whichever is
    more: the fold steps over them one after the other."""
    alone = inner_segments(1, T, H, K, V)
    for n in (2, 8, 64, 1000, 100000):
        assert inner_segments(n, T, H, K, V) <= max(alone, 128), n


def test_segments_of_ordinary_batches():
    """Chunks of a segment, as they were measured: 8 sequences of 4,096 rows of 8 heads 8,
    12 in 8,209 rows of 4 heads 4, 21 in 16,411 rows of 4 heads with 128 columns 5, one
    of 65,536 rows of 4 heads with 128 columns 16."""
    for n, T, H, V, per in ((8, 32768, 8, 64, 8), (12, 8209, 4, 64, 4), (1, 65536, 4, 128, 16), (21, 16411, 4, 128, 5)):
        assert inner_segments(n, T, H, 64, V) == (T - 1) // (per * ROWS), (n, T)
