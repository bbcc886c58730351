"""Site lists and offsets of the gated delta rule as the kernels get them (no GPU
needed)."""
import pytest
import torch

from ssla_amd.delta import _offsets, _sites


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int16, torch.int32, torch.int64, torch.uint32, torch.uint64])
def test_entries_outside_stay_outside(dtype):
    """What 32 bits do not hold must not become another site's number."""
    big = [e for e in ((1 << 32) + 1, (1 << 40), (1 << 63) + 1, (1 << 32) - 1, (1 << 31) + 2, -1, -(1 << 32) + 1)
           if torch.iinfo(dtype).min <= e <= torch.iinfo(dtype).max]
    got = _sites("f", torch.tensor([0, 1, 5] + big, dtype=dtype), 3 + len(big))
    assert got.dtype is torch.int32 and got[:3].tolist() == [0, 1, 5]
    assert all(e < 0 or e >= 0x7fffffff for e in got[3:].tolist())


def test_lists_that_are_not_integers_are_refused():
    for t in (torch.zeros(2), torch.zeros(2, dtype=torch.complex64)):
        with pytest.raises(ValueError, match="integers"):
            _sites("f", t, 2)
        with pytest.raises(ValueError, match="integers"):
            _offsets("f", t, torch.device("cpu"))
