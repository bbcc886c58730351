"""The definitions in oracle/block.py by other means (no GPU needed): the generator's
published answers, the recurrence's gradients by autograd, dropout's shares."""
import numpy as np
import pytest
import torch

from oracle import block


@pytest.mark.parametrize("counter,key,want", [
    ((0, 0, 0, 0), (0, 0), (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
    ((0xffffffff,) * 4, (0xffffffff,) * 2, (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
    ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0),
     (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1))])
def test_generator(counter, key, want):
    """Known answers published with the generator (Random123)."""
    assert tuple(block.philox(np.array([counter]), key)[0]) == want


def test_mask():
    n, p = 80000, 0.3
    keep = block.dropout_keep(n, p, 1234)
    # a share of n draws: five standard deviations
    assert abs(float(keep.double().mean()) - (1 - p)) <= 5 * (p * (1 - p) / n) ** 0.5
    assert torch.equal(block.dropout_keep(100, p, 1234, first=1003), keep[1003:1103])
    for other in (block.dropout_keep(n, p, 1235), block.dropout_keep(n, p, 1234, 1), block.dropout_keep(n, p, 1234 + (1 << 40))):
        both = float((keep & other).double().mean())
        assert abs(both - (1 - p) ** 2) <= 5 * (0.25 / n) ** 0.5
    assert block.dropout_keep(n, 0.0, 1).all() and not block.dropout_keep(n, 1.0, 1).any()
    assert torch.equal(block.dropout_keep(64, p, -1), block.dropout_keep(64, p, (1 << 64) - 1))


@pytest.mark.parametrize("gate", ["value", "log", "sigmoid"])
def test_recurrence(gate):
    gen = torch.Generator().manual_seed(0)
    lens, T, C = [5, 0, 3, 1], 9, 4
    u, g, q = (torch.randn(T, C, dtype=torch.float64, generator=gen, requires_grad=True) for _ in range(3))
    h0 = torch.randn(4, C, dtype=torch.float64, generator=gen, requires_grad=True)
    do, dht = torch.randn(T, C, dtype=torch.float64, generator=gen), torch.randn(4, C, dtype=torch.float64, generator=gen)
    a = {"value": g, "log": g.exp(), "sigmoid": g.sigmoid()}[gate]
    o, last, t = [], [], 0
    for n, rows in enumerate(lens):
        h = h0[n]
        for _ in range(rows):
            h = a[t] * h + u[t]
            o.append(q[t] * h)
            t += 1
        last.append(h)
    o, last = torch.stack(o), torch.stack(last)
    grads = torch.autograd.grad((o, last), (u, g, q, h0), (do, dht))
    got = block.gated_scan(u.detach(), g.detach(), lens, q.detach(), gate, h0.detach(), do, dht, 1e-7)
    for name, want in zip(("o", "ht", "du", "dg", "dq", "dh0"), (o, last, *grads)):
        assert torch.allclose(got[name][0], want.detach(), rtol=1e-12, atol=1e-12), name
        assert bool((got[name][1] >= 0).all())
