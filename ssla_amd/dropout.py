"""Dropout by a counter-based generator on MI355X: no mask is stored.

Element i of a tensor takes 16 bits of Philox4x32-10 at counter ``(i // 8,
subsequence)`` under the key ``seed``, so its fate follows from its place, the seed and
the subsequence alone: the backward draws the same bits again, and
:func:`ssla_amd.norm.residual_norm` drops what :func:`counter_dropout` drops.  It has
no counterpart in the reference, whose ``TemporalDropout``
(layers/temporal_dropout.py:6-59) drops whole events by their order in time.

The kernels are hand-written gfx950 kernels (``ssla_counter_dropout``); there is no
CPU fallback.
"""
from __future__ import annotations

import numbers
from typing import Union

import torch

from . import _lib

__all__ = ["counter_dropout", "CounterDropoutFunction"]


def _seed(name, seed, subsequence, device):
    """The seed as one int64 on `device` (a number's by a fill, which a graph may hold)."""
    if not isinstance(subsequence, numbers.Integral) or not 0 <= subsequence < 1 << 32:
        raise ValueError(f"{name}: subsequence must be an integer in [0, 2^32), got {subsequence!r}")
    if torch.is_tensor(seed):
        if seed.dtype != torch.int64 or seed.numel() != 1:
            raise ValueError(f"{name}: seed must be one int64, got {tuple(seed.shape)} {seed.dtype}")
        if seed.device != device:
            raise ValueError(f"{name}: seed must lie on {device}, got {seed.device}")
        return seed
    if not isinstance(seed, numbers.Integral) or not -(1 << 63) <= seed < 1 << 63:
        raise ValueError(f"{name}: seed must be a 64-bit integer or a tensor of one, got {seed!r}")
    return torch.full((1,), int(seed), dtype=torch.int64, device=device)


def _p(name, p):
    """p in whole steps of 2^-16 (which fp32 holds)."""
    if not isinstance(p, numbers.Real) or not 0 <= p <= 1:
        raise ValueError(f"{name}: p must lie in [0, 1], got {p!r}")
    return round(float(p) * 65536) / 65536


def _drop(x, p, seed, subsequence):
    y = torch.empty_like(x)
    with _lib.on_device_of(x):
        st = _lib.load().ssla_counter_dropout(_lib.ptr(x), x.numel(), p, _lib.ptr(seed), subsequence, _lib.ptr(y),
                                              _lib.DTYPE_CODE[x.dtype], _lib.stream_of(x))
    _lib.check(st, "ssla_counter_dropout")
    return y


class CounterDropoutFunction(torch.autograd.Function):
    """``ssla_counter_dropout`` both ways: keeps the seed (a copy: a caller may count it on
    before the backward), not the mask."""

    @staticmethod
    def forward(ctx, x, p, seed, subsequence):
        seed = seed.clone()
        ctx.save_for_backward(seed)
        ctx.p, ctx.subsequence, ctx.dtype = p, subsequence, x.dtype
        return _drop(x, p, seed, subsequence)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        (seed,) = ctx.saved_tensors
        return _drop(dy.to(ctx.dtype).contiguous(), ctx.p, seed, ctx.subsequence), None, None, None


def counter_dropout(x: torch.Tensor, p: float, seed: Union[int, torch.Tensor], subsequence: int = 0) -> torch.Tensor:
    """x (fp32, bf16 or fp16, any shape) with elements dropped with probability ``p``
    (in steps of 2^-16: ``t = round(p 2^16)``) and the others multiplied by
    ``2^16 / (2^16 - t)``, in x's dtype; what is dropped is 0 whatever it was.

    ``seed``: an integer, or an int64 tensor of one element on x's device, read when the
    kernel runs (in a captured graph a step changes it in place).  ``subsequence`` in
    ``[0, 2^32)`` tells apart the calls under one seed: equal ones drop the same places.
    Places are counted in x's logical order whatever its strides.  Differentiable in
    x (once, in reverse mode: forward-mode tangents are refused)."""
    name = "counter_dropout"
    p = _p(name, p)
    if x.dtype not in _lib.DTYPE_CODE:
        raise TypeError(f"{name}: unsupported dtype {x.dtype}")
    _lib.require_no_tangent(name, x)
    dev = _lib.require_cuda(x)
    seed = _seed(name, seed, subsequence, dev)
    x = x.contiguous()
    if torch.is_grad_enabled() and x.requires_grad:
        return CounterDropoutFunction.apply(x, p, seed, subsequence)
    return _drop(x, p, seed, subsequence)
