"""Group norm with an activation, channels last, on MI355X.

:func:`group_norm_act` normalises ``x [N, ..., C]`` over the positions of a
sample and the ``C / num_groups`` channels of a group, applies the channels'
weight and bias and an activation, in one pass over the data where a sample
fits on the chip.  With one group per head it is the norm behind a linear
attention's output (``[T, H * V]``: every row is a sample; an output gate of a
second tensor is a product of its own behind it); with ``[B, Hg, Wg, C]`` it is
the norm of dense event grids.  It has no counterpart in the reference, whose
layers normalise with ``nn.LayerNorm`` (layers/mos_attention.py:101).

The kernels are hand-written gfx950 kernels (``ssla_group_norm_fwd`` /
``_bwd``); there is no CPU fallback.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib

__all__ = ["group_norm_act", "GroupNormFunction", "ACTIVATIONS"]

ACTIVATIONS = {None: 0, "relu": 1, "silu": 2}


def _ws(nbytes: int, dev):
    return torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None


def _whole(t):
    """t contiguous and, for the kernels' wide loads, not off a 16-byte boundary:
    a view's sums are then taken in the order of a fresh tensor's."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _forward(x, num_groups, w, b, eps, act, stats):
    N, C = x.shape[0], x.shape[-1]
    L = x.numel() // max(N * C, 1)
    y = torch.empty_like(x)
    lib, P = _lib.load(), _lib.ptr
    with _lib.on_device_of(x):
        nbytes = lib.ssla_group_norm_workspace_size(N, L, C, num_groups)
        ws = _ws(nbytes, x.device)
        _lib.check(lib.ssla_group_norm_fwd(P(x), N, L, C, num_groups, P(w), P(b), float(eps), act, P(y), P(stats),
                                           _lib.DTYPE_CODE[x.dtype], P(ws), nbytes, _lib.stream_of(x)),
                   "ssla_group_norm_fwd")
    return y


class GroupNormFunction(torch.autograd.Function):
    """Forward ``ssla_group_norm_fwd``, backward ``ssla_group_norm_bwd``: keeps x
    and each group's mean and reciprocal deviation; the normalised values and
    the activation are computed again.  dx has x's dtype, dweight and dbias are
    fp32 sums over all positions in a fixed order."""

    @staticmethod
    def forward(ctx, x, weight, bias, num_groups, eps, act):
        stats = torch.empty(x.shape[0], num_groups, 2, dtype=torch.float32, device=x.device)
        y = _forward(x, num_groups, weight, bias, eps, act, stats)
        ctx.num_groups, ctx.act = num_groups, act
        ctx.save_for_backward(x, weight, bias, stats)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, bias, stats = ctx.saved_tensors
        N, C, G = x.shape[0], x.shape[-1], ctx.num_groups
        L = x.numel() // max(N * C, 1)
        dy = _whole(dy)
        need = ctx.needs_input_grad
        dx = torch.empty_like(x) if need[0] else None
        dw = torch.empty_like(weight) if need[1] else None
        db = torch.empty_like(bias) if need[2] else None
        lib, P = _lib.load(), _lib.ptr
        with _lib.on_device_of(x):
            nbytes = lib.ssla_group_norm_bwd_workspace_size(N, L, C, G)
            ws = _ws(nbytes, x.device)
            _lib.check(lib.ssla_group_norm_bwd(P(dy), P(x), P(stats), N, L, C, G, P(weight), P(bias), ctx.act, P(dx),
                                               P(dw), P(db), _lib.DTYPE_CODE[x.dtype], P(ws), nbytes,
                                               _lib.stream_of(x)), "ssla_group_norm_bwd")
        return dx, dw, db, None, None, None


def group_norm_act(x: torch.Tensor, num_groups: int, weight: Optional[torch.Tensor] = None,
                   bias: Optional[torch.Tensor] = None, eps: float = 1e-5,
                   activation: Optional[str] = None) -> torch.Tensor:
    """``activation(group_norm(x))`` of channels-last ``x [N, ..., C]`` (fp32,
    bf16 or fp16; another memory order is copied), y in x's dtype.

    The mean and variance of a group run over all positions of a sample
    (``x.shape[1:-1]``; none for ``[N, C]``, where every row is a sample) and
    ``C / num_groups`` neighbouring channels, in fp32.  weight, bias: ``[C]`` or
    None; activation: None, "relu" or "silu".  Differentiable in x, weight and
    bias (once, in reverse mode: forward-mode tangents are refused)."""
    if x.dim() < 2:
        raise ValueError(f"group_norm_act: x must be [N, ..., C], got shape {tuple(x.shape)}")
    C = x.shape[-1]
    if not isinstance(num_groups, int) or num_groups <= 0 or C == 0 or C % num_groups:
        raise ValueError(f"group_norm_act: {C} channels do not divide into {num_groups} groups")
    if activation not in ACTIVATIONS:
        raise ValueError(f"group_norm_act: activation must be one of {list(ACTIVATIONS)}, got {activation!r}")
    if not eps >= 0:
        raise ValueError(f"group_norm_act: eps must not be negative, got {eps}")
    if x.dtype not in _lib.DTYPE_CODE:
        raise TypeError(f"group_norm_act: unsupported dtype {x.dtype}")
    for t, nm in ((weight, "weight"), (bias, "bias")):
        if t is not None and (t.shape != (C,) or not t.is_floating_point()):
            raise ValueError(f"group_norm_act: {nm} must be [{C}] floating point, got {tuple(t.shape)} {t.dtype}")
    _lib.require_no_tangent("group_norm_act", x, weight, bias)
    _lib.require_cuda(x, weight, bias)
    x = _whole(x)
    w, b = (None if t is None else _whole(t.to(torch.float32)) for t in (weight, bias))
    act = ACTIVATIONS[activation]
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, w, b)):
        return GroupNormFunction.apply(x, w, b, num_groups, float(eps), act)
    return _forward(x, num_groups, w, b, eps, act, None)
