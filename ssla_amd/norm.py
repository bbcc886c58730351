"""Norms on MI355X: group norm with an activation, channels last, and the norms
around a block.

:func:`gated_norm` is the norm of an attention's output by heads times its output
gate; :func:`residual_norm` a residual stream's step from one block to the next (the
block's output, its own norm, dropout, scale, the sum, and the next block's norm).
Both work by rows, with a mean or without (``kind`` "layer" or "rms"), in one pass
over the data in either direction.

:func:`group_norm_act` normalises ``x [N, ..., C]`` over the positions of a
sample and the ``C / num_groups`` channels of a group, applies the channels'
weight and bias and an activation, in one pass over the data where a sample
fits on the chip.  With one group per head it is the norm behind a linear
attention's output (``[T, H * V]``: every row is a sample; an output gate of a
second tensor is :func:`gated_norm`'s); with ``[B, Hg, Wg, C]`` it is the norm of
dense event grids.  None of them has a counterpart in the reference, whose
layers normalise with ``nn.LayerNorm`` (layers/mos_attention.py:101).

The kernels are hand-written gfx950 kernels (``ssla_group_norm_*``,
``ssla_gated_norm_*``, ``ssla_residual_norm_*``); there is no CPU fallback.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _lib
from .dropout import _p, _seed

__all__ = ["group_norm_act", "GroupNormFunction", "ACTIVATIONS", "gated_norm", "GatedNormFunction", "residual_norm",
           "ResidualNormFunction", "KINDS", "GATE_ACTIVATIONS"]

ACTIVATIONS = {None: 0, "relu": 1, "silu": 2}
KINDS = {"rms": 0, "layer": 1}
GATE_ACTIVATIONS = {"silu": 2, "sigmoid": 3}
_WIDEST = 8192   # channels of a group


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


# ---------------------------------------------------------- norms around a block --
def _weight(name, nm, t, C):
    """A vector over the channels as the kernels take it (fp32, whole), or None."""
    if t is None:
        return None
    if t.shape != (C,) or not t.is_floating_point():
        raise ValueError(f"{name}: {nm} must be [{C}] floating point, got {tuple(t.shape)} {t.dtype}")
    return _whole(t if t.dtype is torch.float32 else t.float())


def _options(name, eps, kind):
    if kind not in KINDS:
        raise ValueError(f"{name}: kind must be one of {list(KINDS)}, got {kind!r}")
    if not eps >= 0:
        raise ValueError(f"{name}: eps must not be negative, got {eps}")


def _flat(t):
    """t as rows [N, C]; neighbouring channels side by side, the rows may lie apart."""
    t = t.reshape(-1, t.shape[-1]) if t.dim() != 2 else t
    return t if t.stride(1) == 1 and t.stride(0) >= t.shape[1] else t.contiguous()


class GatedNormFunction(torch.autograd.Function):
    """Forward ``ssla_gated_norm_fwd``, backward ``ssla_gated_norm_bwd``: keeps x and the
    gate; the normalised values are computed again.  dx and the gate's gradient have the
    inputs' dtype, those of weight and bias are fp32 sums in a fixed order."""

    @staticmethod
    def forward(ctx, x, z, weight, bias, G, eps, act, kind):
        ctx.save_for_backward(x, z, weight, bias)
        ctx.options = G, eps, act, kind
        return _gated_forward(x, z, weight, bias, G, eps, act, kind)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, z, weight, bias = ctx.saved_tensors
        G, eps, act, kind = ctx.options
        N, C = x.shape
        dy = _whole(dy)
        need = ctx.needs_input_grad
        dx, dz = (torch.empty(N, C, dtype=x.dtype, device=x.device) if n else None for n in need[:2])
        dw, db = (torch.empty_like(t) if t is not None and n else None for t, n in zip((weight, bias), need[2:4]))
        lib, P = _lib.load(), _lib.ptr
        with _lib.on_device_of(x):
            nbytes = lib.ssla_gated_norm_bwd_workspace_size(N, C, G) if dw is not None or db is not None else 0
            ws = _ws(nbytes, x.device)
            st = lib.ssla_gated_norm_bwd(P(dy), P(x), x.stride(0), P(z), z.stride(0), N, C, G, kind, P(weight), P(bias), eps,
                                         act, P(dx), P(dz), P(dw), P(db), _lib.DTYPE_CODE[x.dtype], P(ws), nbytes,
                                         _lib.stream_of(x))
        _lib.check(st, "ssla_gated_norm_bwd")
        return dx, dz, dw, db, None, None, None, None


def _gated_forward(x, z, w, b, G, eps, act, kind):
    N, C = x.shape
    y = torch.empty(N, C, dtype=x.dtype, device=x.device)
    P = _lib.ptr
    with _lib.on_device_of(x):
        st = _lib.load().ssla_gated_norm_fwd(P(x), x.stride(0), P(z), z.stride(0), N, C, G, kind, P(w), P(b), eps, act, P(y),
                                             _lib.DTYPE_CODE[x.dtype], _lib.stream_of(x))
    _lib.check(st, "ssla_gated_norm_fwd")
    return y


def gated_norm(x: torch.Tensor, gate: torch.Tensor, num_groups: int = 1, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, eps: float = 1e-5, activation: str = "silu",
               kind: str = "rms") -> torch.Tensor:
    """``norm(x) activation(gate)`` of x and gate ``[..., C]`` (one dtype of fp32, bf16,
    fp16; slices of a wider projection are taken as they are), in their dtype.

    Every row is normalised in ``num_groups`` groups of neighbouring channels (a head
    each behind an attention; at most 8,192 channels a group) in fp32: ``kind`` "rms"
    divides by the root mean square, "layer" takes the mean out first; eps is added to
    the mean square.  weight, bias: ``[C]`` or None; activation: "silu" or "sigmoid".
    Differentiable in x, gate, weight and bias (once, in reverse mode: forward-mode
    tangents are refused)."""
    name = "gated_norm"
    if x.dim() < 1 or gate.shape != x.shape or x.shape[-1] == 0:
        raise ValueError(f"{name}: x and gate must both be [..., C], got {tuple(x.shape)} and {tuple(gate.shape)}")
    C = x.shape[-1]
    if not isinstance(num_groups, int) or num_groups <= 0 or C % num_groups:
        raise ValueError(f"{name}: {C} channels do not divide into {num_groups} groups")
    if activation not in GATE_ACTIVATIONS:
        raise ValueError(f"{name}: activation must be one of {list(GATE_ACTIVATIONS)}, got {activation!r}")
    _options(name, eps, kind)
    if x.dtype not in _lib.DTYPE_CODE or gate.dtype != x.dtype:
        raise TypeError(f"{name}: x and gate must share fp32, bf16 or fp16 ({x.dtype}, {gate.dtype})")
    if C // num_groups > _WIDEST or C > 1 << 24:
        raise NotImplementedError(f"{name}: at most {_WIDEST} channels in a group and 2^24 in all, got {C} in {num_groups}")
    w, b = _weight(name, "weight", weight, C), _weight(name, "bias", bias, C)
    _lib.require_no_tangent(name, x, gate, weight, bias)
    _lib.require_cuda(x, gate, weight, bias)
    rows, z = _flat(x), _flat(gate)
    options = num_groups, float(eps), GATE_ACTIVATIONS[activation], KINDS[kind]
    grad = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, gate, weight, bias))
    y = (GatedNormFunction.apply if grad else _gated_forward)(rows, z, w, b, *options)
    return y if x.dim() == 2 else y.view(x.shape)   # (a view that changes nothing is a node of its own)


class ResidualNormFunction(torch.autograd.Function):
    """Forward ``ssla_residual_norm_fwd``, backward ``ssla_residual_norm_bwd``: keeps x, the
    residual and the seed; sum, norms and mask are computed again.  The gradients of x and
    the residual have their dtypes, those of the weights are fp32 sums in a fixed order."""

    @staticmethod
    def forward(ctx, x, r, weight, bias, gamma, post_weight, seed, options):
        if seed is not None:
            seed = seed.clone()   # (a caller may count it on before the backward)
        ctx.save_for_backward(x, r, weight, bias, gamma, post_weight, seed)
        ctx.options = options
        ctx.set_materialize_grads(False)
        return _residual_forward(x, r, weight, bias, gamma, post_weight, seed, options)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, ds):
        x, r, weight, bias, gamma, post_weight, seed = ctx.saved_tensors
        eps, kind, alpha, post, p, subsequence = ctx.options
        N, C = x.shape
        need = ctx.needs_input_grad
        if dy is None and ds is None:
            return (None,) * 8
        dy, ds = (None if t is None else _whole(t) for t in (dy, ds))
        dx, dr = (torch.empty_like(t) if n else None for t, n in zip((x, r), need))
        grads = [torch.empty_like(t) if t is not None and n else None
                 for t, n in zip((weight, bias, gamma, post_weight), need[2:6])]
        lib, P = _lib.load(), _lib.ptr
        with _lib.on_device_of(x):
            nbytes = lib.ssla_residual_norm_bwd_workspace_size(N, C) if any(t is not None for t in grads) else 0
            ws = _ws(nbytes, x.device)
            st = lib.ssla_residual_norm_bwd(P(dy), P(ds), P(x), P(r), N, C, kind, P(weight), eps, alpha, P(gamma), post,
                                            P(post_weight), p, P(seed), subsequence, P(dx), P(dr), *map(P, grads),
                                            _lib.DTYPE_CODE[x.dtype], _lib.DTYPE_CODE[r.dtype], P(ws), nbytes,
                                            _lib.stream_of(x))
        _lib.check(st, "ssla_residual_norm_bwd")
        return dx, dr, *grads, None, None


def _residual_forward(x, r, weight, bias, gamma, post_weight, seed, options):
    eps, kind, alpha, post, p, subsequence = options
    N, C = x.shape
    y, s = torch.empty_like(x), torch.empty_like(r)
    P = _lib.ptr
    with _lib.on_device_of(x):
        st = _lib.load().ssla_residual_norm_fwd(P(x), P(r), N, C, kind, P(weight), P(bias), eps, alpha, P(gamma), post,
                                                P(post_weight), p, P(seed), subsequence, P(y), P(s),
                                                _lib.DTYPE_CODE[x.dtype], _lib.DTYPE_CODE[r.dtype], _lib.stream_of(x))
    _lib.check(st, "ssla_residual_norm_fwd")
    return y, s


def residual_norm(x: torch.Tensor, residual: torch.Tensor, weight: Optional[torch.Tensor] = None,
                  bias: Optional[torch.Tensor] = None, eps: float = 1e-5, kind: str = "rms",
                  scale: Union[None, float, torch.Tensor] = None, post_norm: bool = False,
                  post_weight: Optional[torch.Tensor] = None, p: float = 0.0,
                  seed: Union[None, int, torch.Tensor] = None,
                  subsequence: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
    """A residual stream's step behind a block, ``(y, sum)``:

        sum = residual + scale * dropout(x, or its norm by post_weight with post_norm)
        y = norm(sum) * weight + bias

    x ``[..., C]`` is the block's output (fp32, bf16 or fp16; C up to 8,192), residual
    its dtype or fp32; y has x's dtype, sum the residual's.  y is the norm of the sum
    before the sum is rounded.  ``kind`` ("rms" or "layer") and eps hold for both
    norms; weight, bias, post_weight ``[C]`` or None; scale a number, ``[C]`` (a scale a
    channel) or None.  Dropout with probability ``p`` by ``seed`` and ``subsequence`` as
    :func:`ssla_amd.dropout.counter_dropout` (the same places of x are dropped).
    Differentiable in x, residual and all ``[C]`` vectors (once, in reverse mode:
    forward-mode tangents are refused)."""
    name = "residual_norm"
    if x.dim() < 1 or residual.shape != x.shape or x.shape[-1] == 0:
        raise ValueError(f"{name}: x and residual must both be [..., C], got {tuple(x.shape)} and {tuple(residual.shape)}")
    C = x.shape[-1]
    _options(name, eps, kind)
    if x.dtype not in _lib.DTYPE_CODE or residual.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"{name}: x must be fp32, bf16 or fp16 and residual that or fp32 ({x.dtype}, {residual.dtype})")
    if C > _WIDEST:
        raise NotImplementedError(f"{name}: at most {_WIDEST} channels, got {C}")
    if post_weight is not None and not post_norm:
        raise ValueError(f"{name}: post_weight needs post_norm=True")
    alpha, gamma = 1.0, None
    if torch.is_tensor(scale):
        gamma = _weight(name, "scale", scale, C)
    elif scale is not None:
        alpha = float(scale)
    w, b, w2 = (_weight(name, nm, t, C) for nm, t in (("weight", weight), ("bias", bias), ("post_weight", post_weight)))
    steps = _p(name, p)
    tensors = x, residual, weight, bias, scale if gamma is not None else None, post_weight
    _lib.require_no_tangent(name, *tensors)
    dev = _lib.require_cuda(*tensors)
    if p > 0 and seed is None:
        raise ValueError(f"{name}: dropout needs a seed")
    seed = _seed(name, seed, subsequence, dev) if p > 0 else None
    flat = x.dim() == 2
    rows, r = (_whole(t) if flat else _whole(t).view(-1, C) for t in (x, residual))
    options = float(eps), KINDS[kind], alpha, int(bool(post_norm)), steps, subsequence
    grad = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)
    y, s = (ResidualNormFunction.apply if grad else _residual_forward)(rows, r, w, b, gamma, w2, seed, options)
    return (y, s) if flat else (y.view(x.shape), s.view(x.shape))
