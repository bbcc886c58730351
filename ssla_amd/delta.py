"""Gated delta rule on MI355X.

The delta rule is linear attention whose write first takes out what the state
already answers for the key; a scalar gate per head and token lets the state
fade.  Per sequence and head, with state S ``[K, V]``:

    S <- exp(g_t) S;  u_t = beta_t (v_t - S^T k_t);  S <- S + k_t u_t^T
    o_t = scale S^T q_t

It stands beside the gated linear attention of :mod:`ssla_amd.gla` (same packed
layouts, same state tables) and has no counterpart in the reference.

* :func:`chunk_gated_delta` -- packed sequences by chunks of 64 tokens, on the
  matrix cores.
* :func:`fused_recurrent_gated_delta` -- token by token, for short sequences.
* :func:`sparse_delta_scan`, :func:`sparse_delta_step` -- per-site histories,
  and one token of each active site, on a resident state table.

Layouts: q, k ``[T, Hk, K]``, v ``[T, H, V]`` (one dtype of fp32, bf16, fp16),
g (log-gates) and beta ``[T, H]`` floating point, ``cu_seqlens`` ``[N + 1]``,
states fp32 ``[N, H, K, V]``.  ``H`` is a multiple of ``Hk``: value head h reads
key head ``h // (H // Hk)``.  A gate of -inf empties the state.  Tensors with
forward-mode tangents are refused.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib

__all__ = ["chunk_gated_delta", "ChunkGatedDeltaFunction", "fused_recurrent_gated_delta", "sparse_delta_scan", "sparse_delta_step"]


def _shapes(name, q, k, v, g, beta):
    for t, nm in ((q, "q"), (k, "k"), (v, "v")):
        if t.dim() != 3:
            raise ValueError(f"{name}: {nm} must be [T, heads, dim], got shape {tuple(t.shape)}")
    T, Hk, K = q.shape
    H, V = v.shape[1:]
    if k.shape != q.shape:
        raise ValueError(f"{name}: q and k shapes differ: {tuple(q.shape)}, {tuple(k.shape)}")
    if v.shape[0] != T or g.shape != (T, H) or beta.shape != (T, H):
        raise ValueError(f"{name}: v {tuple(v.shape)}, g {tuple(g.shape)} and beta {tuple(beta.shape)} must be [T, H, V], "
                         f"[T, H] and [T, H] with T = {T}")
    if 0 in (Hk, K, H, V) or H % Hk:
        raise ValueError(f"{name}: {H} value heads do not share {Hk} key heads (K={K}, V={V})")
    if not (q.dtype == k.dtype == v.dtype) or q.dtype not in _lib.DTYPE_CODE:
        raise TypeError(f"{name}: q, k, v must share fp32, bf16 or fp16 ({q.dtype}, {k.dtype}, {v.dtype})")
    if not (g.is_floating_point() and beta.is_floating_point()):
        raise TypeError(f"{name}: g and beta must be floating point ({g.dtype}, {beta.dtype})")
    return T, Hk, H, K, V


def _f32(t):
    return (t if t.dtype is torch.float32 else t.float()).contiguous()   # (a .to that does nothing costs as much as a check)


def _offsets(name, cu_seqlens, dev):
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1 or cu_seqlens.is_floating_point() or cu_seqlens.is_complex():
        raise ValueError(f"{name}: cu_seqlens must be integers [N + 1], got {cu_seqlens.dtype} {tuple(cu_seqlens.shape)}")
    return cu_seqlens.to(device=dev, dtype=torch.int64).contiguous()


def _table(name, state, H, K, V):
    if state.dim() != 4 or state.shape[1:] != (H, K, V) or state.dtype != torch.float32 or not state.is_contiguous():
        raise ValueError(f"{name}: state must be contiguous fp32 [n_sites, {H}, {K}, {V}]")


def _recurrent(q, k, v, g, beta, cu, n_seq, scale, h0, ht, state_idx=None, status=None):
    T, Hk, K = q.shape
    H, V = v.shape[1:]
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    g, beta = _f32(g), _f32(beta)
    o = torch.empty(T, H, V, device=v.device, dtype=v.dtype)
    P = _lib.ptr
    with _lib.on_device_of(q):
        st = _lib.load().ssla_gated_delta_recurrent(
            P(q), P(k), P(v), P(g), P(beta), P(cu), n_seq, T, Hk, H, K, V, float(scale), P(h0), P(o), P(ht),
            P(state_idx), 0 if state_idx is None else min(h0.shape[0], 0x7fffffff), P(status), _lib.DTYPE_CODE[q.dtype],
            _lib.stream_of(q))
    _lib.check(st, "ssla_gated_delta_recurrent")
    return o


def _chunk_fwd(q, k, v, g, beta, cu, scale, h0, output_final_state, keep=False):
    """One ssla_gated_delta_chunk_fwd call on contiguous tensors: o, the final
    states, and (keep) what its backward takes over."""
    T, Hk, K = q.shape
    H, V = v.shape[1:]
    N = cu.numel() - 1
    o = torch.empty_like(v)
    ht = torch.empty(N, H, K, V, device=v.device, dtype=torch.float32) if output_final_state else None
    lib, P = _lib.load(), _lib.ptr
    with _lib.on_device_of(q):
        nbytes = lib.ssla_gated_delta_chunk_workspace_size(N, T, H, K, V)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
        segments = None
        if keep:
            segments = torch.empty(lib.ssla_gated_delta_chunk_segments_size(N, T, H, K, V), dtype=torch.uint8,
                                   device=q.device)
        st = lib.ssla_gated_delta_chunk_fwd(P(q), P(k), P(v), P(g), P(beta), P(cu), N, T, Hk, H, K, V, float(scale),
                                            P(h0), P(o), P(ht), P(segments), _lib.DTYPE_CODE[q.dtype], P(ws), nbytes,
                                            _lib.stream_of(q))
    _lib.check(st, "ssla_gated_delta_chunk_fwd")
    return o, ht, segments


_SHORT = 64   # rows of a sequence that ssla_gated_delta_mixed_fwd runs token by token


def _token_rows(K: int) -> int:
    """Rows of an average sequence up to which a batch runs short sequences
    token by token: that kernel's time grows with K, the chunk kernels' hardly.
    Measured on sequences of one length, 4 heads, bf16, chunks against tokens, us:
    32,768 rows, K = 32 68 / 34 at 64 rows and 65 / 38 at 96, K = 64 115 / 119 at 32
    and 84 / 118 at 48, K = 128 807 / 671 at 16 and 556 / 627 at 24; 2,048 rows, where
    the length counts too (a token waits 0.20 to 0.41 us for the one before), K =
    32 20 / 17 at 64 and 23 / 24 at 96, K = 64 23 / 15 at 32, K = 128 64 / 48 at 16."""
    return max(16, min(64, 2048 // K))


def _mixed_fwd(q, k, v, g, beta, cu, scale, h0, output_final_state):
    """One ssla_gated_delta_mixed_fwd call on contiguous tensors: o and the final
    states."""
    T, Hk, K = q.shape
    H, V = v.shape[1:]
    N = cu.numel() - 1
    o = torch.empty_like(v)
    ht = torch.empty(N, H, K, V, device=v.device, dtype=torch.float32) if output_final_state else None
    lib, P = _lib.load(), _lib.ptr
    with _lib.on_device_of(q):
        nbytes = lib.ssla_gated_delta_mixed_workspace_size(T, H, K, V)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
        st = lib.ssla_gated_delta_mixed_fwd(P(q), P(k), P(v), P(g), P(beta), P(cu), N, T, Hk, H, K, V, float(scale), P(h0),
                                            P(o), P(ht), _lib.DTYPE_CODE[q.dtype], P(ws), nbytes, _lib.stream_of(q))
    _lib.check(st, "ssla_gated_delta_mixed_fwd")
    return o, ht


class ChunkGatedDeltaFunction(torch.autograd.Function):
    """Forward ``ssla_gated_delta_chunk_fwd``, backward
    ``ssla_gated_delta_chunk_bwd``: keeps the inputs and, of long sequences, the
    states and maps of their segments; every chunk's state is computed again.  dq, dk, dv have the inputs' dtype, dg, dbeta and dh0 are fp32."""

    @staticmethod
    def forward(ctx, q, k, v, g, beta, h0, cu, scale, output_final_state):
        o, ht, segments = _chunk_fwd(q, k, v, g, beta, cu, scale, h0, output_final_state, keep=True)
        ctx.save_for_backward(q, k, v, g, beta, h0, cu)
        ctx.segments = segments if segments.numel() else None
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return o, ht

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do, dht):
        q, k, v, g, beta, h0, cu = ctx.saved_tensors
        T, Hk, K = q.shape
        H, V = v.shape[1:]
        N = cu.numel() - 1
        do = torch.zeros_like(v) if do is None else do.to(v.dtype).contiguous()
        dht = None if dht is None else dht.to(torch.float32).contiguous()
        dq, dk, dv, dg, dbeta = (torch.empty_like(t) for t in (q, k, v, g, beta))
        dh0 = None if h0 is None else torch.empty_like(h0)
        lib, P = _lib.load(), _lib.ptr
        with _lib.on_device_of(q):
            nbytes = lib.ssla_gated_delta_chunk_bwd_workspace_size(N, T, Hk, H, K, V)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
            st = lib.ssla_gated_delta_chunk_bwd(
                P(q), P(k), P(v), P(g), P(beta), P(cu), N, T, Hk, H, K, V, ctx.scale, P(h0), P(do), P(dht), P(dq), P(dk),
                P(dv), P(dg), P(dbeta), P(dh0), P(ctx.segments), _lib.DTYPE_CODE[q.dtype], P(ws), nbytes, _lib.stream_of(q))
        _lib.check(st, "ssla_gated_delta_chunk_bwd")
        return dq, dk, dv, dg, dbeta, dh0, None, None, None


def chunk_gated_delta(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    g: torch.Tensor,
    beta: torch.Tensor,
    cu_seqlens: torch.Tensor,
    scale: Optional[float] = None,
    initial_state: Optional[torch.Tensor] = None,
    output_final_state: bool = False,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """The rule over packed sequences: o ``[T, H, V]`` in v's dtype and the fp32
    final state ``[N, H, K, V]`` or None.  ``scale`` defaults to ``K ** -0.5``.
    Rows of o outside ``[cu_seqlens[0], cu_seqlens[-1])`` are unspecified.

    K up to 128 runs the chunk kernels (chunks of 64 tokens) and is differentiable
    in q, k, v, g, beta and the initial state (once; rows in no sequence get zeros).
    Their products keep the precision of fp32 for states, gradients and the o of
    fp32 inputs; o of 16-bit inputs leaves out up to 2^-15 of its terms (2^-18 in the
    mean) before its own rounding.  Gates may be positive; the precision holds while no
    consecutive ones inside a chunk are more than 64 in sum (a state that grew by
    more and fades again meets decays whose parts fp32's normal numbers do not
    hold), and past 88 (the end of fp32) values are not finite.  Values smaller than
    2^-110 keep fewer bits for the same reason.  Without a
    gradient, where sequences are so short on average that chunks would stay
    mostly empty, those of up to 64 rows run the token-by-token kernel, longer ones
    the chunk kernels (told on the device); wider keys (K up to 256) run token by
    token, forward only."""
    name = "chunk_gated_delta"
    T, Hk, H, K, V = _shapes(name, q, k, v, g, beta)
    _lib.require_no_tangent(name, q, k, v, g, beta, initial_state)
    dev = _lib.require_cuda(q, k, v, g, beta, initial_state)
    cu = _offsets(name, cu_seqlens, dev)
    N = cu.numel() - 1
    if initial_state is not None and initial_state.shape != (N, H, K, V):
        raise ValueError(f"{name}: initial_state must be {(N, H, K, V)}, got {tuple(initial_state.shape)}")
    scale = K ** -0.5 if scale is None else float(scale)
    h0 = None if initial_state is None else _f32(initial_state)
    grad = torch.is_grad_enabled() and any(
        t is not None and t.requires_grad for t in (q, k, v, g, beta, initial_state))
    if grad and K > 128:
        raise NotImplementedError(f"{name}: the backward takes K up to 128 (got {K}; call it under torch.no_grad())")
    # short on average says nothing of the longest: unless no sequence can be far
    # longer (tokens wait for one another), each is told by its own length
    short = not grad and T <= N * _token_rows(K)
    if not grad and (K > 128 or short and T <= 2 * _SHORT):
        ht = torch.empty(N, H, K, V, device=dev, dtype=torch.float32) if output_final_state else None
        return _recurrent(q, k, v, g, beta, cu, N, scale, h0, ht), ht
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    g, beta = _f32(g), _f32(beta)
    if short:
        return _mixed_fwd(q, k, v, g, beta, cu, scale, h0, output_final_state)
    if grad:
        return ChunkGatedDeltaFunction.apply(q, k, v, g, beta, h0, cu, scale, output_final_state)
    return _chunk_fwd(q, k, v, g, beta, cu, scale, h0, output_final_state)[:2]


def fused_recurrent_gated_delta(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    g: torch.Tensor,
    beta: torch.Tensor,
    cu_seqlens: torch.Tensor,
    scale: Optional[float] = None,
    initial_state: Optional[torch.Tensor] = None,
    output_final_state: bool = False,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """The rule token by token (state in registers, K up to 256): o ``[T, H, V]``
    in v's dtype and the fp32 final state ``[N, H, K, V]`` or None.  ``scale``
    defaults to ``K ** -0.5``.  Rows of o outside ``[cu_seqlens[0],
    cu_seqlens[-1])`` are unspecified.  Makes no host sync; forward only."""
    name = "fused_recurrent_gated_delta"
    T, Hk, H, K, V = _shapes(name, q, k, v, g, beta)
    _lib.require_no_tangent(name, q, k, v, g, beta, initial_state)
    dev = _lib.require_cuda(q, k, v, g, beta, initial_state)
    _lib.require_no_grad(name, q, k, v, g, beta, initial_state)
    cu = _offsets(name, cu_seqlens, dev)
    N = cu.numel() - 1
    if initial_state is not None and initial_state.shape != (N, H, K, V):
        raise ValueError(f"{name}: initial_state must be {(N, H, K, V)}, got {tuple(initial_state.shape)}")
    h0 = None if initial_state is None else _f32(initial_state)
    ht = torch.empty(N, H, K, V, device=dev, dtype=torch.float32) if output_final_state else None
    o = _recurrent(q, k, v, g, beta, cu, N, K ** -0.5 if scale is None else scale, h0, ht)
    return o, ht


def _sites(name, idx, n):
    if idx.shape != (n,) or idx.is_floating_point() or idx.is_complex():
        raise ValueError(f"{name}: the site list must be integers [{n}], got {idx.dtype} {tuple(idx.shape)}")
    if idx.dtype.itemsize == 8:   # (kept out of range where 32 bits do not hold it)
        idx = idx.to(torch.int64).clamp(-1, 0x7fffffff)
    return (idx if idx.dtype is torch.int32 else idx.to(torch.int32)).contiguous()


def sparse_delta_scan(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                      cu_seqlens: torch.Tensor, seq_site: torch.Tensor, state: torch.Tensor,
                      scale: Optional[float] = None, check: bool = False) -> torch.Tensor:
    """Many bins at once: sequence n (rows ``cu_seqlens[n]:cu_seqlens[n+1]``, in
    time order) is the history of site ``seq_site[n]``; its row of ``state``
    (fp32 ``[n_sites, H, K, V]``) is read and written back in place, rows of
    other sites are not touched.  Returns o ``[T, H, V]`` in v's dtype.
    ``seq_site`` must be strictly increasing and inside ``[0, n_sites)``; a
    sequence whose entry is out of range or not above the one before it is
    skipped (zero o rows, state untouched; a site that such a list names twice
    elsewhere is left with an unspecified state); ``check=True`` reads the status
    back after the call (one host sync) and raises ValueError.  Forward only."""
    name = "sparse_delta_scan"
    T, Hk, H, K, V = _shapes(name, q, k, v, g, beta)
    _table(name, state, H, K, V)
    _lib.require_no_tangent(name, q, k, v, g, beta, state)
    dev = _lib.require_cuda(q, k, v, g, beta, state, seq_site)
    _lib.require_no_grad(name, q, k, v, g, beta, state)
    cu = _offsets(name, cu_seqlens, dev)
    idx = _sites(name, seq_site, cu.numel() - 1)
    status = _lib.new_status(dev) if check and idx.numel() else None
    o = _recurrent(q, k, v, g, beta, cu, idx.numel(), K ** -0.5 if scale is None else scale, state, state, idx, status)
    if status is not None and _lib.read_status(status) != _lib.SSLA_OK:
        raise ValueError(f"{name}: seq_site must be strictly increasing and inside [0, {state.shape[0]})")
    return o


def sparse_delta_step(site_idx: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor,
                      beta: torch.Tensor, state: torch.Tensor, scale: Optional[float] = None,
                      check: bool = False) -> torch.Tensor:
    """One token of each active site: row i of q, k, v, g, beta updates
    ``state[site_idx[i]]`` in place and gives row i of o.  The site list, the
    state table and ``check`` are as for :func:`sparse_delta_scan`; without
    ``check`` the call makes no host sync and can be captured in a HIP graph."""
    name = "sparse_delta_step"
    n, Hk, H, K, V = _shapes(name, q, k, v, g, beta)
    _table(name, state, H, K, V)
    _lib.require_no_tangent(name, q, k, v, g, beta, state)
    dev = _lib.require_cuda(q, k, v, g, beta, state, site_idx)
    _lib.require_no_grad(name, q, k, v, g, beta, state)
    idx = _sites(name, site_idx, n)
    status = _lib.new_status(dev) if check and n else None
    o = _recurrent(q, k, v, g, beta, None, n, K ** -0.5 if scale is None else scale, state, state, idx, status)
    if status is not None and _lib.read_status(status) != _lib.SSLA_OK:
        raise ValueError(f"{name}: site_idx must be strictly increasing and inside [0, {state.shape[0]})")
    return o
