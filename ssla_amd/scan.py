"""Sparse sequential scans on MI355X.

* :func:`scan` -- drop-in for ``ops.common.scan.scan(u, g, cu_seqlens)``
  (reference ops/common/scan.py:140-163): varlen diagonal gated scan
  ``h_t = g_t * h_{t-1} + u_t`` with a zero state at each sequence start,
  with its backward (:class:`SequentialScan`).
* :func:`gated_scan` -- the gated recurrence over long sequences (no reference
  function): any length is split along time, states go in and out, the gate may
  be a logit or a logarithm and a read-out gate is multiplied on the way; with
  its backward (:class:`GatedScanFunction`).
* :func:`sparse_gated_step` -- its single tokens, on a resident state table.
* :func:`sparse_gla_step` -- one time bin of the per-site matrix-state GLA
  update at active sites only (no reference function; its math is
  ``naive_gla_recurrent``, reference ops/gla/naive.py:50-111, on a length-1
  sequence per active site whose initial state is the stored site state).
* :func:`sparse_gla_scan` -- the same update over many bins at once, as a
  varlen recurrence per site whose state is gathered from and scattered back
  to the resident state table.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .delta import _f32, _offsets, _sites
from .gla import _recurrent

__all__ = ["scan", "SequentialScan", "gated_scan", "GatedScanFunction", "GATES", "sparse_gated_step", "sparse_gla_step",
           "sparse_gla_scan"]

GATES = {"value": 0, "log": 1, "sigmoid": 2}
_WIDEST = 1 << 20   # elements from row to row: offsets inside a tile of rows are 32 bits


def _scan_fwd(u: torch.Tensor, g: torch.Tensor, cu: torch.Tensor) -> torch.Tensor:
    T, C = u.shape
    h = torch.empty_like(u)
    st = _lib.load().ssla_diag_scan_fwd(_lib.ptr(u), _lib.ptr(g), _lib.ptr(cu), cu.numel() - 1, T, C,
                                        _lib.ptr(h), _lib.stream_of(u))
    _lib.check(st, "ssla_diag_scan_fwd")
    return h


class SequentialScan(torch.autograd.Function):
    """Forward and backward of the varlen diagonal scan (reference
    ops/common/scan.py:89-137): saves g and h, and the backward kernel
    returns (du, dg) with zeros on rows in no sequence."""

    @staticmethod
    def forward(ctx, u, g, cu_seqlens):
        h = _scan_fwd(u, g, cu_seqlens)
        ctx.save_for_backward(g, h, cu_seqlens)
        return h

    @staticmethod
    def backward(ctx, dout):
        g, h, cu = ctx.saved_tensors
        dout = dout.to(torch.float32).contiguous()
        T, C = h.shape
        du, dg = torch.empty_like(h), torch.empty_like(h)
        st = _lib.load().ssla_diag_scan_bwd(_lib.ptr(dout), _lib.ptr(g), _lib.ptr(h), _lib.ptr(cu), cu.numel() - 1,
                                            T, C, _lib.ptr(du), _lib.ptr(dg), _lib.stream_of(h))
        _lib.check(st, "ssla_diag_scan_bwd")
        return du, dg, None


def scan(u: torch.Tensor, g: torch.Tensor, cu_seqlens: torch.Tensor) -> torch.Tensor:
    """Varlen diagonal scan; u, g ``[T, C]`` -> h ``[T, C]`` in u's dtype
    (reference ops/common/scan.py:101, ``torch.zeros_like(u)``; rows in no
    sequence are zero).  The running state is fp32 and each stored row is
    rounded once to u's dtype, as the reference kernel's fp32 ``b_h`` is
    (scan.py:35-43).  Differentiable in u and g (``ssla_diag_scan_bwd``)."""
    if u.dim() != 2 or u.shape != g.shape:
        raise ValueError(f"scan: u and g must both be [T, C], got {tuple(u.shape)}, {tuple(g.shape)}")
    dev = _lib.require_cuda(u, g)
    out_dtype = u.dtype
    u = u.to(torch.float32).contiguous()
    g = g.to(torch.float32).contiguous()
    cu = cu_seqlens.to(device=dev, dtype=torch.int64).contiguous()
    if torch.is_grad_enabled() and (u.requires_grad or g.requires_grad):
        h = SequentialScan.apply(u, g, cu)
    else:
        h = _scan_fwd(u, g, cu)
    return h if out_dtype == torch.float32 else h.to(out_dtype)


def _gated_args(name, u, g, q, gate):
    if u.dim() != 2 or g.shape != u.shape or (q is not None and q.shape != u.shape) or u.shape[1] == 0:
        raise ValueError(f"{name}: u, g and q must all be [T, C], got {tuple(u.shape)}, {tuple(g.shape)}, "
                         f"{None if q is None else tuple(q.shape)}")
    if u.shape[1] > _WIDEST:
        raise NotImplementedError(f"{name}: at most {_WIDEST} channels, got {u.shape[1]}")
    if gate not in GATES:
        raise ValueError(f"{name}: gate must be one of {list(GATES)}, got {gate!r}")
    if u.dtype not in _lib.DTYPE_CODE or (q is not None and q.dtype != u.dtype):
        raise TypeError(f"{name}: u and q must share fp32, bf16 or fp16 ({u.dtype}, {None if q is None else q.dtype})")
    if not g.is_floating_point():
        raise TypeError(f"{name}: g must be floating point ({g.dtype})")


def _rows(t):
    """t with neighbouring channels side by side (the rows may lie apart, as those
    of a slice of a wider projection do)."""
    return t if t is None or t.stride(1) == 1 and t.shape[1] <= t.stride(0) <= _WIDEST else t.contiguous()


def _gated_forward(u, g, q, cu, gate, h0, output_final_state, save=False):
    """One ssla_gated_scan_fwd call: o, the final states, and (save) what its
    backward takes over."""
    T, C = u.shape
    N = cu.numel() - 1
    dev = u.device
    o = torch.empty(T, C, device=dev, dtype=u.dtype)
    ht = torch.empty(N, C, device=dev, dtype=torch.float32) if output_final_state else None
    lib, P = _lib.load(), _lib.ptr
    with _lib.on_device_of(u):
        keep = torch.empty(lib.ssla_gated_scan_keep_size(T, C), dtype=torch.uint8, device=dev) if save else None
        nbytes = lib.ssla_gated_scan_workspace_size(T, C)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
        st = lib.ssla_gated_scan_fwd(P(u), u.stride(0), P(g), g.stride(0), P(q), 0 if q is None else q.stride(0), P(cu), N,
                                     T, C, gate, P(h0), P(o), P(ht), P(keep), _lib.DTYPE_CODE[u.dtype],
                                     _lib.DTYPE_CODE[g.dtype], P(ws), nbytes, _lib.stream_of(u))
    _lib.check(st, "ssla_gated_scan_fwd")
    return o, ht, keep


class GatedScanFunction(torch.autograd.Function):
    """Forward ``ssla_gated_scan_fwd``, backward ``ssla_gated_scan_bwd``: keeps the
    inputs and the states between pieces of the time axis; the others are computed
    again.  The gradients have the inputs' dtypes."""

    @staticmethod
    def forward(ctx, u, g, q, h0, cu, gate, output_final_state):
        o, ht, keep = _gated_forward(u, g, q, cu, gate, h0, output_final_state, save=True)
        ctx.save_for_backward(u, g, q, h0, cu, keep)
        ctx.gate = gate
        ctx.set_materialize_grads(False)
        return o, ht

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do, dht):
        u, g, q, h0, cu, keep = ctx.saved_tensors
        T, C = u.shape
        do = torch.zeros(T, C, device=u.device, dtype=u.dtype) if do is None else do.to(u.dtype).contiguous()
        dht = None if dht is None else _f32(dht)
        du, dg, dq = (None if t is None else torch.empty(T, C, device=u.device, dtype=t.dtype) for t in (u, g, q))
        dh0 = None if h0 is None else torch.empty_like(h0)
        lib, P = _lib.load(), _lib.ptr
        with _lib.on_device_of(u):
            nbytes = lib.ssla_gated_scan_workspace_size(T, C)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=u.device) if nbytes else None
            st = lib.ssla_gated_scan_bwd(P(u), u.stride(0), P(g), g.stride(0), P(q), 0 if q is None else q.stride(0), P(cu),
                                         cu.numel() - 1, T, C, ctx.gate, P(h0), P(keep), P(do), P(dht), P(du), P(dg), P(dq),
                                         P(dh0), _lib.DTYPE_CODE[u.dtype], _lib.DTYPE_CODE[g.dtype], P(ws), nbytes,
                                         _lib.stream_of(u))
        _lib.check(st, "ssla_gated_scan_bwd")
        return du, dg, dq, dh0, None, None, None


def gated_scan(
    u: torch.Tensor,
    g: torch.Tensor,
    cu_seqlens: torch.Tensor,
    q: Optional[torch.Tensor] = None,
    gate: str = "value",
    initial_state: Optional[torch.Tensor] = None,
    output_final_state: bool = False,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """The gated recurrence ``h_t = a_t h_{t-1} + u_t`` of packed sequences, channel
    by channel, and ``o_t = q_t h_t`` (without q: ``h_t``).

    u, q ``[T, C]`` (one dtype of fp32, bf16, fp16), g ``[T, C]`` floating point;
    ``gate`` says what g is: the factor a itself ("value"), its logarithm ("log":
    -inf empties the state) or its logit ("sigmoid").  Slices of a wider projection
    are taken as they are.  Sequence n has the rows ``cu_seqlens[n]:cu_seqlens[n + 1]``
    (any lengths, zero too) and starts from row n of ``initial_state`` (``[N, C]``; None:
    zeros).  Returns o ``[T, C]`` in u's dtype, zeros on rows in no sequence, and the
    fp32 final state ``[N, C]`` or None.

    States are fp32; a long sequence is cut along time and the pieces' states are
    joined in their order, so results do not vary from call to call.  Over a piece
    (up to 512 rows; up to 8,192 in calls of at most 256 channels) the gates are
    multiplied: factors larger than 1 in magnitude hold while such a product, and what
    the piece sums up from a zero state, stay inside fp32 (a zero state passes any
    product, and a gate of 0 empties a finite state whatever the gates beside it).
    An infinite state (or gradient) goes on with the gates' signs until a gate of 0
    (logarithms and logits below about -87 are 0 in fp32) makes it NaN, as row by row.
    Differentiable in u, g, q and the initial state (once, in reverse mode:
    forward-mode tangents are refused).  Makes no host sync."""
    name = "gated_scan"
    _gated_args(name, u, g, q, gate)
    _lib.require_no_tangent(name, u, g, q, initial_state)
    dev = _lib.require_cuda(u, g, q, initial_state)
    cu = _offsets(name, cu_seqlens, dev)
    N, C = cu.numel() - 1, u.shape[1]
    if N > 1 << 30:
        raise NotImplementedError(f"{name}: too many sequences ({N})")
    if initial_state is not None and (initial_state.shape != (N, C) or not initial_state.is_floating_point()):
        raise ValueError(f"{name}: initial_state must be floating point {(N, C)}, got {tuple(initial_state.shape)} "
                         f"{initial_state.dtype}")
    g = g if g.dtype in (u.dtype, torch.float32) else g.float()
    u, g, q = _rows(u), _rows(g), _rows(q)
    h0 = None if initial_state is None else _f32(initial_state)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (u, g, q, h0)):
        return GatedScanFunction.apply(u, g, q, h0, cu, GATES[gate], output_final_state)
    return _gated_forward(u, g, q, cu, GATES[gate], h0, output_final_state)[:2]


def sparse_gated_step(site_idx: torch.Tensor, u: torch.Tensor, g: torch.Tensor, state: torch.Tensor,
                      q: Optional[torch.Tensor] = None, gate: str = "value", check: bool = False) -> torch.Tensor:
    """One token of each active row of a state table: row i of u, g and q
    (``[n, C]``, as for :func:`gated_scan`) updates ``state[site_idx[i]]`` (fp32
    ``[n_sites, C]``) in place and gives row i of o (u's dtype).  ``site_idx``:
    integers, strictly increasing and inside ``[0, n_sites)``; an entry that is
    out of range or not above the one before it is skipped (zero o rows, state
    untouched; a site that such a list names twice elsewhere is left with an
    unspecified state); ``check=True`` reads the status back after the call (one host sync)
    and raises ValueError, without it the call makes no host sync and can be
    captured in a HIP graph.  Forward only."""
    name = "sparse_gated_step"
    _gated_args(name, u, g, q, gate)
    n, C = u.shape
    if n > 1 << 30:
        raise NotImplementedError(f"{name}: too many rows ({n})")
    if state.dim() != 2 or state.shape[1] != C or state.dtype != torch.float32 or not state.is_contiguous():
        raise ValueError(f"{name}: state must be contiguous fp32 [n_sites, {C}]")
    _lib.require_no_tangent(name, u, g, q, state)
    dev = _lib.require_cuda(u, g, q, state, site_idx)
    _lib.require_no_grad(name, u, g, q, state)
    idx = _sites(name, site_idx, n)
    g = g if g.dtype in (u.dtype, torch.float32) else g.float()
    u, g, q = _rows(u), _rows(g), _rows(q)
    o = torch.empty(n, C, device=dev, dtype=u.dtype)
    status = _lib.new_status(dev) if check and n else None
    P = _lib.ptr
    with _lib.on_device_of(u):
        st = _lib.load().ssla_sparse_gated_step(
            P(idx), n, P(u), u.stride(0), P(g), g.stride(0), P(q), 0 if q is None else q.stride(0), P(state),
            min(state.shape[0], 0x7fffffff), C, GATES[gate], P(o), P(status), _lib.DTYPE_CODE[u.dtype],
            _lib.DTYPE_CODE[g.dtype], _lib.stream_of(u))
    _lib.check(st, "ssla_sparse_gated_step")
    if status is not None and _lib.read_status(status) != _lib.SSLA_OK:
        raise ValueError(f"{name}: site_idx must be strictly increasing and inside [0, {state.shape[0]})")
    return o


def sparse_gla_step(site_idx: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                    g: torch.Tensor, state: torch.Tensor, scale: Optional[float] = None,
                    check: bool = False) -> torch.Tensor:
    """Update ``state[site_idx]`` in place for one time bin and return o.

    site_idx: int32 ``[n]`` (strictly increasing, inside ``[0, n_sites)``);
    q, k, g: fp32 ``[n, H, K]``; v: fp32 ``[n, H, V]``; state: fp32
    ``[n_sites, H, K, V]``.  Rows of inactive sites are neither read nor
    written.  An entry out of range or not above the one before it is
    skipped (its o rows are zero, no state changes).  ``check=True`` reads
    the status word back after the call (one host sync) and raises
    ValueError for such an entry; the default makes no host sync, so a
    caller stepping through many bins pays none.
    """
    n, H, K = q.shape
    V = v.shape[-1]
    if k.shape != q.shape or g.shape != q.shape or v.shape[:2] != (n, H):
        raise ValueError("sparse_gla_step: q, k, g must be [n, H, K] and v [n, H, V]")
    if state.dim() != 4 or state.shape[1:] != (H, K, V) or state.dtype != torch.float32:
        raise ValueError(f"sparse_gla_step: state must be fp32 [n_sites, {H}, {K}, {V}]")
    if not state.is_contiguous():
        raise ValueError("sparse_gla_step: state must be contiguous (it is updated in place)")
    if site_idx.shape != (n,):
        raise ValueError("sparse_gla_step: site_idx must be [n]")
    _lib.require_cuda(site_idx, q, k, v, g, state)
    _lib.require_no_grad("sparse_gla_step", q, k, v, g, state)
    if scale is None:
        scale = K ** -0.5
    sidx = site_idx.to(torch.int32).contiguous()
    q, k, v, g = (t.to(torch.float32).contiguous() for t in (q, k, v, g))
    o = torch.empty(n, H, V, device=q.device, dtype=torch.float32)
    lib = _lib.load()
    status = _lib.new_status(q.device) if check and n else None
    st = lib.ssla_sparse_gla_step(_lib.ptr(sidx), n, _lib.ptr(q), _lib.ptr(k), _lib.ptr(v),
                                  _lib.ptr(g), _lib.ptr(state), state.shape[0], H, K, V,
                                  float(scale), _lib.ptr(o), _lib.ptr(status), _lib.stream_of(q))
    _lib.check(st, "ssla_sparse_gla_step")
    if status is not None and _lib.read_status(status) != _lib.SSLA_OK:
        raise ValueError(f"sparse_gla_step: site_idx must be strictly increasing and inside [0, {state.shape[0]})")
    return o


def sparse_gla_scan(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor,
                    cu_seqlens: torch.Tensor, seq_site: torch.Tensor, state: torch.Tensor,
                    scale: Optional[float] = None, check: bool = False) -> torch.Tensor:
    """Many bins at once: sequence n (rows ``cu_seqlens[n]:cu_seqlens[n+1]``,
    ordered in time) is the history of site ``seq_site[n]``; its state row
    is read from and written back to ``state`` in place.  Returns o with
    q's dtype.  ``seq_site`` must be strictly increasing and inside
    ``[0, n_sites)``; a sequence whose entry is not is skipped (zero o rows,
    state untouched); ``check=True`` reads the status back after the call
    (one host sync) and raises ValueError for such a sequence."""
    T, H, K = q.shape
    V = v.shape[-1]
    if state.dim() != 4 or state.shape[1:] != (H, K, V) or state.dtype != torch.float32 \
            or not state.is_contiguous():
        raise ValueError(f"sparse_gla_scan: state must be contiguous fp32 [n_sites, {H}, {K}, {V}]")
    dev = _lib.require_cuda(q, k, v, g, state, seq_site)
    _lib.require_no_grad("sparse_gla_scan", q, k, v, g, state)
    if scale is None:
        scale = K ** -0.5
    cu = cu_seqlens.to(device=dev, dtype=torch.int64).contiguous()
    sidx = seq_site.to(device=dev, dtype=torch.int32).contiguous()
    if sidx.numel() != cu.numel() - 1:
        raise ValueError("sparse_gla_scan: seq_site needs one entry per sequence")
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    g = g.to(torch.float32).contiguous() if g.dtype != q.dtype else g.contiguous()
    o = torch.empty(T, H, V, device=q.device, dtype=q.dtype)
    status = _lib.new_status(dev) if check and sidx.numel() else None
    _recurrent(q, k, v, g, cu, float(scale), state, o, state, sidx, state.shape[0], status)
    if status is not None and _lib.read_status(status) != _lib.SSLA_OK:
        raise ValueError(f"sparse_gla_scan: seq_site must be strictly increasing and inside [0, {state.shape[0]})")
    return o
