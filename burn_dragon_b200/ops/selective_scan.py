"""Selective scan: a diagonal recurrence whose step is an input of its own for every channel (`csrc/selective_scan.cuh`).

    dt'_t = softplus(dt_t + dt_bias)                       (dt_softplus; else dt_t + dt_bias)
    h_t = exp(dt'_t A) h_{t-1} + (dt'_t u_t) (x) B_t        h: [D, N] per sequence
    y_t = h_t C_t + D u_t                                  (the current input is included)

Where `ops.ssd` has one decay per head, here every channel has its step and every state of it a decay A [D, N]; B and
C are shared by the channels, as they are there by the heads. Prompts and training (`selective_scan`), single tokens
(`selective_scan_step`). The spec is the selective state-space layer of Mamba (Gu & Dao, 2023).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.nn.functional as F

from . import native
from . import seqargs as A_


def selective_scan_reference(u, dt, A, Bm, Cm, D=None, *, dt_bias=None, dt_softplus: bool = False, h0=None, lengths=None):
    """Torch statement of `selective_scan`, step by step (any device and floating type, differentiable)."""
    B, T, Dn = u.shape
    ct = torch.promote_types(u.dtype, torch.float32)
    keep = A_.valid_rows(lengths, B, T, u.device)
    pick = lambda t: t.to(ct) if keep is None else torch.where(keep[..., None], t.to(ct), 0.0)            # noqa: E731
    us, Bs, Cs = pick(u), pick(Bm), pick(Cm)
    raw = pick(dt) + dt_bias.to(ct) if dt_bias is not None else pick(dt)
    step = F.softplus(raw) if dt_softplus else raw
    if keep is not None:
        step = torch.where(keep[..., None], step, 0.0)
    hs = (torch.float64 if ct == torch.float64 else torch.float32)
    h = h0.to(hs) if h0 is not None else torch.zeros(B, Dn, A.shape[1], dtype=hs, device=u.device)
    ys = []
    for t in range(T):
        h = torch.exp(step[:, t, :, None] * A.to(ct)) * h + (step[:, t] * us[:, t])[..., None] * Bs[:, t, None]
        ys.append((h * Cs[:, t, None]).sum(-1))
    y = torch.stack(ys, 1) if T else us
    if D is not None:
        y = y + D.to(ct) * us
    if keep is not None:
        y = torch.where(keep[..., None], y, 0.0)
    return y.to(u.dtype), (h if T else h.clone())               # (a state of its own, also behind no rows)


def _check(u, dt, A, Bm, Cm, D, dt_bias, dims: int) -> Tuple[int, int, int]:
    if not (u.dim() == dims and u.is_floating_point()):
        raise ValueError(f"u: expected a floating tensor of {dims} dimensions, got {u.dtype} {tuple(u.shape)}")
    Dn = u.shape[-1]
    if not (Dn >= 1):
        raise ValueError("u: expected at least one channel")
    if not (A.dim() == 2 and A.shape[0] == Dn and 1 <= A.shape[1] <= 64):
        raise ValueError(f"A: expected [{Dn}, N] with N in 1..64, got {tuple(A.shape)}")
    rows, N = u.shape[:-1], A.shape[1]
    A_.check_like(A, u, A.shape, "A")
    A_.check_like(dt, u, u.shape, "dt", u.dtype)
    A_.check_like(Bm, u, (*rows, N), "B", u.dtype)
    A_.check_like(Cm, u, (*rows, N), "C", u.dtype)
    A_.check_like(D, u, (Dn,), "D")
    A_.check_like(dt_bias, u, (Dn,), "dt_bias")
    return rows[0], Dn, N


def _state_type(u: torch.Tensor) -> torch.dtype:
    return torch.float64 if u.dtype == torch.float64 else torch.float32


def selective_scan(u: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, Bm: torch.Tensor, Cm: torch.Tensor, D: Optional[torch.Tensor] = None,
                   *, dt_bias: Optional[torch.Tensor] = None, dt_softplus: bool = False, h0: Optional[torch.Tensor] = None,
                   lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """u, dt [B, T, D], A [D, N] (N <= 64, finite), Bm, Cm [B, T, N], D and dt_bias [D], h0 [B, D, N] (fp32; None: zeros)
    -> (y [B, T, D] in the rows' type, hT [B, D, N] fp32). Rows are fp32, fp16 or bf16, all alike, and may be views into a
    wider projection (elements of a row adjacent). `lengths` [B]: behind a sequence's length the state stays as it
    is, y is 0, and the inputs are not read. Differentiable once in everything but `lengths`, the carried states included (the
    kernels refuse second derivatives and forward-mode tangents); a forward pass under autograd keeps the fp32 states of
    every 16th step (B T D N / 4 bytes, N rounded up to 8, 16, 32 or 64). All states and sums are fp32, sums over rows and
    channels in a fixed order."""
    B, Dn, N = _check(u, dt, A, Bm, Cm, D, dt_bias, 3)
    A_.check_like(h0, u, (B, Dn, N), "h0", _state_type(u))
    lengths = A_.check_lengths(lengths, u, B)
    if not A_.on_kernels(u) or u.shape[0] * u.shape[1] == 0:
        return selective_scan_reference(u, dt, A, Bm, Cm, D, dt_bias=dt_bias, dt_softplus=dt_softplus, h0=h0, lengths=lengths)
    y, hT = native.ops.selective_scan(A_.adjacent(u), A_.adjacent(dt), A_.dense_f32(A), A_.adjacent(Bm), A_.adjacent(Cm), A_.dense_f32(D),
                                      A_.dense_f32(dt_bias), bool(dt_softplus), A_.dense_f32(h0), lengths)
    return y, hT


def selective_scan_step(u: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, Bm: torch.Tensor, Cm: torch.Tensor, h: torch.Tensor,
                        D: Optional[torch.Tensor] = None, *, dt_bias: Optional[torch.Tensor] = None, dt_softplus: bool = False,
                        active: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """`selective_scan` for one row of every stream: u, dt [B, D], Bm, Cm [B, N], h [B, D, N] (fp32) -> (y [B, D], h'). The
    state is left as it was unless `out=h` asks for the update in place (`out`: where h' goes; like h it may be a
    slice of a larger tensor as long as each stream's [D, N] is dense; it is h itself or shares no memory with an input). `active` [B] (bool): a stream marked false gives
    y = 0 and keeps its state. No gradients (a decoding form)."""
    B, Dn, N = _check(u, dt, A, Bm, Cm, D, dt_bias, 2)
    A_.check_like(h, u, (B, Dn, N), "h", _state_type(u))
    active = A_.check_active(active, u, B)
    A_.check_out(out, h, "out")
    if A_.wants_grad(u, dt, A, Bm, Cm, h, D, dt_bias):
        raise ValueError("selective_scan_step has no gradient: call it under torch.no_grad(), or use selective_scan")
    if not A_.on_kernels(u):
        row = lambda t: t.unsqueeze(1)                                                                   # noqa: E731
        y, new = selective_scan_reference(row(u), row(dt), A, row(Bm), row(Cm), D, dt_bias=dt_bias, dt_softplus=dt_softplus, h0=h)
        y = y[:, 0]
        if active is not None:
            y, new = torch.where(active[:, None], y, 0.0), torch.where(active[:, None, None], new, h)
        return y, (new if out is None else out.copy_(new))
    dense = lambda t: (N == 1 or t.stride(2) == 1) and (Dn == 1 or t.stride(1) == N)                     # noqa: E731
    if not (out is None or dense(out)):
        raise ValueError("out: each stream's [D, N] must be dense")
    h = h if dense(h) else h.contiguous()
    y, *new = native.ops.selective_scan_step(A_.adjacent(u), A_.adjacent(dt), A_.dense_f32(A), A_.adjacent(Bm), A_.adjacent(Cm), h,
                                             A_.dense_f32(D), A_.dense_f32(dt_bias), bool(dt_softplus), active, out)
    return y, (new[0] if out is None else out)
