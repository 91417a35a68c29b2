"""Elementwise parts of a Mamba-2 block around the SSD scan: causal depthwise conv1d + SiLU in front,
gated RMSNorm behind. On a GPU both run as one fp32 kernel per direction (`csrc/mamba_ops.cu`) with their
backward passes written out; elsewhere the torch statement of the same function runs under autograd.
The reference has no Mamba path; these serve the Mamba-2 model family of this package (models/mamba.py).

`causal_conv` / `causal_conv_step` are the convolution in its general form: fp32, fp16 or bf16 rows, which may be a
view into a wider projection; a carried state in and out; padded batches; and a form for single tokens
(`csrc/causal_conv.cu`).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.nn.functional as F

from . import native
from . import seqargs as A


def _on_kernels(*ts) -> bool:
    return (native.available() and all(t is None or (t.is_cuda and t.dtype == torch.float32) for t in ts))


# ---- conv1d + SiLU -----------------------------------------------------------------------------------
def conv1d_silu_reference(seq: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor]) -> torch.Tensor:
    """seq [B, T + k - 1, C] (the k - 1 leading rows are the previous segment's tail or zeros), w [C, k],
    bias [C] -> silu(depthwise causal conv) [B, T, C]."""
    out = F.conv1d(seq.transpose(1, 2), w.unsqueeze(1), bias, groups=w.shape[0]).transpose(1, 2)
    return F.silu(out)


class _ConvSilu(torch.autograd.Function):
    @staticmethod
    def forward(ctx, seq, w, bias):
        seq, w = seq.contiguous(), w.contiguous()
        B, Tin, C = seq.shape
        k = w.shape[1]
        out = torch.empty(B, Tin - k + 1, C, device=seq.device, dtype=torch.float32)
        native.ops.conv1d_silu_fwd(seq, w, bias, out)
        ctx.save_for_backward(seq, w, bias)
        return out

    @staticmethod
    def backward(ctx, dout):
        seq, w, bias = ctx.saved_tensors
        dout = dout.contiguous()
        dpre = torch.empty_like(dout)
        dseq = torch.empty_like(seq)
        dw = torch.zeros_like(w)
        db = torch.zeros_like(bias) if bias is not None else None
        native.ops.conv1d_silu_bwd(seq, w, bias, dout, dpre, dseq, dw, db)
        return dseq, dw, db


def conv1d_silu(seq: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor]) -> torch.Tensor:
    if _on_kernels(seq, w, bias) and w.shape[1] <= 8:
        return _ConvSilu.apply(seq, w, bias)
    return conv1d_silu_reference(seq, w, bias)


# ---- causal convolution with a carried state -----------------------------------------------------------
def causal_conv_reference(x, w, bias=None, state=None, lengths=None, activation: Optional[str] = "silu"):
    """Torch statement of `causal_conv` (any device and floating type, differentiable)."""
    B, T, C = x.shape
    k = w.shape[1]
    ct = torch.promote_types(x.dtype, torch.float32)
    keep = A.valid_rows(lengths, B, T, x.device)
    xs = x.to(ct) if keep is None else torch.where(keep[..., None], x.to(ct), 0.0)
    head = state.to(ct) if state is not None else xs.new_zeros(B, k - 1, C)
    seq = torch.cat((head, xs), dim=1)                                         # [B, T + k - 1, C]
    pre = sum(seq[:, j:j + T] * w[:, j].to(ct) for j in range(k))
    if bias is not None:
        pre = pre + bias.to(ct)
    y = F.silu(pre) if activation == "silu" else pre
    if keep is None:
        return y.to(x.dtype), seq[:, T:].to(x.dtype)
    rows = lengths.clamp(0, T).long()[:, None] + torch.arange(k - 1, device=x.device)
    tail = torch.gather(seq, 1, rows[..., None].expand(-1, -1, C))
    return torch.where(keep[..., None], y, 0.0).to(x.dtype), tail.to(x.dtype)


def _check_conv(x, w, bias, activation, dims: int) -> bool:
    if not (x.dim() == dims and x.is_floating_point()):
        raise ValueError(f"x: expected a floating tensor of {dims} dimensions, got {x.dtype} {tuple(x.shape)}")
    C = x.shape[-1]
    if not (w.dim() == 2 and w.shape[0] == C and 1 <= w.shape[1] <= 8):
        raise ValueError(f"w: expected [{C}, k] with k in 1..8, got {tuple(w.shape)}")
    if not (C >= 1):
        raise ValueError("x: expected at least one channel")
    A.check_like(w, x, w.shape, "w")
    A.check_like(bias, x, (C,), "bias")
    if not (activation in (None, "silu")):
        raise ValueError(f"activation: expected None or 'silu', got {activation!r}")
    return activation == "silu"


def causal_conv(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None, *, state: Optional[torch.Tensor] = None,
                lengths: Optional[torch.Tensor] = None, activation: Optional[str] = "silu") -> Tuple[torch.Tensor, torch.Tensor]:
    """Causal depthwise convolution of x [B, T, C] with w [C, k] (k <= 8), bias [C]: with s = [state | x],
    y_t = act(bias + sum_j w[:, j] s_{t+j}). Returns (y [B, T, C], state' [B, k-1, C]): the last k - 1 rows of s, to be
    passed as `state` with the sequence's next rows (None: zeros). Rows are fp32, fp16 or bf16 (y and the states are of
    their type), sums fp32; x and the state may be views whose channels are adjacent. `lengths` [B]: the rows of each sequence that
    count; y is 0 behind them, the state ends there, and whatever x holds there is not read. Differentiable in x, w,
    bias and both states, once (the kernels refuse second derivatives and forward-mode tangents); the sums over rows are made
    in a fixed order."""
    silu = _check_conv(x, w, bias, activation, 3)
    B, T, C = x.shape
    A.check_like(state, x, (B, w.shape[1] - 1, C), "state", x.dtype)
    lengths = A.check_lengths(lengths, x, B)
    if not A.on_kernels(x):
        return causal_conv_reference(x, w, bias, state, lengths, activation)
    y, tail = native.ops.causal_conv(A.adjacent(x), A.dense_f32(w), A.dense_f32(bias), A.adjacent(state), lengths, silu)
    return y, tail


def causal_conv_step(x: torch.Tensor, state: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                     activation: Optional[str] = "silu", active: Optional[torch.Tensor] = None,
                     out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """`causal_conv` for one row of every stream: x [B, C], state [B, k-1, C] -> (y [B, C], state'). The state is left
    as it was unless `out=state` asks for the update in place (`out`: where state' goes, which is the state itself or
    shares no memory with an input). `active` [B] (bool): a stream marked false gives y = 0 and keeps its state. No
    gradients (a decoding form)."""
    silu = _check_conv(x, w, bias, activation, 2)
    B, C = x.shape
    k = w.shape[1]
    A.check_like(state, x, (B, k - 1, C), "state", x.dtype)
    active = A.check_active(active, x, B)
    A.check_out(out, state, "out")
    if A.wants_grad(x, state, w, bias):
        raise ValueError("causal_conv_step has no gradient: call it under torch.no_grad(), or use causal_conv")
    if not A.on_kernels(x):
        y, new = causal_conv_reference(x.unsqueeze(1), w, bias, state, None, activation)
        y = y[:, 0]
        if active is not None:
            y, new = torch.where(active[:, None], y, 0.0), torch.where(active[:, None, None], new, state)
        return y, (new if out is None else out.copy_(new))
    if not (out is None or C == 1 or out.stride(-1) == 1):
        raise ValueError("out: its channels must be adjacent")
    y, *new = native.ops.causal_conv_step(A.adjacent(x), A.adjacent(state), A.dense_f32(w), A.dense_f32(bias), active, silu, out)
    return y, (new[0] if out is None else out)


# ---- gated RMSNorm -----------------------------------------------------------------------------------
def gated_rmsnorm_reference(v: torch.Tensor, z: torch.Tensor, w: torch.Tensor, eps: float = 1e-5) -> torch.Tensor:
    g = v * F.silu(z)
    return g * torch.rsqrt(g.pow(2).mean(-1, keepdim=True) + eps) * w


class _GatedRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, v, z, w, eps):
        v, z, w = v.contiguous(), z.contiguous(), w.contiguous()
        out = torch.empty_like(v)
        rstd = torch.empty(v.numel() // v.shape[-1], device=v.device, dtype=torch.float32)
        native.ops.gated_rmsnorm_fwd(v, z, w, out, rstd, float(eps))
        ctx.save_for_backward(v, z, w, rstd)
        return out

    @staticmethod
    def backward(ctx, dout):
        v, z, w, rstd = ctx.saved_tensors
        dout = dout.contiguous()
        dv, dz = torch.empty_like(v), torch.empty_like(z)
        dw = torch.zeros_like(w)
        native.ops.gated_rmsnorm_bwd(v, z, w, rstd, dout, dv, dz, dw)
        return dv, dz, dw, None


def gated_rmsnorm(v: torch.Tensor, z: torch.Tensor, w: torch.Tensor, eps: float = 1e-5) -> torch.Tensor:
    """rmsnorm(v * silu(z)) * w over the last dimension."""
    if _on_kernels(v, z, w) and v.shape == z.shape and v.shape[-1] <= 12288:
        return _GatedRmsNorm.apply(v, z, w, eps)
    return gated_rmsnorm_reference(v, z, w, eps)
