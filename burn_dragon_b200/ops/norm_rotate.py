"""RMS norm of every query and key head together with its rotation, in one pass (`csrc/norm_rotate.cuh`).

    v = x / sqrt(mean x^2 + eps) * weight + bias          over the Dh channels of a head
    (o_2i, o_2i+1) = (v_2i cos - v_2i+1 sin, v_2i+1 cos + v_2i sin)     for the first pairs; the other channels stay

The angle of a pair comes from the token's position, 2 pi frac(position * freq) with `freqs` as
`reference.build_freqs(..., "rope")` makes them, or is given for every token (the cumulative, learned angles of a
state-space layer whose C and B are the queries and keys). Gradients: q, k, weights, biases, angles.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch

from . import native
from . import seqargs as A


def _turn(v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    n = 2 * cos.shape[-1]
    a, b = v[..., 0:n:2], v[..., 1:n:2]
    return torch.cat((torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2), v[..., n:]), -1)


def _angles_at(positions, freqs: torch.Tensor, B: int, T: int) -> torch.Tensor:
    """[B, T, pairs] in float64: 2 pi frac(position * freq)"""
    pos = positions if isinstance(positions, torch.Tensor) else positions + torch.arange(T, device=freqs.device)
    turns = pos.double()[..., None] * freqs[0::2].double()
    return ((turns - turns.floor()) * (2 * math.pi)).expand(B, T, -1)


def norm_rotate_reference(q, k=None, q_weight=None, k_weight=None, q_bias=None, k_bias=None, *, angles=None, freqs=None, positions=0,
                          lengths=None, eps: float = 1e-5):
    """Torch statement of `norm_rotate` (any device and floating type, differentiable)."""
    B, T = q.shape[:2]
    ct = torch.promote_types(q.dtype, torch.float32)
    if angles is None and freqs is not None:
        angles = _angles_at(positions, freqs, B, T)
    keep = A.valid_rows(lengths, B, T, q.device)
    keep = keep[..., None, None] if keep is not None else None
    outs = []
    for x, w, b in ((q, q_weight, q_bias), (k, k_weight, k_bias)):
        if x is None:
            outs.append(None)
            continue
        xs = x.to(ct) if keep is None else torch.where(keep, x.to(ct), 1.0)     # (1: a norm that exists without eps too)
        v = xs * torch.rsqrt(xs.square().mean(-1, keepdim=True) + eps)
        v = v * w.to(ct) if w is not None else v
        v = v + b.to(ct) if b is not None else v
        if angles is not None:
            an = angles.to(torch.promote_types(angles.dtype, torch.float32))
            an = an if keep is None else torch.where(keep[..., 0], an, 0.0)
            v = _turn(v, an.cos().to(ct)[:, :, None], an.sin().to(ct)[:, :, None])
        outs.append((v if keep is None else torch.where(keep, v, 0.0)).to(x.dtype))
    return tuple(outs)


def norm_rotate(q: torch.Tensor, k: Optional[torch.Tensor] = None, q_weight: Optional[torch.Tensor] = None,
                k_weight: Optional[torch.Tensor] = None, q_bias: Optional[torch.Tensor] = None, k_bias: Optional[torch.Tensor] = None, *,
                angles: Optional[torch.Tensor] = None, freqs: Optional[torch.Tensor] = None,
                positions: Union[int, torch.Tensor] = 0, lengths: Optional[torch.Tensor] = None,
                eps: float = 1e-5) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """RMS norm and rotation of q [B, T, Hq, Dh] and k [B, T, Hk, Dh] (or None): -> (q', k'), contiguous, in their type.
    Rows are fp32, fp16 or bf16 and may be views into a wider projection (channels adjacent); Dh is even and at most
    512. Weights and biases: [Dh] for all heads or [heads, Dh], all of them alike (None: 1 and 0).
    Rotation, if any: `angles` [B, T, pairs] in radians (of any floating type, as exact as that type has them), or `freqs`
    [2 * pairs] in cycles per position with `positions` - the first token's (an int), or [T] or [B, T] integers (the single-token form has T = 1 and one position a stream).
    `lengths` [B]: rows behind a sequence's length give 0 and take no part in any gradient. The kernels refuse second
    derivatives and forward-mode tangents."""
    if not (q.dim() == 4 and q.is_floating_point()):
        raise ValueError(f"q: expected a floating [B, T, heads, Dh] tensor, got {q.dtype} {tuple(q.shape)}")
    B, T, Hq, Dh = q.shape
    if not (Hq >= 1 and Dh >= 2 and Dh % 2 == 0 and Dh <= 512):
        raise ValueError(f"q: expected at least one head and an even Dh up to 512, got {tuple(q.shape)}")
    if not (k is None or (k.dim() == 4 and k.shape[2] >= 1)):
        raise ValueError("k: expected [B, T, heads, Dh]")
    Hk = k.shape[2] if k is not None else 0
    A.check_like(k, q, (B, T, Hk, Dh), "k", q.dtype)
    if not (k is not None or (k_weight is None and k_bias is None)):
        raise ValueError("k_weight and k_bias come with k")
    params = ((q_weight, Hq, "q_weight"), (k_weight, Hk, "k_weight"), (q_bias, Hq, "q_bias"), (k_bias, Hk, "k_bias"))
    per_head = any(t is not None and t.dim() == 2 for t, _, _ in params)
    for t, H, name in params:
        A.check_like(t, q, (H, Dh) if per_head else (Dh,), name)
    if not (angles is None or freqs is None):
        raise ValueError("angles and freqs: one of the two at most")
    pos0 = 0
    if angles is not None:
        if not (angles.dim() == 3 and 2 * angles.shape[2] <= Dh):
            raise ValueError(f"angles: expected [B, T, pairs] with pairs up to {Dh // 2}, got {tuple(angles.shape)}")
        A.check_like(angles, q, (B, T, angles.shape[2]), "angles")
        if not (isinstance(positions, int) and positions == 0):
            raise ValueError("positions come with freqs")
    elif freqs is not None:
        if not (freqs.dim() == 1 and freqs.shape[0] % 2 == 0 and freqs.shape[0] <= Dh):
            raise ValueError(f"freqs: expected an even number up to {Dh}, got {tuple(freqs.shape)}")
        A.check_like(freqs, q, freqs.shape, "freqs")
        if A.wants_grad(freqs):
            raise ValueError("freqs has no gradient; pass angles")
        if isinstance(positions, torch.Tensor):
            if not (positions.dtype in (torch.int32, torch.int64)):
                raise ValueError(f"positions: expected int32 or int64, got {positions.dtype}")
            if not (tuple(positions.shape) in ((T,), (B, T))):
                raise ValueError(f"positions: expected {(T,)} or {(B, T)}, got {tuple(positions.shape)}")
            if not (positions.device == q.device):
                raise ValueError(f"positions is on {positions.device}, expected {q.device}")
        else:
            pos0 = int(positions)
    else:
        if not (isinstance(positions, int) and positions == 0):
            raise ValueError("positions come with freqs")
    lengths = A.check_lengths(lengths, q, B)
    if not A.on_kernels(q):
        return norm_rotate_reference(q, k, q_weight, k_weight, q_bias, k_bias, angles=angles, freqs=freqs, positions=positions,
                                     lengths=lengths, eps=eps)
    if not (B * T <= 1 << 30):
        raise ValueError("more than 2^30 tokens")
    pos = None
    if freqs is not None and freqs.dtype is torch.float64:      # (the kernel has them in 32 bits)
        angles, freqs, positions, pos0 = _angles_at(positions, freqs, B, T), None, 0, 0
    if angles is not None and angles.dtype is torch.float64:
        angles = torch.remainder(angles, 2 * math.pi)    # before the kernel's 32 bits, which leave little of a large angle
    if isinstance(positions, torch.Tensor):
        pos = positions if positions.dim() == 2 else positions.expand(B, T)
    out = native.ops.norm_rotate(
        A.adjacent(q), A.adjacent(k), A.dense_f32(q_weight), A.dense_f32(k_weight), A.dense_f32(q_bias), A.dense_f32(k_bias),
        A.adjacent(angles.float()) if angles is not None else None, A.dense_f32(freqs), pos, pos0, lengths, float(eps))
    return out[0], (out[1] if k is not None else None)
