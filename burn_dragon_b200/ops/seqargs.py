"""Argument checks shared by the operators over padded sequences (`mamba_ops.causal_conv`, `norm_rotate`, `selective_scan`)."""
from __future__ import annotations

from typing import Optional

import torch

from . import native

KERNEL_TYPES = (torch.float32, torch.float16, torch.bfloat16)


def on_kernels(t: torch.Tensor) -> bool:
    """Do calls with this tensor run on the CUDA kernels? (float64 and CPU tensors take the torch statement.)"""
    return t.is_cuda and t.dtype in KERNEL_TYPES and native.load()


def check_like(t: Optional[torch.Tensor], ref: torch.Tensor, shape: tuple, name: str, dtype: Optional[torch.dtype] = None) -> None:
    """`t` (or None) has this shape, is on the device of `ref`, and is of `dtype` (None: any floating type)."""
    if t is None:
        return
    if t.shape != shape:
        raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.device != ref.device:
        raise ValueError(f"{name} is on {t.device}, expected {ref.device}")
    if (t.dtype is not dtype) if dtype is not None else not t.is_floating_point():
        raise ValueError(f"{name}: expected {dtype if dtype is not None else 'a floating type'}, got {t.dtype}")


def check_lengths(lengths: Optional[torch.Tensor], ref: torch.Tensor, B: int) -> Optional[torch.Tensor]:
    """int32 / int64 [B] on the device of `ref`, contiguous. Values are not read here (that would wait for the device);
    every path takes a value outside [0, T] as the nearer of the two."""
    if lengths is None:
        return None
    if lengths.shape != (B,):
        raise ValueError(f"lengths: expected shape {(B,)}, got {tuple(lengths.shape)}")
    if lengths.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"lengths: expected int32 or int64, got {lengths.dtype}")
    if lengths.device != ref.device:
        raise ValueError(f"lengths is on {lengths.device}, expected {ref.device}")
    return lengths.contiguous()


def check_active(active: Optional[torch.Tensor], ref: torch.Tensor, B: int) -> Optional[torch.Tensor]:
    if active is None:
        return None
    check_like(active, ref, (B,), "active", torch.bool)
    return active.contiguous()


def valid_rows(lengths: Optional[torch.Tensor], B: int, T: int, device) -> Optional[torch.Tensor]:
    """[B, T] truth values, or None where every row counts."""
    if lengths is None:
        return None
    return torch.arange(T, device=device) < lengths.clamp(0, T)[:, None]


def adjacent(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """The tensor with elements of its last dimension adjacent (a copy only where they are not)."""
    return t if t is None or t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def dense_f32(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """A parameter as the kernels read it."""
    if t is None or (t.dtype is torch.float32 and t.is_contiguous()):
        return t
    return t.float().contiguous()


def wants_grad(*ts: Optional[torch.Tensor]) -> bool:
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return False


def _meet(delta: int, dims: list) -> bool:
    """Do two tensors of these (stride, size) meet, `delta` elements apart? Strides fall and no row overlaps another."""
    if not dims:
        return delta == 0
    (st, n), rest = dims[0], dims[1:]
    return any(abs(k) < n and _meet(delta - k * st, rest) for k in (delta // st, delta // st + 1))


def check_out(out: Optional[torch.Tensor], src: torch.Tensor, name: str) -> None:
    """`out` of a single-token step: shaped like the state, which it may be; memory it shares with the state otherwise would
    be overwritten before it is read."""
    if out is None:
        return
    check_like(out, src, src.shape, name, src.dtype)
    if torch.is_grad_enabled() and out.requires_grad:
        raise ValueError(f"{name} requires a gradient; a step form has none")
    sizes = out.shape
    strides = [st if n > 1 else 0 for st, n in zip(out.stride(), sizes)]             # (a stride that is never taken means nothing)
    from_strides = [st if n > 1 else 0 for st, n in zip(src.stride(), sizes)]
    same = out.data_ptr() == src.data_ptr() and strides == from_strides
    dims = sorted((st, n) for st, n in zip(strides, out.shape) if n > 1)
    reach = 1                                            # elements that the dimensions of smaller stride span
    for st, n in dims:
        if st < reach:
            raise ValueError(f"{name}: its rows overlap one another")
        reach = st * (n - 1) + reach
    if same or not out.numel():
        return
    # by their addresses: two storages may be made over the same memory
    span = lambda t: (t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum((n - 1) * st for n, st in zip(t.shape, t.stride()))))  # noqa: E731
    (a0, a1), (b0, b1) = span(out), span(src)
    if a1 <= b0 or b1 <= a0:
        return
    if strides == from_strides:                          # slices of one buffer, which may interleave
        delta, odd = divmod(out.data_ptr() - src.data_ptr(), out.element_size())
        if not (odd or _meet(delta, dims[::-1])):
            return
    raise ValueError(f"{name} overlaps the state without being it")
