"""Checks and layouts of the attention operators' operands."""

from __future__ import annotations

import math

import torch
from torch import Tensor

from .. import _lib


def pair(m: Tensor, S: Tensor, name: str, ref: Tensor, shape) -> tuple[Tensor, Tensor]:
    """A mean and its variance in one layout with a unit last stride."""
    if (isinstance(m, Tensor) and isinstance(S, Tensor) and m.dtype is torch.float32 and S.dtype is torch.float32
            and m.get_device() == ref.get_device() == S.get_device() and m.shape == shape == S.shape):
        st = m.stride()
        if st == S.stride() and (st[-1] == 1 or shape[-1] == 1):
            return m, S
    _lib.check_with(m, "m" + name, ref, shape)
    _lib.check_with(S, "S" + name, ref, shape)
    if m.stride() != S.stride() or (m.stride(-1) != 1 and m.shape[-1] != 1):
        m, S = m.contiguous(), S.contiguous()
    return m, S


def mean(m: Tensor, name: str, ref: Tensor, shape) -> Tensor:
    _lib.check_with(m, "m" + name, ref, shape)
    return m if m.stride(-1) == 1 or m.shape[-1] == 1 else m.contiguous()


def heads(t: Tensor) -> _lib.Heads:
    st = t.stride()
    return _lib.Heads(st[0], st[1], st[2]) if t.dim() == 4 else _lib.Heads(st[0], 0, st[1])


def dense_like(t: Tensor, shape) -> Tensor:
    """An output of t's shape, dense (the shorter way to it where t is)."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(shape)


def written(ts, names, ref: Tensor, shape) -> None:
    """Outputs of a caller's: one layout with a unit last stride, every element its own place."""
    for t, n in zip(ts, names):
        _lib.check_with(t, n, ref, shape)
        st = t.stride()
        if st != ts[0].stride() or (st[-1] != 1 and shape[-1] > 1):
            raise ValueError(f"{', '.join(names)}: expected one layout with a last stride of 1, {n} has {st}")
        if any(k == 0 and m > 1 for k, m in zip(st, shape)):
            raise ValueError(f"{n}: an output's elements share their places, strides are {st}")


def shape_of(t: Tensor, name: str, dims: int) -> torch.Size:
    _lib.check(t, name, contiguous=False)
    if t.dim() != dims or min(t.shape[-2:]) == 0:
        what = "(B, T, H, D)" if dims == 4 else "(B, H, D)"
        raise ValueError(f"{name}: expected {what} with heads and features, got {tuple(t.shape)}")
    return t.shape


def finite_scale(scale: float) -> float:
    scale = float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    return scale


def counts(t: Tensor | None, name: str, ref: Tensor, B: int) -> tuple[Tensor | None, int]:
    """One integer a sequence, and its bytes (0 without a tensor)."""
    if t is None:
        return None, 0
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name}: expected an int32 or int64 tensor")
    if t.device != ref.device or tuple(t.shape) != (B,):
        raise ValueError(f"{name}: expected ({B},) on {ref.device}, got {tuple(t.shape)} on {t.device}")
    return t.contiguous(), t.element_size()


def key_heads(G: int, H: int) -> None:
    if H % G:
        raise ValueError(f"{H} query heads cannot share {G} key heads evenly")
