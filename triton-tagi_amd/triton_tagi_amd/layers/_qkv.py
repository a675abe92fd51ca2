"""The query, key and value projections of the attention layers.

Three Linear layers hold the parameters (the reference's layout and attributes,
triton_tagi/layers/multihead_attention.py:64-152); forward and backward run them as one
product each, over parameters that live side by side.
"""

from __future__ import annotations

import contextlib

import torch
from torch import Tensor

from .. import _overlap
from ..base import LearnableLayer
from ..kernels.common import linear_param_deltas
from ..update.parameters import update_parameters_multi
from .linear import Linear


class QkvProjections(LearnableLayer):
    """Base of the attention layers; expects embed_dim, has_bias, init_method, gain_weight,
    gain_bias and device to be set before ``_make_projections``."""

    def _make_projections(self, width: int) -> None:
        kw = dict(device=self.device, init_method=self.init_method, gain_w=self.gain_weight, gain_b=self.gain_bias,
                  bias=self.has_bias)
        self.q_proj = Linear(self.embed_dim, width, **kw)
        self.k_proj = Linear(self.embed_dim, width, **kw)
        self.v_proj = Linear(self.embed_dim, width, **kw)

    def _projections(self):
        return (self.q_proj, self.k_proj, self.v_proj)

    _QKV_ATTRS = ("mw", "Sw", "mb", "Sb")

    def _qkv_params(self) -> dict:
        """The three projections' parameters side by side: (E, 3E) weights and (1, 3E)
        biases, which the fused projection product and the update read directly. Each
        projection's mw, Sw, mb, Sb are column views of them, so in-place changes to either
        are seen by both (checkpoint restore copies in place). Built at the first forward;
        rebuilt from the projections' tensors if any of them was replaced since."""
        projs = self._projections()
        bufs = getattr(self, "_qkv", None)
        if bufs is not None and self._qkv_intact(bufs):
            return bufs
        bufs = {}
        for attr in self._QKV_ATTRS:
            parts = [getattr(p, attr) for p in projs]
            if parts[0] is None:
                continue
            buf = torch.cat(parts, 1)
            n = parts[0].shape[1]
            for i, p in enumerate(projs):
                setattr(p, attr, buf[:, i * n:(i + 1) * n])
            bufs[attr] = buf
        self._qkv = bufs
        return bufs

    def _qkv_intact(self, bufs: dict) -> bool:
        for attr, buf in bufs.items():
            n = buf.shape[1] // 3
            for i, p in enumerate(self._projections()):
                t = getattr(p, attr, None)
                if not (isinstance(t, Tensor) and t.device == buf.device and t.dtype == buf.dtype
                        and tuple(t.shape) == (buf.shape[0], n) and t.stride() == buf.stride()
                        and t.data_ptr() == buf.data_ptr() + i * n * buf.element_size()):
                    return False
        return True

    def sublayers(self) -> tuple:
        return self._projections()

    def _projection_param_deltas(self, c: dict, dqkv_m: Tensor, dqkv_S: Tensor) -> None:
        """Stores the three projections' parameter deltas, one product over the side-by-side
        deltas (B*S, 3E) of their outputs (on the side stream within a step when large).
        ``c`` holds what the forward read: ma_in, w_S, b_S."""
        E = self.embed_dim
        L = 3 * E
        dev = dqkv_m.device
        projs = self._projections()
        ma_in = c["ma_in"]
        ctx = _overlap.active()
        big = ma_in.shape[0] * E * L >= _overlap.MIN_MACS_LINEAR
        side = ctx.fork(dev, ma_in, dqkv_m, dqkv_S, c["w_S"], c["b_S"]) if ctx is not None and big else None
        with torch.cuda.stream(side) if side is not None else contextlib.nullcontext():
            dmw, dSw, dmb, dSb = linear_param_deltas(ma_in, dqkv_m, dqkv_S, c["w_S"], c["b_S"])
        # each projection's deltas are column views of the (E, 3E) ones, as its parameters
        # are of the side-by-side buffers the update applies them to
        self._qkv_deltas = (dmw, dSw, dmb, dSb)
        for i, p in enumerate(projs):
            cols = slice(i * E, (i + 1) * E)
            p.delta_mw, p.delta_Sw = dmw[:, cols], dSw[:, cols]
            if self.has_bias:
                p.delta_mb, p.delta_Sb = dmb[:, cols], dSb[:, cols]

    def _update_items(self):
        return self.q_proj._update_items() + self.k_proj._update_items() + self.v_proj._update_items()

    def _update_groups(self):
        """The update over the side-by-side buffers: two groups (weights, biases) instead
        of six, the same values element by element."""
        bufs = getattr(self, "_qkv", None)
        deltas = getattr(self, "_qkv_deltas", None)
        if bufs is None or deltas is None or not self._qkv_intact(bufs):
            return self._update_items()
        dmw, dSw, dmb, dSb = deltas
        groups = [(bufs["mw"], bufs["Sw"], dmw, dSw)]
        if self.has_bias:
            groups.append((bufs["mb"], bufs["Sb"], dmb, dSb))
        return groups

    def update(self, cap_factor: float) -> None:
        update_parameters_multi(self._update_groups(), cap_factor)

    @property
    def num_parameters(self) -> int:
        return self.q_proj.num_parameters + self.k_proj.num_parameters + self.v_proj.num_parameters
