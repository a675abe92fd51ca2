"""Residual connection with RMSNorm around a branch of layers (no counterpart in the
reference, whose residual block (triton_tagi/layers/resblock.py:216-472) is convolutional).

    z = RMSNorm(x + branch(x))

The sum and the norm are one pass (``kernels.add_rms_norm``); backward, the deltas at the sum
go to the branch and, beside it, to the input, and what comes back is added.
"""

from __future__ import annotations

from torch import Tensor

from ..base import LearnableLayer
from ..kernels.residual_norm import add_rms_norm, add_rms_norm_backward
from ..update.parameters import update_layers
from .resblock import delta_merge
from .rms_norm import RMSNorm


class ResidualRMSNorm(LearnableLayer):
    _backward_reads = "_sum"

    def __init__(self, layers: list, normalized_shape, eps: float = 1e-6, gain_w: float = 1.0,
                 device: str = "cuda") -> None:
        self.layers = list(layers)
        self.norm = RMSNorm(normalized_shape, eps=eps, gain_w=gain_w, device=device)
        self.device = self.norm.device
        self.training = True
        self._sum: tuple[Tensor, Tensor] | None = None  # the sum's means and 1/rms

    def sublayers(self) -> tuple:
        return (*self.layers, self.norm)

    def _learnable_layers(self) -> list:
        return [layer for layer in self.sublayers() if isinstance(layer, LearnableLayer)]

    @property
    def _learnable(self) -> list:
        """The layers that hold tensors of their own, nested ones in place (what a checkpoint
        saves, in this order)."""
        out = []
        for layer in self._learnable_layers():
            nested = getattr(layer, "_learnable", None)
            if nested is None:
                nested = [p for p in layer.sublayers() if isinstance(p, LearnableLayer)] or [layer]
            out.extend(nested)
        return out

    def train(self) -> None:
        self.training = True
        for layer in self.sublayers():
            if hasattr(layer, "training"):
                layer.train()

    def eval(self) -> None:
        self.training = False
        for layer in self.sublayers():
            if hasattr(layer, "training"):
                layer.eval()

    def _close(self, bm: Tensor, bS: Tensor, ma: Tensor, Sa: Tensor):
        if bm.shape != ma.shape:
            raise ValueError(f"ResidualRMSNorm: the branch maps {tuple(ma.shape)} to {tuple(bm.shape)}")
        n = self.norm
        return add_rms_norm(bm, bS, ma, Sa, n.mw, n.Sw, n.eps, need_sum_var=False)

    def forward(self, ma: Tensor, Sa: Tensor) -> tuple[Tensor, Tensor]:
        from .fused import forward_chain

        bm, bS = forward_chain(self.layers, ma, Sa)
        mz, Sz, ms, _, inv = self._close(bm, bS, ma, Sa)
        self._sum = (ms, inv)
        return mz, Sz

    def backward(self, delta_mz: Tensor, delta_Sz: Tensor) -> tuple[Tensor, Tensor]:
        from .fused import backward_chain

        ms, inv = self._kept()
        n = self.norm
        dm, dS, n.delta_mw, n.delta_Sw = add_rms_norm_backward(delta_mz.reshape(ms.shape), delta_Sz.reshape(ms.shape),
                                                               ms, inv, n.mw, n.Sw)
        om, oS = backward_chain(self.layers, dm, dS)
        if om.data_ptr() == dm.data_ptr():  # layers that pass their deltas on unchanged
            om, oS = om.clone(), oS.clone()
        om, oS = om.reshape(ms.shape).contiguous(), oS.reshape(ms.shape).contiguous()
        delta_merge(dm, dS, om, oS)
        return om, oS

    # ---------------------------------------------------------------------------- update
    def _update_items(self):
        items = []
        for layer in self._learnable_layers():
            got = layer._update_items()
            if got is None:
                return None
            items.extend(got)
        return items

    def _update_parts(self):
        return self._learnable_layers()

    def _update_groups(self):
        """Groups of every layer inside; None (all through ``update``) where a layer has none or
        its backward applied its update."""
        items = []
        for layer in self._learnable_layers():
            got = None if layer._updated_in_backward else layer._update_groups()
            if got is None:
                return None
            items.extend(got)
        return items

    def update(self, cap_factor: float) -> None:
        update_layers(self._learnable_layers(), cap_factor)

    @property
    def num_parameters(self) -> int:
        return sum(layer.num_parameters for layer in self._learnable_layers())

    def __repr__(self) -> str:
        return f"ResidualRMSNorm({self.layers}, normalized_shape={self.norm.normalized_shape})"
