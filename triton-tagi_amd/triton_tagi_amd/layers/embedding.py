"""Bayesian Embedding (mirrors triton_tagi/layers/embedding.py:39-168).

Forward: (mu, S) = (mw[cat], Sw[cat]) for the integer ids carried in ``ma`` (cast toward
zero, like ``.long()``); ids equal to padding_idx give zeros. Backward accumulates
delta_mw[cat] += delta_mu * Sw[cat], delta_Sw[cat] += delta_S * Sw[cat]^2 and returns
zero input deltas (the index is discrete).

Two additions without a counterpart in the reference: ``output_scale`` c multiplies the
moments looked up (means by c, variances by c^2; with it the deltas sum c delta_mu Sw and
(c Sw)^2 delta_S), and ``sorted_deltas`` forms the deltas by sorting the tokens instead of
scanning them once per category, which a large table needs. Within ``update_in_backward``
the sorted form applies the capped update to the rows that occur as it forms their deltas;
the deltas of the whole table are stored as well unless its ``keep_deltas`` is false.
"""

from __future__ import annotations

import math

import torch
from torch import Tensor

from .. import _lib
from ..base import LearnableLayer
from ..kernels.embedding import embedding_lookup, embedding_param_deltas, embedding_update
from ..param_init import gaussian_param_init
from ..update import in_backward
from ..update.parameters import update_parameters


class Embedding(LearnableLayer):
    _backward_reads = "cat_idx"

    def __init__(self, num_embeddings: int, embedding_dim: int, input_size: int = 0, scale: float = 1.0,
                 padding_idx: int = -1, device: str = "cuda", output_scale: float = 1.0,
                 sorted_deltas: bool | None = None) -> None:
        """``sorted_deltas``: None takes the sorted form where ``output_scale`` is not 1 (the
        scan knows no scale) and the scan otherwise. The sorted form also takes integer ids."""
        output_scale = float(output_scale)
        if not math.isfinite(output_scale):
            raise ValueError(f"output_scale must be finite, got {output_scale}")
        if sorted_deltas is None:
            sorted_deltas = output_scale != 1.0
        if not sorted_deltas and output_scale != 1.0:
            raise ValueError("an output_scale needs sorted_deltas")
        self.output_scale = output_scale
        self.sorted_deltas = bool(sorted_deltas)
        self.num_embeddings = num_embeddings
        self.embedding_dim = embedding_dim
        self.input_size = input_size
        self.scale = scale
        self.padding_idx = padding_idx
        self.device = torch.device(device)
        self.has_bias = False
        self.mw, self.Sw = gaussian_param_init(scale, 1.0, (num_embeddings, embedding_dim), device=self.device)
        self.mb = self.Sb = None
        self.cat_idx: Tensor | None = None  # float token ids as given
        self.delta_mw = self.delta_Sw = self.delta_mb = self.delta_Sb = None

    def forward(self, ma: Tensor, Sa: Tensor) -> tuple[Tensor, Tensor]:
        if ma.dim() == 3 and ma.shape[-1] == 1:
            ma = ma.squeeze(-1)
        if self.sorted_deltas:
            self.cat_idx = ma.contiguous()
            return embedding_lookup(self.cat_idx, self.mw, self.Sw, self.output_scale, self.padding_idx)
        tokens = _lib.check(ma.contiguous(), "ma")
        self.cat_idx = tokens
        D = self.embedding_dim
        mz = torch.empty(*tokens.shape, D, device=tokens.device, dtype=torch.float32)
        Sz = torch.empty_like(mz)
        _lib.call("tagi_embedding_fwd", tokens.data_ptr(), self.mw.data_ptr(), self.Sw.data_ptr(), mz.data_ptr(),
                  Sz.data_ptr(), tokens.numel(), self.num_embeddings, D, int(self.padding_idx),
                  _lib.stream_of(tokens))
        return mz, Sz

    def backward(self, delta_mz: Tensor, delta_Sz: Tensor) -> tuple[Tensor, Tensor]:
        tokens = self.backward_param_deltas(delta_mz, delta_Sz)
        zeros = torch.zeros(tokens.shape, device=tokens.device, dtype=delta_mz.dtype)
        return zeros, zeros.clone()

    def backward_param_deltas(self, delta_mz: Tensor, delta_Sz: Tensor):
        """The parameter deltas of ``backward`` without the (zero) deltas of the token ids;
        returns the ids."""
        tokens = self._kept()
        if self.sorted_deltas:
            upd = in_backward.active()
            if upd is not None:
                self.delta_mw, self.delta_Sw = embedding_update(
                    tokens, delta_mz, delta_Sz, self.mw, self.Sw, upd.cap_factor, self.output_scale, self.padding_idx,
                    upd.keep_deltas)
            else:
                self.delta_mw, self.delta_Sw = embedding_param_deltas(
                    tokens, delta_mz, delta_Sz, self.Sw, self.output_scale, self.padding_idx)
            self._updated_in_backward = upd is not None
            return tokens
        D = self.embedding_dim
        dm = _lib.check(delta_mz.reshape(-1, D).contiguous(), "delta_mz")
        dS = _lib.check(delta_Sz.reshape(-1, D).contiguous(), "delta_Sz")
        n = tokens.numel()
        self.delta_mw = torch.empty_like(self.mw)
        self.delta_Sw = torch.empty_like(self.Sw)
        ws = _lib.workspace(_lib.query("tagi_embedding_bwd_ws_bytes", n, self.num_embeddings, D), dm.device)
        wp, wb = _lib.ws_args(ws)
        _lib.call("tagi_embedding_bwd", tokens.data_ptr(), dm.data_ptr(), dS.data_ptr(), self.Sw.data_ptr(),
                  self.delta_mw.data_ptr(), self.delta_Sw.data_ptr(), n, self.num_embeddings, D,
                  int(self.padding_idx), wp, wb, _lib.stream_of(dm))
        return tokens

    def _update_items(self):
        return [(self.mw, self.Sw, self.delta_mw, self.delta_Sw)]

    def update(self, cap_factor: float) -> None:
        if self._updated_in_backward:  # the backward pass applied it (update_in_backward)
            self._updated_in_backward = False
            return
        update_parameters(self.mw, self.Sw, self.delta_mw, self.delta_Sw, cap_factor)

    @property
    def num_parameters(self) -> int:
        return 2 * self.mw.numel()

    def __repr__(self) -> str:
        return (f"Embedding(num_embeddings={self.num_embeddings}, embedding_dim={self.embedding_dim}, "
                f"padding_idx={self.padding_idx}, scale={self.scale})")
