"""Causal linear attention with a decay for each head (no counterpart in the reference).

Projections as in MultiheadAttentionV2 (three Linear layers, one product over weights side
by side); heads are read in place from the (B*S, 3E) result. The mixer is
``kernels.linear_attention``: each head carries a head_dim x head_dim Gaussian state that
every token decays, adds k v^T to and reads with q / sqrt(head_dim).

Training runs whole sequences (``forward`` / ``backward``, from a zero state). Serving runs a
prompt and keeps the state (``prompt``), then one token at a time (``step``): the state's
size does not grow with the sequence.
"""

from __future__ import annotations

import math

import torch
from torch import Tensor

from ..kernels.common import fused_backward_delta, linear_forward
from ..kernels.linear_attention import (linear_attention, linear_attention_backward_packed, linear_attention_step)
from ._qkv import QkvProjections


def default_decays(num_heads: int) -> list[float]:
    """1 - 2^-(5 + 3 h / (H - 1)): memories of 32 to 256 tokens, evenly spread over their logarithm."""
    return [1.0 - 2.0 ** -(5.0 + 3.0 * h / max(1, num_heads - 1)) for h in range(num_heads)]


class LinearAttention(QkvProjections):
    _backward_reads = "_cache"

    def __init__(self, embed_dim: int, num_heads: int, decay=None, bias: bool = False, gain_weight: float = 1.0,
                 gain_bias: float = 1.0, init_method: str = "He", device: str = "cuda") -> None:
        """``decay``: one number in [0, 1] for every head or a sequence of num_heads;
        ``default_decays`` without."""
        if embed_dim % num_heads != 0:
            raise ValueError(f"embed_dim ({embed_dim}) must be divisible by num_heads ({num_heads})")
        if embed_dim // num_heads > 128:
            raise ValueError(f"LinearAttention supports head dimensions up to 128, got {embed_dim // num_heads}")
        if decay is None:
            decay = default_decays(num_heads)
        elif isinstance(decay, (int, float)):
            decay = [decay] * num_heads
        self.decay = tuple(float(d) for d in decay)
        if len(self.decay) != num_heads or not all(0.0 <= d <= 1.0 for d in self.decay):
            raise ValueError(f"decay: expected {num_heads} numbers in [0, 1], got {self.decay}")
        self.embed_dim = embed_dim
        self.num_heads = num_heads
        self.head_dim = embed_dim // num_heads
        self.has_bias = bias
        self.init_method = init_method
        self.gain_weight = gain_weight
        self.gain_bias = gain_bias
        self.device = torch.device(device)
        self._make_projections(embed_dim)
        self._scale = 1.0 / math.sqrt(self.head_dim)
        # on each device they were used on: the decays, and the numbers they were made from
        self._decays: dict[torch.device, tuple[Tensor, tuple]] = {}
        self._cache: dict | None = None

    def _decay_on(self, device: torch.device) -> Tensor:
        t, made_from = self._decays.get(device, (None, None))
        decay = tuple(self.decay)
        if made_from != decay:
            new = torch.tensor(decay, dtype=torch.float32, device=device)
            t = new if t is None else t.copy_(new)  # in place: recorded graphs read it
            self._decays[device] = t, decay
        return t

    def _project(self, ma: Tensor, Sa: Tensor) -> tuple[dict, list[Tensor]]:
        """What the backward reads, and the six (..., H, D) operands in place."""
        E = self.embed_dim
        if ma.shape[-1] != E:
            raise ValueError(f"Expected last dim {E}, got {ma.shape[-1]}")
        flat_m = ma.reshape(-1, E).contiguous()
        flat_S = None if Sa is None else Sa.reshape(-1, E).contiguous()
        qkv = self._qkv_params()
        w_m, w_S, b_m, b_S = (qkv.get(a) for a in self._QKV_ATTRS)
        heads = (*ma.shape[:-1], self.num_heads, self.head_dim)
        if flat_m.shape[0] == 0:  # no tokens: nothing to project
            qkv_m = qkv_S = torch.empty(0, 3 * E, device=ma.device)
        else:
            qkv_m, qkv_S = linear_forward(flat_m, flat_S, w_m, w_S, b_m, b_S)
        ops = [t[:, i * E:(i + 1) * E].view(heads) for i in range(3) for t in (qkv_m, qkv_S)]
        return dict(ma_in=flat_m, w_m=w_m, w_S=w_S, b_S=b_S), ops

    def forward(self, ma: Tensor, Sa: Tensor, lengths: Tensor | None = None) -> tuple[Tensor, Tensor]:
        """(B, S, E) moments to (B, S, E). ``lengths`` (B,): sequences of a padded batch end
        there; their later tokens get zeros and leave no deltas."""
        if ma.dim() != 3:
            raise ValueError(f"LinearAttention: expected (batch, sequence, features), got {tuple(ma.shape)}")
        cache, ops = self._project(ma, Sa)
        for p in self._projections():
            p.ma_in, p._input_shape = cache["ma_in"], ma.shape
        mo, So = linear_attention(*ops, self._decay_on(ma.device), scale=self._scale, lengths=lengths)
        self._cache = dict(cache, qkv=ops[::2], lengths=lengths)  # the means
        return mo.view(ma.shape), So.view(ma.shape)

    def backward(self, delta_mz: Tensor, delta_Sz: Tensor) -> tuple[Tensor, Tensor]:
        c = self._kept()
        q, k, v = c["qkv"]
        B, S, E = *q.shape[:2], self.embed_dim
        dm, dS = linear_attention_backward_packed(q, k, v, delta_mz.reshape(q.shape), delta_Sz.reshape(q.shape),
                                                  self._decay_on(q.device), self._scale, c["lengths"])
        dm, dS = dm.view(B * S, 3 * E), dS.view(B * S, 3 * E)
        self._projection_param_deltas(c, dm, dS)
        dma, dSa = fused_backward_delta(dm, dS, c["w_m"])  # the three projections' sum
        return dma.reshape(B, S, E), dSa.reshape(B, S, E)

    # ------------------------------------------------------------------------- serving
    def new_state(self, batch: int, device=None) -> tuple[Tensor, Tensor]:
        """The state of ``batch`` sequences before their first token."""
        shape = (batch, self.num_heads, self.head_dim, self.head_dim)
        dev = self.device if device is None else torch.device(device)
        return torch.zeros(shape, device=dev), torch.zeros(shape, device=dev)

    def prompt(self, ma: Tensor, Sa: Tensor, lengths: Tensor | None = None, state=None):
        """``forward`` from ``state`` (zeros without) that keeps nothing for a backward:
        (mo, So, the state after each sequence's last token)."""
        if ma.dim() != 3:
            raise ValueError(f"LinearAttention: expected (batch, sequence, features), got {tuple(ma.shape)}")
        _, ops = self._project(ma, Sa)
        mo, So, end = linear_attention(*ops, self._decay_on(ma.device), scale=self._scale, lengths=lengths, state=state,
                                       return_state=True)
        return mo.view(ma.shape), So.view(ma.shape), end

    def step(self, ma: Tensor, Sa: Tensor, state, active: Tensor | None = None) -> tuple[Tensor, Tensor]:
        """One token of every sequence, (B, E) or (B, 1, E); ``state`` is advanced in place.
        ``active`` (B,): sequences that are off keep their state and get zeros."""
        if ma.dim() not in (2, 3) or (ma.dim() == 3 and ma.shape[1] != 1):
            raise ValueError(f"LinearAttention.step: expected (batch, features) or (batch, 1, features), "
                             f"got {tuple(ma.shape)}")
        B = ma.shape[0]
        _, ops = self._project(ma.reshape(B, -1), None if Sa is None else Sa.reshape(B, -1))
        mo, So = linear_attention_step(*ops, state, self._decay_on(ma.device), scale=self._scale, active=active)
        return mo.view(ma.shape), So.view(ma.shape)

    def __repr__(self) -> str:
        return f"LinearAttention(embed_dim={self.embed_dim}, num_heads={self.num_heads}, bias={self.has_bias})"
