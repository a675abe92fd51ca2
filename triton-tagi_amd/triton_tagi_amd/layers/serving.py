"""Prompts and single tokens through a list of layers with carried states.

Layers that mix tokens keep a state (LinearAttention: its own; ResidualRMSNorm: those of its
branch); layers that act on each token by itself run as they are. Anything else (attention
over a whole sequence, positional encodings, convolutions) is refused: fed token by token it
would answer wrongly.

The layers' forwards run here and replace what a backward reads, so ``Sequential`` makes every
layer forget it afterwards: a backward after a prompt or a token needs a forward of its own, and
says so.
"""

from __future__ import annotations

import torch
from torch import Tensor

from .embedding import Embedding
from .layernorm import LayerNorm
from .linear import Linear
from .linear_attention import LinearAttention
from .relu import ReLU
from .remax import Remax
from .residual_norm import ResidualRMSNorm
from .rms_norm import RMSNorm

_TOKENWISE = (Embedding, Linear, ReLU, Remax, RMSNorm, LayerNorm)


def check_layers(layers) -> None:
    for layer in layers:
        if isinstance(layer, ResidualRMSNorm):
            check_layers(layer.layers)
        elif not isinstance(layer, (*_TOKENWISE, LinearAttention)):
            raise TypeError(f"{type(layer).__name__} cannot run with a carried state")


def _tokenwise(layer, ma: Tensor, Sa: Tensor | None):
    if isinstance(layer, Remax):  # rows over the last dim
        mz, Sz = layer.forward(ma.reshape(-1, ma.shape[-1]), Sa.reshape(-1, ma.shape[-1]))
        return mz.view(ma.shape), Sz.view(ma.shape)
    return layer.forward(ma, Sa)


def run_prompt(layers, ma: Tensor, Sa: Tensor | None, lengths: Tensor | None, states):
    """(ma, Sa, states) of whole sequences; ``states`` of an earlier call, or None."""
    out = []
    if states is not None and len(states) != len(layers):
        raise ValueError(f"states: {len(states)} entries for {len(layers)} layers")
    for i, layer in enumerate(layers):
        state = None if states is None else states[i]
        if isinstance(layer, LinearAttention):
            ma, Sa, state = layer.prompt(ma, Sa, lengths, state)
        elif isinstance(layer, ResidualRMSNorm):
            bm, bS, state = run_prompt(layer.layers, ma, Sa, lengths, state)
            ma, Sa = layer._close(bm, bS, ma, Sa)[:2]
        else:
            ma, Sa = _tokenwise(layer, ma, Sa)
        out.append(state)
    return ma, Sa, out


def run_step(layers, ma: Tensor, Sa: Tensor | None, states, active: Tensor | None):
    """(ma, Sa) of one token of every sequence; the states are advanced in place."""
    if len(states) != len(layers):
        raise ValueError(f"states: {len(states)} entries for {len(layers)} layers")
    for layer, state in zip(layers, states):
        if isinstance(layer, LinearAttention):
            ma, Sa = layer.step(ma, Sa, state, active)
        elif isinstance(layer, ResidualRMSNorm):
            bm, bS = run_step(layer.layers, ma, Sa, state, active)
            ma, Sa = layer._close(bm, bS, ma, Sa)[:2]
        else:
            ma, Sa = _tokenwise(layer, ma, Sa)
    return ma, Sa
