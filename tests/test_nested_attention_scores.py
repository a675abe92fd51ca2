"""Sequential.get_attention_scores over attention layers at the top and inside residual blocks."""

from __future__ import annotations

import pytest
import torch

from triton_tagi_amd import Linear, LinearAttention, MultiheadAttentionV2, ResidualRMSNorm, Sequential

E = 4


def attention(value):
    layer = MultiheadAttentionV2(E, 2, 3, device="cpu")
    layer._attn_mu, layer._attn_var = torch.full((1,), value), torch.full((1,), -value)  # as a forward leaves them
    return layer


def test_layers_inside_blocks_are_found():
    kw = dict(device="cpu")
    net = Sequential([
        attention(1.0),
        ResidualRMSNorm([Linear(E, E, **kw), attention(2.0)], E, **kw),
        ResidualRMSNorm([ResidualRMSNorm([attention(3.0)], E, **kw), attention(4.0)], E, **kw),
        ResidualRMSNorm([LinearAttention(E, 2, **kw)], E, **kw),
        attention(5.0),
    ], device="cpu")
    got = net.get_attention_scores()
    assert {k: (m.item(), v.item()) for k, (m, v) in got.items()} == {
        0: (1.0, -1.0), (1, 1): (2.0, -2.0), (2, 0, 0): (3.0, -3.0), (2, 1): (4.0, -4.0), 4: (5.0, -5.0)}


def test_networks_without_attention_scores_say_so():
    kw = dict(device="cpu")
    net = Sequential([Linear(E, E, **kw), ResidualRMSNorm([LinearAttention(E, 2, **kw)], E, **kw)], device="cpu")
    with pytest.raises(RuntimeError, match="No attention layers"):
        net.get_attention_scores()
    net = Sequential([ResidualRMSNorm([MultiheadAttentionV2(E, 2, 3, **kw)], E, **kw)], device="cpu")
    with pytest.raises(RuntimeError, match="forward first"):
        net.get_attention_scores()
