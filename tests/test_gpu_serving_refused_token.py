"""A refused token leaves every layer's state alone, so that the caller can go on without the sequence
that is full: layers before the one that refuses had taken the token already."""

from __future__ import annotations

import math

import pytest
import torch

from test_gpu_remax_layers import E, G, H, V, batch
from test_gpu_sequence_layers import near

pytestmark = pytest.mark.gpu


def network(first):
    from triton_tagi_amd import Embedding, Linear, RemaxAttention, ResidualRMSNorm, Sequential

    torch.manual_seed(0)
    cpu = dict(device="cpu")
    return Sequential([
        Embedding(V, E, scale=0.25, output_scale=math.sqrt(E), **cpu),
        ResidualRMSNorm([first(cpu), Linear(E, E, gain_w=0.5, **cpu)], E, **cpu),
        ResidualRMSNorm([RemaxAttention(E, H, G, max_len=6, page_size=4, gain_weight=0.5, **cpu),
                         Linear(E, E, gain_w=0.5, **cpu)], E, **cpu),
        Linear(E, V, **cpu),
    ], device="cuda:0")


def linear(cpu):
    from triton_tagi_amd import LinearAttention

    return LinearAttention(E, H, bias=True, gain_weight=0.5, **cpu)


def longer(cpu):
    from triton_tagi_amd import RemaxAttention

    return RemaxAttention(E, H, G, max_len=20, page_size=4, gain_weight=0.5, **cpu)


@pytest.mark.parametrize("first", [linear, longer])
def test_the_others_go_on(first, dev):
    net = network(first)
    x = batch(2, 6, 3)[0].clamp_min(1).to(dev)
    mu, var = net.forward(x)
    _, _, states = net.prompt(x, lengths=torch.tensor([6, 3], device=dev))
    on = torch.tensor([False, True], device=dev)
    for t in range(3, 6):
        for _ in range(2):
            with pytest.raises(ValueError, match="max_len is 6"):
                net.decode(x[:, t:t + 1], states)
        m, S = net.decode(x[:, t:t + 1], states, active=on)
        near(m[1, 0], mu[1, t], f"token {t}"), near(S[1, 0], var[1, t], f"token {t}")
    with pytest.raises(ValueError, match="max_len is 6"):
        net.decode(x[:, :1], states, active=on)


def test_states_of_another_batch(dev):
    net = network(linear)
    x = batch(2, 6, 3)[0].clamp_min(1).to(dev)
    mu, _ = net.forward(x)
    _, _, states = net.prompt(x[:, :3])
    other = net.prompt(x[:1, :3])[2]
    with pytest.raises(ValueError, match="AttentionState of 2"):
        net.decode(x[:, 3:4], [states[0], states[1], other[2], states[3]])
    near(net.decode(x[:, 3:4], states)[0][:, 0], mu[:, 3], "token")
