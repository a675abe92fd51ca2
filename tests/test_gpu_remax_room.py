"""The room of a served sequence is its own: max_len tokens of it, whatever else ran beside it."""

from __future__ import annotations

import pytest
import torch

from test_gpu_remax_layers import batch, network
from test_gpu_sequence_layers import near

pytestmark = pytest.mark.gpu


def test_sequences_that_take_turns(dev):
    """Each of two sequences is decoded to its last token while the other is off."""
    net = network(max_len=12, page_size=4)
    x = batch(2, 12, 3)[0].to(dev)
    mu, _ = net.forward(x)
    _, _, states = net.prompt(x[:, :2])
    state = states[1][0]
    for t in range(2, 12):
        for b in range(2):
            on = torch.arange(2, device=dev) == b
            m, _ = net.decode(x[:, t:t + 1], states, active=on)
            near(m[b, 0], mu[b, t], f"sequence {b}, token {t}")
    assert state.lengths.tolist() == [12, 12]
    off = torch.zeros(2, dtype=torch.bool, device=dev)
    for _ in range(3):  # nobody's token takes nobody's room
        net.decode(x[:, :1], states, active=off)
    for on in (None, torch.tensor([True, False], device=dev)):
        with pytest.raises(ValueError, match="max_len is 12"):
            net.decode(x[:, :1], states, active=on)
    assert state.lengths.tolist() == [12, 12]


def test_one_sequence_goes_on_beside_a_full_one(dev):
    net = network(max_len=12, page_size=4)
    x = batch(2, 12, 3)[0].to(dev)
    mu, _ = net.forward(x)
    _, _, states = net.prompt(x, lengths=torch.tensor([12, 5], device=dev))
    on = torch.tensor([False, True], device=dev)
    for t in range(5, 12):
        near(net.decode(x[:, t:t + 1], states, active=on)[0][1, 0], mu[1, t], f"token {t}")
    with pytest.raises(ValueError, match="max_len is 12"):
        net.decode(x[:, :1], states, active=on)


def test_ragged_prompts_up_to_the_room(dev):
    """Padded widths add up to more than a sequence's room, its own tokens do not."""
    net = network(max_len=40)
    x = batch(2, 40, 3)[0].to(dev)
    mu, _ = net.forward(x)
    _, _, states = net.prompt(x[:, :12], lengths=torch.tensor([12, 5], device=dev))
    # the second sequence's next 30 tokens, none of the first's
    pm, _, more = net.prompt(x[:, 5:35], lengths=torch.tensor([0, 30], device=dev), states=states)
    near(pm[1], mu[1, 5:35], "second prompt")
    assert not pm[0].isnan().any() and more[1][0].lengths.tolist() == [12, 35]
    pm, _, last = net.prompt(x[:, 12:40], lengths=torch.tensor([28, 5], device=dev), states=more)
    near(pm[0], mu[0, 12:40], "third prompt")
    assert last[1][0].lengths.tolist() == [40, 40]
    with pytest.raises(ValueError, match="max_len is 40"):
        net.prompt(x[:, :7], lengths=torch.tensor([1, 6], device=dev), states=more)
    # a first prompt padded beyond the room
    wide = torch.cat([x, x], 1)
    pm, _, first = net.prompt(wide, lengths=torch.tensor([40, 7], device=dev))
    near(pm[0, :40], mu[0], "padded"), near(pm[1, :7], mu[1, :7], "padded")
    assert first[1][0].lengths.tolist() == [40, 7]
    with pytest.raises(ValueError, match="max_len is 40"):
        net.prompt(wide, lengths=torch.tensor([41, 7], device=dev))


def test_a_recorded_token_beside_a_full_sequence(dev):
    """Who takes part in a replay is not known when it is recorded."""
    net = network(max_len=12, page_size=4)
    x = batch(2, 12, 3)[0].to(dev)
    mu, _ = net.forward(x)
    lengths = torch.tensor([12, 5], device=dev)
    tok, on = x[:, 5:6].clone(), torch.tensor([False, True], device=dev)
    net.decode(tok, net.prompt(x, lengths=lengths)[2], active=on)
    _, _, states = net.prompt(x, lengths=lengths)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m, _ = net.decode(tok, states, active=on)
    for t in range(5, 12):
        tok.copy_(x[:, t:t + 1])
        graph.replay()
        near(m[1, 0], mu[1, t], f"token {t}")
    assert states[1][0].lengths.tolist() == [12, 12]
    with pytest.raises(ValueError, match="max_len is 12"):
        net.decode(tok, states, active=on)
