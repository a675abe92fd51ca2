"""States that recorded tokens advance, used afterwards by calls that are not recorded.

A replay advances the lengths on the GPU and not the host's count of them, so what follows must not go by
that count: a token and a prompt after replays see every key, and the room is that of the lengths.
"""

from __future__ import annotations

import pytest
import torch

from test_gpu_remax_layers import batch, network
from test_gpu_sequence_layers import near

pytestmark = pytest.mark.gpu


def recorded_token(net, states, tok, warm):
    """A graph of one token on ``states``; ``warm``: states of the same sizes that it may spoil."""
    net.decode(tok, warm)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = net.decode(tok, states)
    return graph, out


@pytest.mark.parametrize("replays", [6, 300])
def test_eager_calls_after_replays(dev, replays):
    net = network(max_len=400)
    n = 10 + replays
    x = batch(3, n + 8, 8)[0].to(dev)
    mu, var = net.forward(x)
    _, _, states = net.prompt(x[:, :10])
    tok = x[:, 10:11].clone()
    graph, (m, S) = recorded_token(net, states, tok, net.prompt(x[:, :10])[2])
    for t in range(10, n):
        tok.copy_(x[:, t:t + 1])
        graph.replay()
    near(m[:, 0], mu[:, n - 1], "the last replay")
    state = states[1][0]
    assert state.lengths.tolist() == [n] * 3
    # a prompt that continues, and a copy that is decoded
    pm, pS, more = net.prompt(x[:, n:n + 4], states=states)
    near(pm, mu[:, n:n + 4], "prompt"), near(pS, var[:, n:n + 4], "prompt")
    m1, S1 = net.decode(x[:, n + 4:n + 5], more)
    near(m1[:, 0], mu[:, n + 4], "token after the prompt"), near(S1[:, 0], var[:, n + 4], "token after the prompt")
    # the state itself: an eager token, a replay, an eager token
    m2, S2 = net.decode(x[:, n:n + 1], states)
    near(m2[:, 0], mu[:, n], "eager token"), near(S2[:, 0], var[:, n], "eager token")
    tok.copy_(x[:, n + 1:n + 2])
    graph.replay()
    near(m[:, 0], mu[:, n + 1], "replay"), near(S[:, 0], var[:, n + 1], "replay")
    m3, _ = net.decode(x[:, n + 2:n + 3], states)
    near(m3[:, 0], mu[:, n + 2], "eager token after it")
    assert state.lengths.tolist() == [n + 3] * 3


def test_the_room_after_replays(dev):
    net = network(max_len=16)
    x = batch(2, 20, 8)[0].to(dev)
    _, _, states = net.prompt(x[:, :4])
    tok = x[:, 4:5].clone()
    graph, _ = recorded_token(net, states, tok, net.prompt(x[:, :4])[2])
    for _ in range(11):
        graph.replay()
    with pytest.raises(ValueError, match="max_len is 16"):
        net.prompt(x[:, 15:17], states=states)
    net.decode(x[:, 15:16], states)
    for _ in range(2):  # a refused token leaves the state alone
        with pytest.raises(ValueError, match="max_len is 16"):
            net.decode(x[:, 16:17], states)
    assert states[1][0].lengths.tolist() == [16, 16]


def test_a_state_made_without_a_count(dev):
    """A state of a user's own: its lengths alone say how many tokens there are."""
    from triton_tagi_amd.layers import AttentionState

    net = network(max_len=300)
    x = batch(2, 280, 8)[0].to(dev)
    mu, _ = net.forward(x)
    _, _, states = net.prompt(x[:, :270])
    s = states[1][0]
    own = [None, [AttentionState(s.cache, s.table, s.lengths), None], states[2], None]
    pm, _, _ = net.prompt(x[:, 270:274], states=own)
    near(pm, mu[:, 270:274], "prompt")
    for t in range(270, 273):
        near(net.decode(x[:, t:t + 1], own)[0][:, 0], mu[:, t], f"token {t}")


def test_recorded_prompts(dev):
    """A prompt that continues a state, recorded with a token after it: every replay starts from the
    state as it then is, and the states it leaves hold what the last replay wrote."""
    net = network(max_len=64)
    x = batch(2, 40, 8)[0].to(dev)
    mu, _ = net.forward(x)
    _, _, states = net.prompt(x[:, :5])
    part, tok = x[:, 5:9].clone(), x[:, 9:10].clone()
    net.decode(tok, net.prompt(part, states=states)[2])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pm, _, more = net.prompt(part, states=states)
        m, _ = net.decode(tok, more)
    for _ in range(3):
        graph.replay()
        near(pm, mu[:, 5:9], "prompt"), near(m[:, 0], mu[:, 9], "token")
        assert more[1][0].lengths.tolist() == [10, 10] and states[1][0].lengths.tolist() == [5, 5]
        # eager tokens on what the replay left, until the next replay begins anew
        for t in range(10, 13):
            near(net.decode(x[:, t:t + 1], more)[0][:, 0], mu[:, t], f"token {t}")
    # the state that the graph reads goes on by itself
    for t in range(5, 7):
        net.decode(x[:, t:t + 1], states)
    part.copy_(x[:, 7:11]), tok.copy_(x[:, 11:12])
    graph.replay()
    near(pm, mu[:, 7:11], "prompt of a later state"), near(m[:, 0], mu[:, 11], "token of a later state")


def test_recorded_first_prompts(dev):
    """A first prompt of a padded batch and a token after it, recorded: every replay begins anew."""
    net = network(max_len=32, page_size=4)
    x = batch(3, 20, 9)[0].to(dev)
    mu, _ = net.forward(x)
    part, tok, n = x[:, :8].clone(), x[:, 8:9].clone(), torch.tensor([8, 8, 8], device=dev)
    _, _, warm = net.prompt(part, lengths=n)
    net.decode(tok, warm)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pm, _, states = net.prompt(part, lengths=n)
        m, _ = net.decode(tok, states)
    for cut in (8, 3, 6):
        n.fill_(cut)
        tok.copy_(x[:, cut:cut + 1])
        for _ in range(2):
            graph.replay()
            near(pm[:, :cut], mu[:, :cut], f"prompt of {cut}"), near(m[:, 0], mu[:, cut], f"token after {cut}")
            assert states[1][0].lengths.tolist() == [cut + 1] * 3
            net.forward(x)
        near(net.decode(x[:, cut + 1:cut + 2], states)[0][:, 0], mu[:, cut + 1], "eager token")
        near(net.prompt(x[:, cut + 2:cut + 5], states=states)[0], mu[:, cut + 2:cut + 5], "eager prompt")
