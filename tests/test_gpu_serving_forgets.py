"""What a prompt or a token leaves behind for a backward: nothing. The layers that act on each
token by themselves replace what they keep as well, so their backward is refused too, before it
stores a delta or updates a parameter, until a forward of its own."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

V, E = 11, 8


def network(mixer=False, remax=False):
    from triton_tagi_amd import (Embedding, LayerNorm, Linear, LinearAttention, ReLU, Remax, ResidualRMSNorm, RMSNorm,
                                 Sequential)

    torch.manual_seed(3)
    kw = dict(device="cpu")
    block = [LinearAttention(E, 2, **kw)] if mixer else [Linear(E, E, **kw), Remax() if remax else ReLU()]
    return Sequential([Embedding(V, E, sorted_deltas=True, **kw), ResidualRMSNorm(block, E, **kw), Linear(E, E, **kw),
                       ReLU(), RMSNorm(E, **kw), LayerNorm(E, **kw), Linear(E, V, **kw)], device="cuda:0")


def parameters(layers):
    for layer in layers:
        yield from (t for n in ("mw", "Sw", "mb", "Sb") if isinstance(t := getattr(layer, n, None), torch.Tensor))
        yield from parameters(layer.sublayers())


@pytest.mark.parametrize("mixer", [False, True])
@pytest.mark.parametrize("serve", ["prompt", "decode", "refused prompt"])
def test_backward_after_serving_is_refused_before_it_changes_anything(dev, serve, mixer):
    from triton_tagi_amd.update.in_backward import update_in_backward

    net, other = network(mixer), network(mixer)
    T = 1 if serve == "decode" else 6  # as many tokens as the backward's deltas: shapes give nothing away
    x = torch.randint(0, V, (2, T), generator=torch.Generator().manual_seed(1)).to(dev)
    delta = torch.full((2, T, V), 0.1, device=dev)
    states = net.prompt(x)[2]
    net.forward(x)
    if serve == "prompt":
        net.prompt(x.flip(0))
    elif serve == "decode":
        net.decode(x.flip(0), states)
    elif mixer:  # fails inside the network, after the first layers have run
        with pytest.raises(ValueError, match="lengths"):
            net.prompt(x.flip(0), lengths=torch.ones(3, dtype=torch.int64, device=dev))
    else:
        with pytest.raises(ValueError, match="states"):
            net.prompt(x.flip(0), states=[None, [None], None, None, None, None, None])
    before = [t.clone() for t in parameters(net.layers)]
    with update_in_backward(2.0), pytest.raises(RuntimeError, match="backward without a forward"):
        net.backward(delta, -delta)
    assert all(torch.equal(a, b) for a, b in zip(before, parameters(net.layers)))
    assert all(getattr(layer, "delta_mw", None) is None for layer in net.layers)
    for n in (net, other):  # a forward of its own puts it right
        n.forward(x)
        n.backward(delta, -delta)
        n.update(2.0)
    for a, b in zip(parameters(net.layers), parameters(other.layers)):
        assert torch.equal(a, b)


def test_every_layer_of_a_served_network_says_so(dev):
    net = network(remax=True)  # Remax takes rows in training, sequences when serving
    x = torch.zeros(2, 3, device=dev)
    net.prompt(x)
    d = torch.zeros(2, 3, E, device=dev)
    blocks = [*net.layers, *net.layers[1].layers]
    for layer in blocks:
        out = torch.zeros(2, 3, V, device=dev) if layer is net.layers[-1] else d
        with pytest.raises(RuntimeError, match=f"{type(layer).__name__}: backward without a forward"):
            layer.backward(out, out)
    for layer in (net.layers[0], net.layers[2]):  # as first layer of a step
        with pytest.raises(RuntimeError, match="without a forward"):
            layer.backward_param_deltas(d, d)


def test_training_steps_beside_serving(dev):
    """step, prompt, step: the steps are those of a network that never served."""
    a, b = network(True), network(True)
    x = torch.randint(0, V, (3, 5), generator=torch.Generator().manual_seed(2)).to(dev)
    y = torch.nn.functional.one_hot(x, V).float()
    for _ in range(2):
        a.step(x, y, 1.0)
        _, _, states = a.prompt(x)
        a.decode(x[:, :1], states)
        b.step(x, y, 1.0)
        for p, q in zip(parameters(a.layers), parameters(b.layers)):
            assert torch.equal(p, q)
