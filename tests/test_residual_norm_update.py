"""Updates of nested residual blocks, counted on the CPU: every parameter tensor once a step.

A layer whose backward applied its update (``update_in_backward``) is left out once; a layer
that shows no parameter groups is updated through its own ``update``. The update functions are
replaced by counters, so no kernel runs.
"""

from __future__ import annotations

import itertools

import pytest
import torch

from triton_tagi_amd import Embedding, Linear, ReLU, ResidualRMSNorm, Sequential
from triton_tagi_amd.base import LearnableLayer

E = 4


class OwnUpdate(LearnableLayer):
    """A layer without groups: the base class's default."""

    def __init__(self):
        self.updates = 0

    def forward(self, ma, Sa):
        return ma, Sa

    def backward(self, delta_ma, delta_Sa):
        return delta_ma, delta_Sa

    def update(self, cap_factor):
        self.updates += 1

    @property
    def num_parameters(self):
        return 0


@pytest.fixture
def counts(monkeypatch):
    """Updates per parameter tensor (by identity), wherever they are applied."""
    seen: dict[int, int] = {}

    def one(m, S, dm, dS, cap):
        for t in (m, S):
            seen[id(t)] = seen.get(id(t), 0) + 1

    def multi(items, cap):
        for it in items:
            one(*it, cap)

    import sys

    for name, module in list(sys.modules.items()):
        if name.startswith("triton_tagi_amd"):
            if hasattr(module, "update_parameters"):
                monkeypatch.setattr(module, "update_parameters", one)
            if hasattr(module, "update_parameters_multi"):
                monkeypatch.setattr(module, "update_parameters_multi", multi)
    return seen


def with_deltas(layer):
    for n in ("mw", "Sw", "mb", "Sb"):
        t = getattr(layer, n, None)
        setattr(layer, "delta_" + n, None if t is None else torch.zeros_like(t))
    return layer


def leaves(layers):
    for layer in layers:
        if isinstance(layer, ResidualRMSNorm):
            yield from leaves(layer.sublayers())
        elif isinstance(layer, (Linear, Embedding)) or hasattr(layer, "ni"):
            yield layer


@pytest.mark.parametrize("flagged", [(), (0,), (1,), (2,), (0, 1, 2)])
@pytest.mark.parametrize("own_at", [None, 0, 1, 2])
@pytest.mark.parametrize("depth", [0, 1, 2])
def test_nested_blocks_update_every_parameter_once(counts, depth, own_at, flagged):
    """Linear layers at three levels of nesting, any of them updated in the backward pass, and a
    layer without groups at any level beside them."""
    def block(level):
        inside = [with_deltas(Linear(E, E, device="cpu")), ReLU()]
        if own_at == level:
            inside.append(OwnUpdate())
        if level < depth:
            inside.insert(1, block(level + 1))
        return ResidualRMSNorm(inside, E, device="cpu")

    net = Sequential([with_deltas(Linear(E, E, device="cpu")), block(0), with_deltas(Linear(E, E, device="cpu"))],
                     device="cpu")
    found = list(leaves(net.layers))
    linears = [layer for layer in found if isinstance(layer, Linear)]
    for layer in found:
        with_deltas(layer)
    for step in range(2):  # a flag counts for one step
        counts.clear()
        skip = [linears[i] for i in flagged if i < len(linears)] if step == 0 else []
        for layer in skip:
            layer._updated_in_backward = True
        net.update(2.0)
        for layer in found:
            for n in ("mw", "Sw", "mb", "Sb"):
                t = getattr(layer, n, None)
                if t is not None:
                    assert counts.get(id(t), 0) == (0 if layer in skip else 1), (step, layer, n)
            assert not layer._updated_in_backward
    if own_at is not None and own_at <= depth:
        own = [x for x in itertools.chain(*_walk(net.layers)) if isinstance(x, OwnUpdate)]
        assert [x.updates for x in own] == [2]


def _walk(layers):
    yield layers
    for layer in layers:
        yield from _walk(list(layer.sublayers()))


def test_asking_for_groups_changes_nothing(counts):
    """``_update_groups`` may be asked any number of times before the update, by a container of
    containers too."""
    inner = ResidualRMSNorm([with_deltas(Linear(E, E, device="cpu"))], E, device="cpu")
    outer = ResidualRMSNorm([inner, OwnUpdate()], E, device="cpu")
    lin = inner.layers[0]
    for n in (inner.norm, outer.norm):
        with_deltas(n)
    lin._updated_in_backward = True
    for _ in range(2):
        inner._update_groups(), outer._update_groups()
        assert lin._updated_in_backward
    outer.update(2.0)
    assert not lin._updated_in_backward and not any(id(t) in counts for t in (lin.mw, lin.Sw, lin.mb, lin.Sb))
    assert counts[id(inner.norm.mw)] == counts[id(outer.norm.mw)] == 1


def test_a_flagged_table_inside_a_block(counts):
    """The sorted Embedding flags itself as Linear does."""
    table = with_deltas(Embedding(5, E, sorted_deltas=True, device="cpu"))
    inner = ResidualRMSNorm([table], E, device="cpu")
    net = Sequential([ResidualRMSNorm([inner, OwnUpdate()], E, device="cpu")], device="cpu")
    for layer in leaves(net.layers):
        with_deltas(layer)
    table._updated_in_backward = True
    net.update(2.0)
    assert id(table.mw) not in counts
    net.update(2.0)
    assert counts[id(table.mw)] == 1
