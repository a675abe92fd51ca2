"""A causal network of the sequence layers, as it is trained and served: scaled Embedding ->
ResidualRMSNorm around LinearAttention -> ResidualRMSNorm around an MLP -> Linear.

The step is compared with a float64 composition of the oracle's primitives at the engine's
bar (1e-4 of the value or of the tensor's root mean square, whichever is larger); paths that
run the same kernels are compared bit for bit.
"""

from __future__ import annotations

import math

import pytest
import torch

from oracle import tagi_oracle as O
from test_gpu_sequence_ops import lin_backward_reference, lin_reference

pytestmark = pytest.mark.gpu

V, E, H = 37, 48, 3


def d64(t):
    return t.detach().to("cpu", torch.float64)


def near(got, ref, what):
    got, ref = d64(got), d64(ref)
    assert got.shape == ref.shape, what
    bound = 1e-4 * torch.maximum(ref.abs(), ref.square().mean().sqrt()) + 1e-9
    over = (got - ref).abs() - bound
    assert (over <= 0).all(), f"{what}: over by {over.max().item():.3g}"


def layers(vocab=V, sorted_deltas=None, device="cpu"):
    from triton_tagi_amd import Embedding, Linear, LinearAttention, ReLU, ResidualRMSNorm

    kw = dict(device=device)
    return [
        Embedding(vocab, E, scale=0.25, output_scale=math.sqrt(E), padding_idx=0, sorted_deltas=sorted_deltas, **kw),
        ResidualRMSNorm([LinearAttention(E, H, bias=True, gain_weight=0.5, **kw)], E, **kw),
        ResidualRMSNorm([Linear(E, 2 * E, gain_w=0.5, **kw), ReLU(), Linear(2 * E, E, gain_w=0.5, **kw)], E, **kw),
        Linear(E, vocab, **kw),
    ]


def network(seed=0, **kw):
    from triton_tagi_amd import Sequential

    torch.manual_seed(seed)
    return Sequential(layers(**kw), device="cuda:0")


def batch(B, T, seed, vocab=V):
    r = torch.Generator().manual_seed(seed)
    x = torch.randint(0, vocab, (B, T), generator=r)
    y = torch.nn.functional.one_hot(torch.randint(0, vocab, (B, T), generator=r), vocab).float()
    return x, y


def parameters(net):
    """Every parameter tensor of the network, and each one's float64 copy at the call."""
    out = {}
    for i, layer in enumerate(net.layers):
        for j, part in enumerate(getattr(layer, "_learnable", [layer])):
            for n in ("mw", "Sw", "mb", "Sb"):
                t = getattr(part, n, None)
                if isinstance(t, torch.Tensor):
                    out[i, j, n] = t
    return out


def reference_step(net, x, y, sigma_v):
    """One step from the network's present parameters in float64: predictions, new parameters."""
    p = {k: d64(t).clone() for k, t in parameters(net).items()}
    B, T = x.shape
    rows, D = B * T, E // H
    lin = lambda i, j: (p[i, j, "mw"], p[i, j, "Sw"], p[i, j, "mb"].reshape(1, -1), p[i, j, "Sb"].reshape(1, -1))  # noqa: E731
    new = {}

    def update(key, dm, dS):
        i, j, n = key
        m, S = p[i, j, "m" + n], p[i, j, "S" + n]
        new[i, j, "m" + n], new[i, j, "S" + n] = O.capped_update(m, S, dm.reshape(m.shape), dS.reshape(S.shape),
                                                                 O.get_cap_factor(B))

    def linear_back(i, j, a, dz, dS):
        mw, Sw, _, Sb = lin(i, j)
        gm, gb, gS, gSb = O.linear_param_grads(a, dz, dS)
        update((i, j, "w"), Sw * gm, Sw * Sw * gS)
        update((i, j, "b"), Sb * gb, Sb * Sb * gSb)
        return O.linear_backward_delta(dz, dS, mw)

    def norm(i, j, m, S):
        inv = ((m * m + S).mean(1, keepdim=True) + 1e-6).rsqrt()
        g, Sg = p[i, j, "mw"], p[i, j, "Sw"]
        return m * inv * g, inv * inv * (S * (g * g + Sg) + Sg * m * m), inv

    def norm_back(i, j, m, inv, dz, dS):
        g, Sg = p[i, j, "mw"], p[i, j, "Sw"]
        update((i, j, "w"), Sg * (dz * m * inv).sum(0), Sg * Sg * (dS * (m * inv) ** 2).sum(0))
        return dz * inv * g, dS * (inv * g) ** 2

    c, ids = math.sqrt(E), x.reshape(-1)
    real = (ids != 0)[:, None]
    m0, S0 = torch.where(real, c * p[0, 0, "mw"][ids], 0.0), torch.where(real, c * c * p[0, 0, "Sw"][ids], 0.0)
    # attention block: parts 0, 1, 2 are the projections, 3 the norm
    qkv = [O.linear_moments(m0, S0, *lin(1, j)) for j in range(3)]
    heads = [t.reshape(B, T, H, D) for mS in qkv for t in mS]
    dec = d64(torch.tensor(net.layers[1].layers[0].decay))
    mo, So, _, _ = lin_reference(*heads, dec, 1 / math.sqrt(D))
    s1, V1 = mo.reshape(rows, E) + m0, So.reshape(rows, E) + S0
    m1, S1, inv1 = norm(1, 3, s1, V1)
    # MLP block
    hm, hS = O.linear_moments(m1, S1, *lin(2, 0))
    am, aS, J = O.relu_moments(hm, hS)
    bm, bS = O.linear_moments(am, aS, *lin(2, 1))
    s2, V2 = bm + m1, bS + S1
    m2, S2, inv2 = norm(2, 2, s2, V2)
    mz, Sz = O.linear_moments(m2, S2, *lin(3, 0))
    dz, dS = O.innovation(d64(y).reshape(rows, -1), mz, Sz, sigma_v)
    dz, dS = linear_back(3, 0, m2, dz, dS)
    dz, dS = norm_back(2, 2, s2, inv2, dz, dS)
    bz, bS = linear_back(2, 1, am, dz, dS)
    bz, bS = linear_back(2, 0, m1, bz * J, bS * J * J)
    dz, dS = norm_back(1, 3, s1, inv1, dz + bz, dS + bS)
    dq = lin_backward_reference(heads[0], heads[2], heads[4], dz.reshape(B, T, H, D), dS.reshape(B, T, H, D), dec,
                                1 / math.sqrt(D))
    for j in range(3):
        a, b = linear_back(1, j, m0, dq[2 * j].reshape(rows, E), dq[2 * j + 1].reshape(rows, E))
        dz, dS = dz + a, dS + b
    Sw = p[0, 0, "Sw"]
    keep = ids != 0
    update((0, 0, "w"), c * Sw * torch.zeros_like(Sw).index_add_(0, ids[keep], dz[keep]),
           (c * Sw) ** 2 * torch.zeros_like(Sw).index_add_(0, ids[keep], dS[keep]))
    return mz.reshape(B, T, -1), Sz.reshape(B, T, -1), new


@pytest.mark.parametrize("B,T,ids", [(4, 19, torch.float32), (1, 1, torch.int64), (3, 130, torch.int32)])
def test_step_against_the_oracle(dev, B, T, ids):
    net = network()
    x, y = batch(B, T, 3 * T + B)
    mz, Sz, new = reference_step(net, x, y, 2.0)
    got = net.step(x.to(dev, ids), y.to(dev), 2.0)
    near(got[0], mz, "mu")
    near(got[1], Sz, "var")
    have = parameters(net)
    assert set(have) == set(new)
    for k, t in new.items():
        near(have[k], t, str(k))


def test_update_in_backward_and_afterwards_are_the_same_step(dev):
    """step() applies updates inside the backward pass; backward() then update() gives the
    same bits, and the deltas stay on the layers in both."""
    from triton_tagi_amd import compute_innovation, get_cap_factor

    a, b = network(), network()
    x, y = batch(4, 33, 1)
    x, y = x.float().to(dev), y.to(dev)
    for _ in range(2):
        a.step(x, y, 2.0)
        mu, var = b.forward(x)
        b.backward(*compute_innovation(y, mu, var, 2.0))
        b.update(get_cap_factor(4))
        for k, t in parameters(a).items():
            assert torch.equal(t, parameters(b)[k]), k
        assert torch.equal(a.layers[0].delta_mw, b.layers[0].delta_mw)


def test_sorted_deltas_match_the_scan(dev):
    """An Embedding without a scale: the sorted form's step against the scanning form's."""
    from triton_tagi_amd import Embedding, Linear, Sequential

    nets = []
    for form in (False, True):
        torch.manual_seed(2)
        nets.append(Sequential([Embedding(V, E, scale=0.25, padding_idx=3, sorted_deltas=form, device="cpu"),
                                Linear(E, V, device="cpu")], device="cuda:0"))
    x, y = batch(8, 40, 6)
    for net in nets:
        net.step(x.float().to(dev), y.to(dev), 2.0)
    near(nets[1].layers[0].delta_mw, nets[0].layers[0].delta_mw, "delta_mw")
    near(nets[1].layers[0].mw, nets[0].layers[0].mw, "mw")
    near(nets[1].layers[0].Sw, nets[0].layers[0].Sw, "Sw")


@pytest.mark.parametrize("split", [1, 8, 20])
def test_prompt_and_decode_follow_forward(dev, split):
    """A prompt, then token by token: the moments of the whole sequences (the state passes
    between kernels that sum in different orders)."""
    net = network()
    x, _ = batch(5, 21, 9)
    x = x.to(dev)
    mu, var = net.forward(x.float())
    pm, pS, states = net.prompt(x[:, :split].float())
    near(pm, mu[:, :split], "prompt")
    for t in range(split, 21):
        m, S = net.decode(x[:, t:t + 1], states)
        near(m[:, 0], mu[:, t], f"token {t}")
        near(S[:, 0], var[:, t], f"token {t}")


def test_ragged_prompt_and_inactive_sequences(dev):
    """A padded batch gives each sequence its own answers, and a sequence that is off keeps its
    state while the others go on."""
    net = network()
    x, _ = batch(4, 12, 4)
    x = x.to(dev)
    n = torch.tensor([12, 5, 1, 0], device=dev, dtype=torch.int32)
    pm, pS, states = net.prompt(x, lengths=n)
    for b in range(4):
        k = int(n[b])
        if k:
            m, S, own = net.prompt(x[b:b + 1, :k])
            near(pm[b:b + 1, :k], m, "means")
            near(pS[b:b + 1, :k], S, "variances")
            for i in range(2):
                near(states[1][0][i][b:b + 1], own[1][0][i], "state")
        else:
            assert (states[1][0][0][b] == 0).all() and (states[1][0][1][b] == 0).all()
    before = [t.clone() for t in states[1][0]]
    on = torch.tensor([True, False, True, False], device=dev)
    m, S = net.decode(x[:, :1], states, active=on)
    for i in range(2):
        assert torch.equal(states[1][0][i][~on], before[i][~on])
        assert not torch.equal(states[1][0][i][on], before[i][on])
    full, _, _ = net.prompt(torch.cat([x[:1], x[:1, :1]], 1))
    near(m[:1], full[:, 12:], "next token")


def test_lengths_in_training(dev):
    """forward(lengths=) and backward of the layer: padded tokens give and take nothing."""
    from triton_tagi_amd import LinearAttention

    torch.manual_seed(1)
    layer = LinearAttention(E, H, device="cuda:0")
    r = torch.Generator().manual_seed(2)
    m, S = torch.randn(2, 9, E, generator=r).to(dev), torch.rand(2, 9, E, generator=r).to(dev)
    dm, dS = torch.randn(2, 9, E, generator=r).to(dev), -torch.rand(2, 9, E, generator=r).to(dev)
    mo, So = layer.forward(m, S, lengths=torch.tensor([9, 4], device=dev))
    assert (mo[1, 4:] == 0).all() and (So[1, 4:] == 0).all()
    dma, dSa = layer.backward(dm, dS)
    assert (dma[1, 4:] == 0).all() and (dSa[1, 4:] == 0).all()
    d_all = [p.delta_mw.clone() for p in layer._projections()]
    one, two = layer.forward(m[:1], S[:1]), None
    a0 = layer.backward(dm[:1], dS[:1])
    d0 = [p.delta_mw.clone() for p in layer._projections()]
    two = layer.forward(m[1:, :4], S[1:, :4])
    a1 = layer.backward(dm[1:, :4], dS[1:, :4])
    d1 = [p.delta_mw.clone() for p in layer._projections()]
    near(mo[:1], one[0], "mo"), near(mo[1:, :4], two[0], "mo")
    near(dma[:1], a0[0], "dma"), near(dma[1:, :4], a1[0], "dma")
    for x, y, z in zip(d_all, d0, d1):
        near(x, y + z, "delta_mw")


def test_step_graph_replays_match_eager_steps(dev):
    a, b = network(), network()
    x, y = batch(6, 65, 5)
    x, y = x.float().to(dev), y.to(dev)
    a.forward(x)  # an eager pass of the same layers lives while the graph is recorded
    graph = b.capture_step(x, y, 2.0)  # runs one eager step
    a.step(x, y, 2.0)
    torch.cuda.synchronize()
    for r in range(4):
        gm, gS = graph.replay()
        em, eS = a.step(x, y, 2.0)
        torch.cuda.synchronize()
        assert torch.equal(gm, em) and torch.equal(gS, eS), r
        for k, t in parameters(a).items():
            assert torch.equal(t, parameters(b)[k]), (r, k)
        torch.randn(1000, device=dev).sum().item()


def test_decode_graph_replays_match_eager_tokens(dev):
    net = network()
    x, _ = batch(3, 30, 8)
    x = x.to(dev)
    _, _, states = net.prompt(x[:, :10])
    _, _, eager = net.prompt(x[:, :10])
    tok = x[:, 10:11].clone()
    net.decode(tok, net.prompt(x[:, :10])[2])  # first-call work is not recorded
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m, S = net.decode(tok, states)
    for t in range(10, 16):
        tok.copy_(x[:, t:t + 1])
        graph.replay()
        em, eS = net.decode(x[:, t:t + 1], eager)
        torch.cuda.synchronize()
        assert torch.equal(m, em) and torch.equal(S, eS), t
        for i in range(2):
            assert torch.equal(states[1][0][i], eager[1][0][i]), t


def test_two_graphs_do_not_share_workspaces(dev):
    """Split prompts and sorted deltas recorded twice, replayed in turn and beside eager calls."""
    from triton_tagi_amd.kernels import embedding_param_deltas, linear_attention

    r = torch.Generator().manual_seed(1)
    graphs, outs, want, keep = [], [], [], []  # a graph reads its inputs where they were: they stay alive
    for s in range(2):
        x = [t.to(dev) for t in (torch.randn(1, 900, 2, 32, generator=r) for _ in range(3))]
        S = [t.to(dev) for t in (torch.rand(1, 900, 2, 32, generator=r) for _ in range(3))]
        dec = torch.tensor([0.99, 0.9], device=dev)
        ids = torch.randint(0, 50, (3000,), generator=r).to(dev)
        dm, Sw = torch.randn(3000, 64, generator=r).to(dev), torch.rand(50, 64, generator=r).to(dev)

        def both(x=x, S=S, dec=dec, ids=ids, dm=dm, Sw=Sw):
            return (*linear_attention(x[0], S[0], x[1], S[1], x[2], S[2], dec), *embedding_param_deltas(ids, dm, dm, Sw))

        keep.append(both)
        want.append([t.clone() for t in both()])
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(both())
    for k in (0, 1, 0, 0, 1):
        graphs[k].replay()
        graphs[1 - k].replay()
        torch.cuda.synchronize()
        for j in range(2):
            for a, b in zip(outs[j], want[j]):
                assert torch.equal(a, b)


def test_another_stream(dev):
    net = network()
    x, _ = batch(2, 16, 3)
    x = x.to(dev)
    want = net.forward(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = net.forward(x)
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_checkpoint_round_trip(dev, tmp_path):
    from triton_tagi_amd import RunDir

    a, b = network(0), network(1)
    x, y = batch(4, 9, 2)
    a.step(x.float().to(dev), y.to(dev), 2.0)
    run = RunDir("d", "a", "o", base=str(tmp_path))
    run.save_checkpoint(a, 3, {})
    assert run.load_checkpoint(b) == 3
    for k, t in parameters(a).items():
        assert torch.equal(t, parameters(b)[k]), k
    assert torch.equal(a.forward(x.float().to(dev))[0], b.forward(x.float().to(dev))[0])


@pytest.mark.parametrize("serve", ["prompt", "decode"])
def test_backward_after_serving_needs_a_forward(dev, serve):
    """A prompt or token between forward and backward replaces what the layers keep: refused,
    and a forward of its own puts the backward right again."""
    net, other = network(), network()
    x, _ = batch(2, 6, 3)
    x = x.to(dev).float()
    delta = torch.ones(2, 6, V, device=dev)
    _, _, states = net.prompt(x)
    net.forward(x)
    net.prompt(x.flip(1)) if serve == "prompt" else net.decode(x[:, :1], states)
    # by the head's Linear where the token counts differ, else by the first layer that mixes tokens
    with pytest.raises((RuntimeError, ValueError), match="without a forward|weight deltas"):
        net.backward(delta, -delta)
    other.forward(x), net.forward(x)
    other.backward(delta, -delta), net.backward(delta, -delta)
    for a, b in zip(net.layers, other.layers):
        for (_, _, m, S), (_, _, om, oS) in zip(a._update_items(), b._update_items()):
            assert torch.equal(m, om) and torch.equal(S, oS)


def test_prompts_without_tokens(dev):
    """No sequence or no token is refused; sequences whose lengths are all zero leave zero states."""
    net = network()
    x = batch(3, 5, 1)[0].to(dev)
    for empty in (x[:0], x[:, :0]):
        with pytest.raises(ValueError, match="at least one"):
            net.prompt(empty)
    _, _, states = net.prompt(x, lengths=torch.zeros(3, dtype=torch.int64, device=dev))
    M, P = states[1][0]
    assert M.shape == (3, H, E // H, E // H) and not M.any() and not P.any()
    m, S = net.decode(x[:, :1], states)
    want, wS, _ = net.prompt(x[:, :1])
    near(m, want, "first token"), near(S, wS, "its variances")


def test_layers_refuse(dev):
    from triton_tagi_amd import (Embedding, Linear, LinearAttention, MultiheadAttentionV2, PositionalEncoding, ReLU,
                                 ResidualRMSNorm, Sequential)

    with pytest.raises(ValueError):
        Embedding(4, 4, output_scale=2.0, sorted_deltas=False)
    with pytest.raises(ValueError):
        Embedding(4, 4, output_scale=math.nan)
    for bad in ((48, 5, None), (512, 2, None), (48, 3, [0.5, 0.5]), (48, 3, 1.5), (48, 3, -0.1)):
        with pytest.raises(ValueError):
            LinearAttention(*bad)
    layer = LinearAttention(E, H)
    with pytest.raises(RuntimeError, match="without a forward"):
        layer.backward(torch.zeros(1, 2, E, device=dev), torch.zeros(1, 2, E, device=dev))
    with pytest.raises(ValueError):
        layer.forward(torch.zeros(2, E, device=dev), torch.zeros(2, E, device=dev))
    with pytest.raises(ValueError):
        layer.forward(torch.zeros(2, 3, E + 1, device=dev), torch.zeros(2, 3, E + 1, device=dev))
    with pytest.raises(ValueError):
        layer.step(torch.zeros(2, 3, E, device=dev), torch.zeros(2, 3, E, device=dev), layer.new_state(2))
    with pytest.raises(ValueError, match="maps"):
        ResidualRMSNorm([Linear(E, 2 * E)], E).forward(torch.zeros(2, E, device=dev), torch.zeros(2, E, device=dev))
    x = torch.zeros(2, 1, device=dev)
    for other in (PositionalEncoding(E), MultiheadAttentionV2(E, H, 16)):
        net = Sequential([Embedding(V, E), ResidualRMSNorm([other], E)])
        with pytest.raises(TypeError, match="carried state"):
            net.prompt(x)
    net = Sequential([Linear(4, 4), ReLU()])
    with pytest.raises(ValueError, match="one token"):
        net.decode(torch.zeros(2, 3, 4, device=dev), [None, None])
    with pytest.raises(ValueError, match="states"):
        net.decode(torch.zeros(2, 1, 4, device=dev), [None])
