"""A causal network around RemaxAttention, as it is trained and served: scaled Embedding ->
ResidualRMSNorm around the attention and its output projection -> ResidualRMSNorm around an MLP ->
Linear. The step is compared with float64 compositions of the oracle's primitives at the engine's bar
(1e-4 of the value or of the tensor's root mean square); paths that run the same kernels bit for bit.
"""

from __future__ import annotations

import math

import pytest
import torch

from oracle import tagi_oracle as O
from remax_reference import attention
from test_gpu_qk_rotary import angles, turn, turn_var, units
from test_gpu_sequence_layers import d64, near, parameters

pytestmark = pytest.mark.gpu

V, E, H, G = 37, 48, 6, 2
D = E // H


def network(seed=0, vocab=V, **kw):
    from triton_tagi_amd import Embedding, Linear, ReLU, RemaxAttention, ResidualRMSNorm, Sequential

    torch.manual_seed(seed)
    cpu = dict(device="cpu")
    kw = dict(dict(max_len=40, page_size=8, bias=True, gain_weight=0.5), **kw)
    return Sequential([
        Embedding(vocab, E, scale=0.25, output_scale=math.sqrt(E), padding_idx=0, **cpu),
        ResidualRMSNorm([RemaxAttention(E, H, G, **kw, **cpu), Linear(E, E, gain_w=0.5, **cpu)], E, **cpu),
        ResidualRMSNorm([Linear(E, 2 * E, gain_w=0.5, **cpu), ReLU(), Linear(2 * E, E, gain_w=0.5, **cpu)], E, **cpu),
        Linear(E, vocab, **cpu),
    ], device="cuda:0")


def batch(B, T, seed):
    r = torch.Generator().manual_seed(seed)
    x = torch.randint(0, V, (B, T), generator=r)
    return x, torch.nn.functional.one_hot(torch.randint(0, V, (B, T), generator=r), V).float()


def reference_step(net, x, y, sigma_v):
    p = {k: d64(t).clone() for k, t in parameters(net).items()}
    B, T = x.shape
    rows = B * T
    lin = lambda i, j: (p[i, j, "mw"], p[i, j, "Sw"], p[i, j, "mb"].reshape(1, -1), p[i, j, "Sb"].reshape(1, -1))  # noqa: E731
    new = {}

    def update(i, j, n, dm, dS):
        m, S = p[i, j, "m" + n], p[i, j, "S" + n]
        new[i, j, "m" + n], new[i, j, "S" + n] = O.capped_update(m, S, dm.reshape(m.shape), dS.reshape(S.shape),
                                                                 O.get_cap_factor(B))

    def linear_back(i, j, a, dz, dS):
        mw, Sw, _, Sb = lin(i, j)
        gm, gb, gS, gSb = O.linear_param_grads(a, dz, dS)
        update(i, j, "w", Sw * gm, Sw * Sw * gS)
        update(i, j, "b", Sb * gb, Sb * Sb * gSb)
        return O.linear_backward_delta(dz, dS, mw)

    def norm(i, j, m, S):
        inv = ((m * m + S).mean(-1, keepdim=True) + 1e-6).rsqrt()
        g, Sg = p[i, j, "mw"], p[i, j, "Sw"]
        return m * inv * g, inv * inv * (S * (g * g + Sg) + Sg * m * m), inv

    def norm_back(i, j, m, inv, dz, dS):
        g, Sg = p[i, j, "mw"], p[i, j, "Sw"]
        lead = tuple(range(dz.dim() - 1))
        update(i, j, "w", Sg * (dz * m * inv).sum(lead), Sg * Sg * (dS * (m * inv) ** 2).sum(lead))
        return dz * inv * g, dS * (inv * g) ** 2

    c, ids = math.sqrt(E), x.reshape(-1)
    real = (ids != 0)[:, None]
    m0, S0 = torch.where(real, c * p[0, 0, "mw"][ids], 0.0), torch.where(real, c * c * p[0, 0, "Sw"][ids], 0.0)
    # attention block: projections 0, 1, 2, norms of queries and keys 3, 4, the Linear 5, the norm 6
    raw = [t.reshape(B, T, n, D) for j, n in ((0, H), (1, G), (2, G)) for t in O.linear_moments(m0, S0, *lin(1, j))]
    cos, sin = angles(torch.arange(T).expand(B, T), 10000.0 ** (-torch.arange(D // 2).double() / (D // 2)), (D // 2,))
    at = units(D, D // 2, False)
    ops, inv = [], []
    for j in range(2):
        m, S, i = norm(1, 3 + j, raw[2 * j], raw[2 * j + 1])
        ops += [turn(m, cos, sin, at), turn_var(S, cos, sin, at)]
        inv.append(i)
    ops += raw[4:]
    (mo, _), (So, _) = attention(*ops, 1 / math.sqrt(D))
    am, aS = mo.reshape(rows, E), So.reshape(rows, E)
    om, oS = O.linear_moments(am, aS, *lin(1, 5))
    s1, V1 = om + m0, oS + S0
    m1, S1, inv1 = norm(1, 6, s1, V1)
    hm, hS = O.linear_moments(m1, S1, *lin(2, 0))
    rm, rS, J = O.relu_moments(hm, hS)
    bm, bS = O.linear_moments(rm, rS, *lin(2, 1))
    s2, V2 = bm + m1, bS + S1
    m2, S2, inv2 = norm(2, 2, s2, V2)
    mz, Sz = O.linear_moments(m2, S2, *lin(3, 0))
    dz, dS = O.innovation(d64(y).reshape(rows, -1), mz, Sz, sigma_v)
    dz, dS = linear_back(3, 0, m2, dz, dS)
    dz, dS = norm_back(2, 2, s2, inv2, dz, dS)
    bz, bS = linear_back(2, 1, rm, dz, dS)
    bz, bS = linear_back(2, 0, m1, bz * J, bS * J * J)
    dz, dS = norm_back(1, 6, s1, inv1, dz + bz, dS + bS)
    az, aS_ = linear_back(1, 5, am, dz, dS)
    d = [t for t, _ in attention(*ops, 1 / math.sqrt(D), deltas=(az.reshape(B, T, H, D), aS_.reshape(B, T, H, D)))[2:]]
    for j in range(2):
        back, var = turn(d[2 * j], cos, sin, at, True), turn_var(d[2 * j + 1], cos, sin, at)
        d[2 * j], d[2 * j + 1] = norm_back(1, 3 + j, raw[2 * j], inv[j], back, var)
    for j, n in enumerate((H, G, G)):
        a, b = linear_back(1, j, m0, d[2 * j].reshape(rows, n * D), d[2 * j + 1].reshape(rows, n * D))
        dz, dS = dz + a, dS + b
    Sw = p[0, 0, "Sw"]
    keep = ids != 0
    update(0, 0, "w", c * Sw * torch.zeros_like(Sw).index_add_(0, ids[keep], dz[keep]),
           (c * Sw) ** 2 * torch.zeros_like(Sw).index_add_(0, ids[keep], dS[keep]))
    return mz.reshape(B, T, -1), Sz.reshape(B, T, -1), new


@pytest.mark.parametrize("B,T", [(4, 19), (1, 1), (3, 130)])
def test_step_against_the_oracle(dev, B, T):
    net = network()
    x, y = batch(B, T, 3 * T + B)
    mz, Sz, new = reference_step(net, x, y, 2.0)
    got = net.step(x.to(dev), y.to(dev), 2.0)
    near(got[0], mz, "mu"), near(got[1], Sz, "var")
    have = parameters(net)
    assert set(have) == set(new)
    for k, t in new.items():
        near(have[k], t, str(k))


@pytest.mark.parametrize("split", [1, 8, 20])
def test_prompt_and_decode_follow_forward(dev, split):
    net = network()
    x = batch(5, 21, 9)[0].to(dev)
    mu, var = net.forward(x)
    pm, pS, states = net.prompt(x[:, :split])
    near(pm, mu[:, :split], "prompt"), near(pS, var[:, :split], "prompt")
    for t in range(split, 21):
        m, S = net.decode(x[:, t:t + 1], states)
        near(m[:, 0], mu[:, t], f"token {t}"), near(S[:, 0], var[:, t], f"token {t}")


def test_a_prompt_goes_on_from_a_state_and_leaves_it(dev):
    net = network()
    x = batch(3, 30, 2)[0].to(dev)
    mu, var = net.forward(x)
    _, _, states = net.prompt(x[:, :11])
    kept = states[1][0].clone()
    for _ in range(2):  # the same state twice
        pm, pS, more = net.prompt(x[:, 11:24], states=states)
        near(pm, mu[:, 11:24], "second prompt"), near(pS, var[:, 11:24], "second prompt")
    for a, b in zip((*states[1][0].cache[:4], states[1][0].lengths), (*kept.cache[:4], kept.lengths)):
        assert torch.equal(a, b)
    assert states[1][0].used == 11 and more[1][0].used == 24
    m, _ = net.decode(x[:, 24:25], more)
    near(m[:, 0], mu[:, 24], "token")
    m, _ = net.decode(x[:, 11:12], states)
    near(m[:, 0], mu[:, 11], "token after the first prompt")


def test_ragged_prompts_and_inactive_sequences(dev):
    net = network()
    x = batch(4, 12, 4)[0].to(dev)
    n = torch.tensor([12, 5, 1, 0], device=dev, dtype=torch.int32)
    pm, pS, states = net.prompt(x, lengths=n)
    state = states[1][0]
    assert state.lengths.tolist() == [12, 5, 1, 0]
    for b in range(3):
        k = int(n[b])
        m, S, _ = net.prompt(x[b:b + 1, :k])
        near(pm[b:b + 1, :k], m, "means"), near(pS[b:b + 1, :k], S, "variances")
    on = torch.tensor([True, False, True, False], device=dev)
    before = state.clone()
    m, S = net.decode(x[:, :1], states, active=on)
    assert state.lengths.tolist() == [13, 5, 2, 0]
    for a, b in zip(state.cache[:4], before.cache[:4]):
        width = state.table.shape[1]
        for i in (1, 3):
            assert torch.equal(a[i * width:(i + 1) * width], b[i * width:(i + 1) * width])
    full = net.prompt(torch.cat([x[:1], x[:1, :1]], 1))[0]
    near(m[:1], full[:, 12:], "next token")
    # the ragged batch goes on with a ragged prompt
    m, S, more = net.prompt(x[:, :6], lengths=torch.tensor([6, 2, 0, 3], device=dev), states=states)
    assert more[1][0].lengths.tolist() == [19, 7, 2, 3]
    want = net.prompt(torch.cat([x[1:2, :5], x[1:2, :2]], 1))[0]
    near(m[1:2, :2], want[:, 5:], "continued")
    near(m[3:4, :3], net.prompt(x[3:4, :3])[0], "begun")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_rounded_caches_hold_the_rounded_tokens(dev, dtype):
    """A token on a rounded cache is the attention over that cache's values, bit for bit the kernels'."""
    from triton_tagi_amd import RemaxAttention
    from triton_tagi_amd import kernels as K

    torch.manual_seed(3)
    layer = RemaxAttention(64, 4, 2, max_len=30, page_size=4, cache_dtype=dtype, device="cuda:0")
    r = torch.Generator().manual_seed(4)
    m, S = torch.randn(2, 12, 64, generator=r).to(dev), 0.1 * torch.rand(2, 12, 64, generator=r).to(dev)
    _, _, state = layer.prompt(m[:, :11], S[:, :11])
    assert state.cache.km.dtype is dtype
    keys = K.cache_read(state.cache, state.table, state.lengths, 11)
    _, ops = layer._project(m[:, :11], S[:, :11], layer._positions(m[:, :11], None, None))
    for a, b in zip(keys, ops[2:]):
        if dtype is torch.bfloat16:
            assert torch.equal(a, b.to(dtype).float())
        else:  # half a step of e4m3, or of the smallest step under a row's largest value
            top = b.abs().amax(-1, keepdim=True)
            assert ((a - b).abs() <= torch.maximum(2.0**-4 * b.abs(), top * 2.0**-17)).all()
    out = layer.step(m[:, 11], S[:, 11], state)
    _, one = layer._project(m[:, 11:], S[:, 11:], torch.full((2, 1), 11, device=dev))
    want = K.remax_attention_step(one[0][:, 0], one[1][:, 0], state.cache, state.table, state.lengths, layer._scale,
                                  max_len=1024)
    assert torch.equal(out[0], want[0].view(2, 64)) and torch.equal(out[1], want[1].view(2, 64))


def test_lengths_in_training(dev):
    from triton_tagi_amd import RemaxAttention

    torch.manual_seed(1)
    layer = RemaxAttention(E, H, G, device="cuda:0")
    r = torch.Generator().manual_seed(2)
    m, S = torch.randn(2, 9, E, generator=r).to(dev), torch.rand(2, 9, E, generator=r).to(dev)
    dm, dS = torch.randn(2, 9, E, generator=r).to(dev), -torch.rand(2, 9, E, generator=r).to(dev)
    mo, So = layer.forward(m, S, lengths=torch.tensor([9, 4], device=dev))
    assert not mo[1, 4:].any() and not So[1, 4:].any()
    dma, dSa = layer.backward(dm, dS)
    assert not dma[1, 4:].any() and not dSa[1, 4:].any()
    every = [p.delta_mw.clone() for p in layer.sublayers()]
    one = layer.forward(m[:1], S[:1])
    a0 = layer.backward(dm[:1], dS[:1])
    d0 = [p.delta_mw.clone() for p in layer.sublayers()]
    two = layer.forward(m[1:, :4], S[1:, :4])
    a1 = layer.backward(dm[1:, :4], dS[1:, :4])
    d1 = [p.delta_mw.clone() for p in layer.sublayers()]
    near(mo[:1], one[0], "mo"), near(mo[1:, :4], two[0], "mo")
    near(dma[:1], a0[0], "dma"), near(dma[1:, :4], a1[0], "dma")
    for x, y, z in zip(every, d0, d1):
        near(x, y + z, "delta_mw")


def test_positions_of_several_axes(dev):
    """The same position on every axis is one axis; shifting every position turns queries and keys alike."""
    from triton_tagi_amd import RemaxAttention

    layers = []
    for sections in (None, (1, 2, 1)):
        torch.manual_seed(5)
        layers.append(RemaxAttention(32, 4, 2, rotary_sections=sections, device="cuda:0"))
    r = torch.Generator().manual_seed(6)
    m, S = torch.randn(2, 9, 32, generator=r).to(dev), torch.rand(2, 9, 32, generator=r).to(dev)
    one = layers[0].forward(m, S)
    t = torch.arange(9, device=dev).expand(2, 9)
    axes = layers[1].forward(m, S, positions=t[..., None].expand(2, 9, 3))
    assert torch.equal(one[0], axes[0]) and torch.equal(one[1], axes[1])
    assert torch.equal(layers[0].forward(m, S, positions=t)[0], one[0])
    with pytest.raises(ValueError, match="positions"):
        layers[1].forward(m, S)


@pytest.mark.parametrize("kw", [dict(qk_norm=False), dict(rotary=False), dict(qk_norm=False, rotary=False, bias=False)])
def test_without_norms_or_positions(dev, kw):
    net = network(**kw)
    x, y = batch(2, 14, 7)
    mu, _ = net.forward(x.to(dev))
    pm, _, states = net.prompt(x[:, :13].to(dev))
    near(pm, mu[:, :13], "prompt")
    near(net.decode(x[:, 13:].to(dev), states)[0][:, 0], mu[:, 13], "token")
    before = {k: t.clone() for k, t in parameters(net).items()}
    net.step(x.to(dev), y.to(dev), 2.0)
    assert any(not torch.equal(t, before[k]) for k, t in parameters(net).items() if k[0] == 1)
    assert all(torch.isfinite(t).all() for t in parameters(net).values())


def test_step_graph_replays_match_eager_steps(dev):
    a, b = network(), network()
    x, y = batch(6, 65, 5)
    x, y = x.float().to(dev), y.to(dev)
    a.forward(x)
    graph = b.capture_step(x, y, 2.0)
    a.step(x, y, 2.0)
    torch.cuda.synchronize()
    for r in range(3):
        gm, gS = graph.replay()
        em, eS = a.step(x, y, 2.0)
        torch.cuda.synchronize()
        assert torch.equal(gm, em) and torch.equal(gS, eS), r
        for k, t in parameters(a).items():
            assert torch.equal(t, parameters(b)[k]), (r, k)


def test_decode_graph_replays_match_eager_tokens(dev):
    """The recorded token keeps the cache's whole room; eager ones a bound: the sums split differently."""
    net = network()
    x = batch(3, 30, 8)[0].to(dev)
    _, _, states = net.prompt(x[:, :10])
    _, _, eager = net.prompt(x[:, :10])
    tok = x[:, 10:11].clone()
    net.decode(tok, net.prompt(x[:, :10])[2])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m, S = net.decode(tok, states)
    for t in range(10, 16):
        tok.copy_(x[:, t:t + 1])
        graph.replay()
        em, eS = net.decode(x[:, t:t + 1], eager)
        torch.cuda.synchronize()
        near(m, em, f"token {t}"), near(S, eS, f"token {t}")
        assert torch.equal(states[1][0].lengths, eager[1][0].lengths)


def test_update_in_backward_and_afterwards_are_the_same_step(dev):
    from triton_tagi_amd import compute_innovation, get_cap_factor

    a, b = network(), network()
    x, y = batch(4, 33, 1)
    x, y = x.to(dev), y.to(dev)
    for _ in range(2):
        a.step(x, y, 2.0)
        mu, var = b.forward(x)
        b.backward(*compute_innovation(y, mu, var, 2.0))
        b.update(get_cap_factor(4))
        for k, t in parameters(a).items():
            assert torch.equal(t, parameters(b)[k]), k


def test_checkpoints_round_trip(dev, tmp_path):
    from triton_tagi_amd import RemaxAttention, RunDir, Sequential

    a, b = network(0), network(1)
    x, y = batch(4, 9, 2)
    a.step(x.to(dev), y.to(dev), 2.0)
    run = RunDir("d", "a", "o", base=str(tmp_path))
    run.save_checkpoint(a, 3, {})
    assert run.load_checkpoint(b) == 3
    for k, t in parameters(a).items():
        assert torch.equal(t, parameters(b)[k]), k
    assert torch.equal(a.forward(x.to(dev))[0], b.forward(x.to(dev))[0])
    nets = [Sequential([RemaxAttention(E, H, G, device="cpu")], device="cuda:0") for _ in range(2)]  # on its own
    run.save_checkpoint(nets[0], 4, {})
    run.load_checkpoint(nets[1])
    for p, q in zip(nets[0].layers[0].sublayers(), nets[1].layers[0].sublayers()):
        assert torch.equal(p.mw, q.mw) and torch.equal(p.Sw, q.Sw)


def test_backward_after_serving_needs_a_forward(dev):
    net = network()
    x = batch(2, 6, 3)[0].to(dev)
    delta = torch.ones(2, 6, V, device=dev)
    net.forward(x)
    net.prompt(x.flip(1))
    with pytest.raises(RuntimeError, match="without a forward"):
        net.layers[1].layers[0].backward(delta[..., :E], delta[..., :E])
    net.forward(x)
    net.backward(delta, -delta)


def test_the_room_of_a_sequence(dev):
    net = network(max_len=9, page_size=4)
    x = batch(2, 12, 3)[0].to(dev)
    with pytest.raises(ValueError, match="max_len is 9"):
        net.prompt(x[:, :10])
    _, _, states = net.prompt(x[:, :8])
    with pytest.raises(ValueError, match="max_len"):
        net.prompt(x[:, :2], states=states)
    net.decode(x[:, 8:9], states)
    with pytest.raises(ValueError, match="max_len"):
        net.decode(x[:, 9:10], states)
    assert states[1][0].lengths.tolist() == [9, 9]


def test_refusals(dev):
    from triton_tagi_amd import RemaxAttention

    for bad in (dict(embed_dim=48, num_heads=5), dict(embed_dim=48, num_heads=6, num_kv_heads=4),
                dict(embed_dim=512, num_heads=2), dict(embed_dim=9, num_heads=3), dict(embed_dim=48, num_heads=6, max_len=0),
                dict(embed_dim=48, num_heads=6, rotary_sections=(1, 1)),
                dict(embed_dim=48, num_heads=6, rotary=False, rotary_sections=(4,))):
        with pytest.raises(ValueError):
            RemaxAttention(**bad)
    layer = RemaxAttention(E, H, rotary=False)
    z = torch.zeros(2, 3, E, device=dev)
    with pytest.raises(RuntimeError, match="without a forward"):
        layer.backward(z, z)
    with pytest.raises(ValueError):
        layer.forward(z[0], z[0])
    with pytest.raises(ValueError):
        layer.forward(z[..., 1:], z[..., 1:])
    with pytest.raises(ValueError, match="positions"):
        layer.forward(z, z, positions=torch.zeros(2, 3, dtype=torch.int64, device=dev))
    with pytest.raises(ValueError, match="features"):
        layer.step(z, z, layer.new_state(2))
    with pytest.raises(ValueError, match="state"):
        layer.step(z[:, 0], z[:, 0], layer.new_state(3))
    with pytest.raises(TypeError, match="active"):
        layer.step(z[:, 0], z[:, 0], layer.new_state(2), active=torch.ones(2, device=dev))
