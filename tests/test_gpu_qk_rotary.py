"""RMSNorm of query and key heads with their rotation, against float64.

Bounds, U = 2^-24: a head's sum of squares adds 16 positive terms a lane and joins 32 lanes at most
(21 roundings), its root halves that, the weights and products add 8: 20 U of the normed value. A
turn adds the angle's rounding (pi U), its sine and cosine (4 U) and three roundings, squared twice
that: 32 U of |a| + |b| for means, 48 U of A + B for variances. A weight's delta is a sum of rows:
rows of a thread, the block's groups and 32: (rows / 64 + 256 / lanes + 64) U of the sum of magnitudes
at the sizes here.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24


def d64(t):
    return t.detach().to("cpu", torch.float64)


def units(D, pairs, interleaved):
    i = torch.arange(pairs)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)


def turn(x, c, s, at, transposed=False):
    a, b = x[..., at[0]], x[..., at[1]]
    s = -s if transposed else s
    y = x.clone()
    y[..., at[0]], y[..., at[1]] = a * c - b * s, a * s + b * c
    return y


def turn_var(X, c, s, at):
    a, b = X[..., at[0]], X[..., at[1]]
    Y = X.clone()
    Y[..., at[0]], Y[..., at[1]] = a * c * c + b * s * s, a * s * s + b * c * c
    return Y


def spread(x, at):  # |a| + |b| at both features of a pair
    x = x.abs()
    y = x.clone()
    y[..., at[0]] = y[..., at[1]] = x[..., at[0]] + x[..., at[1]]
    return y


def angles(positions, freq, sections):
    pos = d64(positions)
    pos = pos[..., None] if pos.dim() == 2 else pos
    axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)], dtype=torch.long)
    t = (pos[..., axis] * d64(freq))[:, :, None]
    return t.cos(), t.sin()


def reference(m, S, mw, Sw, c, s, at, eps, deltas=None):
    """[(value, bound)]: mean, variance; with deltas also dm, dS and, with weights, dmw, dSw."""
    m, S = d64(m), d64(S)
    one = torch.ones(m.shape[-1], dtype=torch.float64)
    if mw is None:
        inv, g, Sg = 1.0, one, 0 * one
    else:
        inv, g, Sg = 1 / ((m * m + S).mean(-1, keepdim=True) + eps).sqrt(), d64(mw), d64(Sw)
    n, N = m * inv * g, inv**2 * (S * (g * g + Sg) + Sg * m * m)
    out = [(turn(n, c, s, at), 32 * U * spread(n, at)), (turn_var(N, c, s, at), 48 * U * spread(N, at))]
    if deltas:
        dm, dS = (d64(t) for t in deltas)
        back, Back = turn(dm, c, s, at, True), turn_var(dS, c, s, at)
        w = inv * g
        out += [(back * w, 48 * U * spread(dm, at) * w.abs()), (Back * w * w, 64 * U * spread(dS, at) * w * w)]
        if mw is not None:
            rows, lanes = m[..., 0].numel(), max(1, m.shape[-1] // 8)
            r = (rows / 64 + 256 / lanes + 64) * U
            x, X = m * inv, (m * inv) ** 2
            out += [(Sg * (back * x).sum((0, 1, 2)), r * Sg * (spread(dm, at) * x.abs()).sum((0, 1, 2))),
                    (Sg**2 * (Back * X).sum((0, 1, 2)), r * Sg**2 * (spread(dS, at) * X).sum((0, 1, 2)))]
    return out


def close(got, ref, what):
    got, (value, bound) = d64(got), ref
    assert got.shape == value.shape, what
    assert torch.isfinite(got).all(), what
    over = (got - value).abs() - bound - 1e-30
    assert not got.numel() or over.max() <= 0, f"{what}: over by {over.max().item():.3g}"


# B, T, H, G, D, axes, pairs, interleaved, weights
CASES = [
    (1, 1, 1, 1, 2, 1, 1, False, True),
    (2, 3, 2, 1, 8, 1, 4, False, True),
    (1, 5, 3, 3, 7, 1, 3, True, True),
    (2, 17, 4, 2, 80, 3, 33, True, True),
    (2, 17, 4, 2, 80, 3, 33, False, True),
    (1, 200, 6, 2, 64, 2, 32, False, True),
    (3, 40, 8, 8, 128, 1, 64, False, True),
    (3, 40, 8, 1, 128, 4, 64, True, False),
    (1, 9, 5, 2, 256, 1, 100, False, True),
    (2, 31, 2, 2, 32, 1, 8, False, False),
    (1, 3000, 1, 1, 1, 0, 0, False, True),
    (2, 33, 30, 10, 48, 0, 0, False, True),
    (1, 2, 300, 40, 16, 2, 8, True, True),
]


def case_inputs(case, dev, seed=0, far=1000):
    B, T, H, G, D, axes, pairs, interleaved, weights = case
    r = torch.Generator().manual_seed(seed)
    q = [2 * torch.randn(B, T, H, D, generator=r), 0.1 * torch.rand(B, T, H, D, generator=r)]
    k = [2 * torch.randn(B, T, G, D, generator=r), 0.1 * torch.rand(B, T, G, D, generator=r)]
    d = [torch.randn(B, T, n, D, generator=r) for n in (H, H, G, G)]
    w = [1 + 0.1 * torch.randn(D, generator=r), 0.02 * torch.rand(D, generator=r), 1 + 0.1 * torch.randn(D, generator=r),
         0.02 * torch.rand(D, generator=r)] if weights else None
    kw = {}
    if axes:
        shape = (B, T) if axes == 1 else (B, T, axes)
        pos = torch.randint(-far, far, shape, generator=r)
        freq = 10000.0 ** (-torch.arange(pairs, dtype=torch.float64) / pairs)
        cut = sorted(torch.randint(0, pairs + 1, (axes - 1,), generator=r).tolist())
        sec = tuple(b - a for a, b in zip([0, *cut], [*cut, pairs]))
        kw = dict(positions=pos.to(dev), frequencies=freq.to(dev), sections=sec, interleaved=interleaved)
    to = lambda ts: [t.to(dev) for t in ts]  # noqa: E731
    return to(q), to(k), to(d), (None if w is None else tuple(to(w))), kw


def check(case, dev, **more):
    from triton_tagi_amd import kernels as K

    q, k, d, w, kw = case_inputs(case, dev, **more)
    D, pairs = case[4], case[6]
    at = units(D, pairs, case[7])
    if kw:
        c, s = angles(kw["positions"], kw["frequencies"], kw["sections"])
    else:
        c = s = torch.zeros(1, 1, 1, 0, dtype=torch.float64)
    *out, inv = K.qk_norm_rotary(*q, *k, weights=w, eps=1e-5, **kw)
    back = K.qk_norm_rotary_backward(*d, q[0], k[0], inv, weights=w, **kw)
    rq = reference(*q, *(w[:2] if w else (None, None)), c, s, at, 1e-5, d[:2])
    rk = reference(*k, *(w[2:] if w else (None, None)), c, s, at, 1e-5, d[2:])
    ref = [*rq[:2], *rk[:2], *rq[2:4], *rk[2:4], *rq[4:], *rk[4:]]
    got = [*out, *back]
    assert len(got) == len(ref)
    for i, (g, r) in enumerate(zip(got, ref)):
        close(g, r, f"output {i}")


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(int(x)) for x in c))
def test_against_float64(case, dev):
    check(case, dev)


def test_far_positions(dev):
    """Angles of positions beyond 2^24 are as exact as near ones: 2^-53 of 10^9 radians is 1e-7, so
    the bound's pi U holds up to about there."""
    check((2, 6, 2, 1, 32, 1, 16, False, True), dev, far=1 << 28)


def test_no_tokens(dev):
    from triton_tagi_amd import kernels as K

    for shape in ((0, 3), (2, 0)):
        q, k = torch.zeros(*shape, 2, 8, device=dev), torch.zeros(*shape, 1, 8, device=dev)
        w = tuple(torch.ones(8, device=dev) for _ in range(4))
        out = K.qk_norm_rotary(q, q, k, k, weights=w)
        assert out[0].shape == q.shape and out[4].shape == (*shape, 3)
        back = K.qk_norm_rotary_backward(q, q, k, k, q, k, out[4], weights=w)
        assert len(back) == 8 and not any(t.any() for t in back[4:])


def test_strides_and_positions_of_either_type(dev):
    from triton_tagi_amd import kernels as K

    case = (2, 19, 3, 2, 40, 1, 20, False, True)
    q, k, d, w, kw = case_inputs(case, dev)
    ref = K.qk_norm_rotary(*q, *k, weights=w, **kw)
    buf = [torch.full((2, 19, 5 * 40 + 1), float("nan"), device=dev) for _ in range(2)]
    views = []
    for b, x, y in zip(buf, q[:1] + q[1:], k[:1] + k[1:]):
        b[..., 1:].unflatten(-1, (5, 40))[:, :, :3].copy_(x)
        b[..., 1:].unflatten(-1, (5, 40))[:, :, 3:].copy_(y)
        v = b[..., 1:].unflatten(-1, (5, 40))
        views.append((v[:, :, :3], v[:, :, 3:]))
    kw["positions"] = kw["positions"].int()
    got = K.qk_norm_rotary(views[0][0], views[1][0], views[0][1], views[1][1], weights=w, **kw)
    for a, b in zip(got, ref):
        assert torch.equal(a, b)
    back = K.qk_norm_rotary_backward(*d, q[0], k[0], ref[4], weights=w, **kw)
    dt = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in d]
    for a, b in zip(K.qk_norm_rotary_backward(*dt, views[0][0], views[0][1], ref[4], weights=w, **kw), back):
        assert torch.equal(a, b)


def test_captured_and_replayed(dev):
    from triton_tagi_amd import kernels as K

    q, k, d, w, kw = case_inputs((2, 300, 4, 2, 64, 1, 32, False, True), dev)

    def call():
        *out, inv = K.qk_norm_rotary(*q, *k, weights=w, **kw)
        return (*out, *K.qk_norm_rotary_backward(*d, q[0], k[0], inv, weights=w, **kw))

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for _ in range(3):
        kw["positions"].add_(7)
        q[0].mul_(1.1)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, call()):
            assert torch.equal(a, b)
