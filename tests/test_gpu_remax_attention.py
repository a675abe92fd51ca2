"""Remax attention over sequences, forward and backward, against float64 (bounds: remax_reference)."""

from __future__ import annotations

import math

import pytest
import torch

from remax_reference import attention, within

pytestmark = pytest.mark.gpu

NAMES = ("mo", "So", "dmq", "dSq", "dmk", "dSk", "dmv", "dSv")


def inputs(B, T, N, H, G, D, seed, dev, spread=1.0):
    r = torch.Generator().manual_seed(seed)

    def pair(*shape):
        return spread * torch.randn(*shape, generator=r), 0.005 + 0.1 * torch.rand(*shape, generator=r)

    x = [*pair(B, T, H, D), *pair(B, N, G, D), *pair(B, N, G, D)]
    d = [0.1 * torch.randn(B, T, H, D, generator=r), -1e-4 - 0.02 * torch.rand(B, T, H, D, generator=r)]
    return [t.to(dev) for t in x], [t.to(dev) for t in d]


def run(x, d, **kw):
    from triton_tagi_amd import kernels as K

    mo, So, rows = K.remax_attention(*x, return_rows=True, **kw)
    return (mo, So, *K.remax_attention_backward(*x[:5], *d, rows, **kw))


def check(x, d, scale, causal=True, lengths=None, starts=None):
    dev = x[0].device
    kw = dict(scale=scale, causal=causal,
              lengths=None if lengths is None else torch.tensor(lengths, device=dev),
              starts=None if starts is None else torch.tensor(starts, device=dev, dtype=torch.int32))
    got = run(x, d, **kw)
    ref = attention(*x, scale, causal, lengths, starts, deltas=d)
    for g, r, n in zip(got, ref, NAMES):
        within(g, r, n)
    return got


# B, T, N, H, G, D, causal, lengths, starts
CASES = [
    (1, 1, 1, 1, 1, 1, True, None, None),
    (1, 1, 1, 2, 1, 8, False, None, None),
    (2, 5, 5, 2, 2, 3, True, None, None),
    (2, 16, 16, 2, 1, 16, True, None, None),
    (1, 33, 33, 4, 2, 33, True, None, None),
    (2, 64, 64, 3, 3, 64, False, None, None),
    (2, 65, 65, 6, 2, 80, True, None, None),
    (1, 129, 129, 2, 1, 128, True, None, None),
    (3, 40, 40, 2, 2, 32, True, [0, 40, 17], None),
    (3, 40, 40, 4, 1, 24, False, [1, 0, 39], None),
    (2, 7, 100, 4, 2, 48, True, None, [93, 50]),
    (3, 9, 70, 2, 1, 20, True, [70, 30, 12], [61, 25, 40]),
    (2, 12, 30, 2, 2, 64, True, None, [-5, 25]),
    (2, 12, 30, 2, 2, 64, False, [30, 18], [-5, 10]),
    (1, 2, 1500, 8, 2, 64, True, None, [1498]),
    (2, 70, 600, 3, 1, 128, True, [600, 333], [530, 263]),
    (1, 600, 600, 5, 1, 12, True, None, None),
    (4, 3, 3, 1, 1, 128, True, [-2, 9, 2, 0], None),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c[:6]) + ("c" if c[6] else "f"))
def test_against_float64(case, dev):
    B, T, N, H, G, D, causal, lengths, starts = case
    x, d = inputs(B, T, N, H, G, D, 1, dev)
    check(x, d, 1.0 / math.sqrt(D), causal, lengths, starts)


@pytest.mark.parametrize("spread", [0.05, 3.0])
def test_flat_and_peaked_scores(spread, dev):
    """Scores near 0, where every weight counts, and far ones, where most lie under the floors."""
    x, d = inputs(2, 50, 50, 2, 1, 32, 2, dev, spread)
    check(x, d, 1.0 / math.sqrt(32))


def test_nothing_seen(dev):
    from triton_tagi_amd import kernels as K

    x, d = inputs(2, 6, 4, 2, 1, 16, 3, dev)
    for kw in (dict(lengths=torch.zeros(2, dtype=torch.int64, device=dev)),
               dict(starts=torch.full((2,), 4, device=dev)), dict(starts=torch.full((2,), -(1 << 40), device=dev)),
               dict(starts=torch.full((2,), 1 << 40, device=dev))):
        for t in run(x, d, scale=0.25, **kw):
            assert not t.any()
    x, d = inputs(2, 6, 0, 2, 1, 16, 3, dev)  # no keys
    for t in run(x, d):
        assert not t.any()
    x, d = inputs(2, 0, 5, 2, 1, 16, 3, dev)  # no queries
    got = run(x, d)
    assert got[0].shape == (2, 0, 2, 16) and not any(t.any() for t in got)
    x, d = inputs(0, 3, 5, 2, 1, 16, 3, dev)
    assert K.remax_attention(*x)[0].shape == (0, 3, 2, 16)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -torch.finfo(torch.float32).max])
def test_what_is_masked_may_hold_anything(bad, dev):
    B, T, H, G, D = 3, 37, 4, 2, 40
    lengths = [20, 37, 0]
    x, d = inputs(B, T, T, H, G, D, 4, dev)
    ref = attention(*x, 0.2, True, lengths, None, deltas=d)
    for t in (*x, *d):
        for b, n in enumerate(lengths):
            t[b, n:] = bad
    for causal in (True, False):
        got = run(x, d, scale=0.2, causal=causal, lengths=torch.tensor(lengths, device=dev))
        if causal:
            for g, r, n in zip(got, ref, NAMES):
                within(g, r, n)
        assert all(torch.isfinite(g).all() for g in got)


def test_heads_read_in_place(dev):
    """Queries, keys and values side by side in one buffer, odd offsets; deltas with strides too."""
    B, T, H, G, D = 2, 45, 4, 2, 20
    x, d = inputs(B, T, T, H, G, D, 5, dev)
    ref = run(x, d, scale=0.3)
    wide = (H + 2 * G) * D + 3
    views = []
    for kind in (0, 1):
        buf = torch.full((B, T, wide), float("nan"), device=dev)
        at = 1
        for i, n in ((0, H), (2, G), (4, G)):
            v = buf[..., at:at + n * D].unflatten(-1, (n, D))
            v.copy_(x[i + kind])
            views.append((i + kind, v))
            at += n * D
    y = [v for _, v in sorted(views, key=lambda p: p[0])]
    dt = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in d]
    for a, b, n in zip(run(y, dt, scale=0.3), ref, NAMES):
        assert torch.equal(a, b), n
    # means and variances of different layouts, a last stride that is not 1
    z = [t.transpose(-1, -2).contiguous().transpose(-1, -2) if i % 2 else t for i, t in enumerate(x)]
    for a, b, n in zip(run(z, d, scale=0.3), ref, NAMES):
        assert torch.equal(a, b), n


def test_variances_of_zero(dev):
    """Deterministic queries and keys: variances count as 1e-20, weights follow the means."""
    from triton_tagi_amd import kernels as K

    x, _ = inputs(1, 20, 20, 2, 1, 16, 6, dev)
    x[1].zero_(), x[3].zero_()
    got = K.remax_attention(*x, scale=0.25)
    for g, r, n in zip(got, attention(*x, 0.25), NAMES):
        within(g, r, n)


def test_a_chunk_of_queries_equals_the_whole(dev):
    """The last queries on their own, at their positions, over the same keys."""
    from triton_tagi_amd import kernels as K

    x, _ = inputs(2, 90, 90, 4, 2, 64, 7, dev)
    mo, So = K.remax_attention(*x, scale=0.125)
    m1, S1 = K.remax_attention(*(t[:, 61:] for t in x[:2]), *x[2:], scale=0.125, starts=torch.tensor([61, 61], device=dev))
    ref = attention(*x, 0.125)
    for got, whole, r in ((m1, mo, ref[0]), (S1, So, ref[1])):
        part = (r[0][:, 61:], r[1][:, 61:])
        within(got, part, "chunk")
        within(whole[:, 61:], part, "whole")


def test_runs_repeat_and_streams(dev):
    """The same bits in every run, on another stream, and in two calls at once."""
    x, d = inputs(2, 200, 200, 4, 2, 64, 8, dev)
    ref = run(x, d, scale=0.125)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(run(x, d, scale=0.125))
    torch.cuda.synchronize()
    for g in got:
        for a, b, n in zip(g, ref, NAMES):
            assert torch.equal(a, b), n


def test_captured_and_replayed(dev):
    from triton_tagi_amd import kernels as K

    x, d = inputs(1, 30, 700, 4, 2, 64, 9, dev)
    kw = dict(scale=0.125, starts=torch.tensor([670], device=dev))
    run(x, d, **kw)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs of the same call, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(x, d, **kw)
        graphs.append((graph, out))
    for i in range(3):
        for t in (*x, *d):
            t.mul_(0.9)
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        eager = run(x, d, **kw)
        for _, out in graphs:
            for a, b, n in zip(out, eager, NAMES):
                assert torch.equal(a, b), (i, n)
    assert K is not None


def test_deltas_against_differences(dev):
    """The deltas of the values are the outputs' derivatives: mo is linear in the values' means."""
    from triton_tagi_amd import kernels as K

    x, d = inputs(1, 12, 12, 2, 1, 8, 10, dev)
    _, _, rows = K.remax_attention(*x, scale=0.35, return_rows=True)
    dmv = K.remax_attention_backward(*x[:5], *d, rows, scale=0.35)[4]
    base = K.remax_attention(*x, scale=0.35)[0].double()
    for j in (0, 5, 11):
        y = [t.clone() for t in x]
        y[4][0, j, 0, 3] += 1.0
        diff = ((K.remax_attention(*y, scale=0.35)[0].double() - base) * d[0].double()).sum()
        # the difference of outputs of magnitude 1 rounds 12 x 2 values, each 2^-22 at most
        assert abs(diff.item() - dmv[0, j, 0, 3].item()) < 24 * 2.0**-22


def test_score_deltas_against_differences(dev):
    """e = c J (dm v^T) with J the Remax's Jacobian: the diagonal of da/dz scaled by cov / v. One
    key far above the others makes every other weight's own derivative the whole of it."""
    from triton_tagi_amd import kernels as K

    x, d = inputs(1, 4, 4, 1, 1, 4, 11, dev)
    _, _, rows = K.remax_attention(*x, scale=0.5, return_rows=True)
    dmq, dSq, dmk, dSk = K.remax_attention_backward(*x[:5], *d, rows, scale=0.5)[:4]
    # linear in the deltas, quadratic maps of J in the variances'
    got = K.remax_attention_backward(*x[:5], 2 * d[0], 4 * d[1], rows, scale=0.5)[:4]
    for a, b, f in ((got[0], dmq, 2), (got[1], dSq, 4), (got[2], dmk, 2), (got[3], dSk, 4)):
        assert torch.equal(a, b * f)
