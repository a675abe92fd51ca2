"""Attention over sequences and over a cache at the sizes where another form of a kernel takes over,
and rows of few keys, whose weights hang on differences (bounds: remax_reference)."""

from __future__ import annotations

import math

import pytest
import torch

from remax_reference import attention, within
from test_gpu_kv_cache import BF16, F32, FP8, cache_of, rows_of, values
from test_gpu_remax_attention import check, inputs

pytestmark = pytest.mark.gpu


# heads on both sides of 32, 64 and 96 features, whole groups of eight and not
@pytest.mark.parametrize("D", [31, 32, 34, 40, 63, 64, 65, 72, 89, 95, 96, 97, 104, 127])
def test_head_dimensions(D, dev):
    x, d = inputs(2, 37, 90, 4, 2, D, 20 + D, dev)
    check(x, d, 1.0 / math.sqrt(D), True, [90, 61], [53, 10])


# a row of one block more or less: 16 rows a wave, 4 or 8 waves, tiles of 32 keys, splits of 256 keys
@pytest.mark.parametrize("T,N,R,D", [(127, 127, 1, 32), (128, 129, 1, 64), (43, 257, 3, 96), (65, 513, 1, 128),
                                     (1, 2049, 2, 64), (9, 1030, 1, 96)])
def test_edges_of_blocks_and_splits(T, N, R, D, dev):
    x, d = inputs(1, T, N, 2 * R, 2, D, T + N, dev)
    check(x, d, 1.0 / math.sqrt(D), True, None, [N - T])


@pytest.mark.parametrize("D", [24, 32, 64, 80, 96, 128])
def test_one_key(D, dev):
    """A row that sees one key: the weight is 1 and has no variance, so mo = v and So = Sv. The key's
    moments and the row's sums are the same numbers: p = mm / mt is 1 to 2 roundings (a reciprocal and a
    product), and the relative variance k = (vm u^2 + 0) / d^2 with u = 1 - p <= 2^-22 is at most
    x 2^-44 with x = vm / mm^2, below 1e4 for these scores (m / sd > -3.5: checked): 1e-9, of which
    mv^2 <= 25 makes 3e-8 of So, under 1e-5 of Sv >= 5e-3. The rest are roundings of w s^-1 (2 and a
    reciprocal's 1), its square, and the matrix cores' sums of six products, cut off at 2^-23 each."""
    from triton_tagi_amd import kernels as K

    x, _ = inputs(300, 1, 1, 4, 2, D, 5 + D, dev)
    scale = 1.0 / math.sqrt(D)
    mq, Sq, mk, Sk = (t.double() for t in x[:4])
    k, S = mk.repeat_interleave(2, 2), Sk.repeat_interleave(2, 2)
    z, v = scale * (mq * k).sum(-1), scale**2 * (Sq * (k * k + S) + mq * mq * S).sum(-1)
    keep = (z / v.sqrt() > -3.5)[..., None]  # further down the floors of 1e-6 have a say
    mo, So = K.remax_attention(*x, scale=scale)
    mv, Sv = (t.double().repeat_interleave(2, 2) for t in x[4:])
    assert keep.float().mean() > 0.5  # of the inputs: most rows count
    b = 16 * 2.0**-23
    assert (((mo - mv).abs() - b * mv.abs()) * keep).max() <= 0
    assert (((So - Sv).abs() - 2 * b * Sv - 1e-9 * mv * mv) * keep).max() <= 0
    # the same row as one query over a cache
    cache = K.new_kv_cache(300, 2, 1, D, F32, dev)
    table = torch.arange(300, device=dev, dtype=torch.int32)[:, None]
    K.cache_write(cache, *x[2:], table)
    m1, S1 = K.remax_attention_step(x[0][:, 0], x[1][:, 0], cache, table, torch.ones(300, device=dev, dtype=torch.int32),
                                    scale=scale)
    assert (((m1[:, None] - mv).abs() - b * mv.abs()) * keep).max() <= 0
    assert (((S1[:, None] - Sv).abs() - 2 * b * Sv - 1e-9 * mv * mv) * keep).max() <= 0


# heads on a key head: 1 to 4 share a product's columns, more take them one by one
@pytest.mark.parametrize("dtype", [F32, BF16, FP8])
@pytest.mark.parametrize("R,D", [(1, 30), (2, 64), (3, 96), (4, 128), (5, 128), (16, 64), (17, 32), (4, 61), (7, 125)])
def test_step_heads(dtype, R, D, dev):
    from triton_tagi_amd import kernels as K

    B, G, page, longest = 2, 2, 24, 150
    cache = cache_of(dev, 16, G, page, D, dtype)
    table = torch.randperm(16, generator=torch.Generator().manual_seed(R))[:14].view(B, 7).int().to(dev)
    K.cache_write(cache, *rows_of(B, longest, G, D, R + D, dev), table)
    ln = torch.tensor([longest, 67], device=dev)
    r = torch.Generator().manual_seed(D)
    mq, Sq = torch.randn(B, R * G, D, generator=r).to(dev), (0.05 * torch.rand(B, R * G, D, generator=r)).to(dev)
    mo, So = K.remax_attention_step(mq, Sq, cache, table, ln, scale=1 / math.sqrt(D))
    pools = values(cache)
    at = torch.arange(longest)
    for b in range(B):
        n = int(ln[b])
        pg = table[b].cpu().long()[at[:n] // page]
        keys = [p[pg, :, at[:n] % page] for p in pools]  # (n, G, D)
        ref = attention(mq[b, None, None], Sq[b, None, None], *(k[None] for k in keys), 1 / math.sqrt(D), causal=False,
                        starts=[n - 1])
        within(mo[b, None, None], ref[0], f"mo {b}"), within(So[b, None, None], ref[1], f"So {b}")


@pytest.mark.parametrize("dtype", [F32, BF16, FP8])
@pytest.mark.parametrize("R,D", [(4, 128), (3, 96), (4, 64), (1, 32), (2, 40)])
def test_step_in_one_launch_and_in_three(dtype, R, D, dev):
    """The same lengths under a bound that one block holds and under one that it does not."""
    from triton_tagi_amd import kernels as K

    B, G, page, longest = 3, 2, 32, 256
    cache = cache_of(dev, 30, G, page, D, dtype)
    table = torch.randperm(30, generator=torch.Generator().manual_seed(R))[:27].view(B, 9).int().to(dev)
    K.cache_write(cache, *rows_of(B, longest, G, D, 7 * R + D, dev), table)
    ln = torch.tensor([longest, 0, 201], device=dev)
    r = torch.Generator().manual_seed(D)
    mq, Sq = torch.randn(B, R * G, D, generator=r).to(dev), (0.05 * torch.rand(B, R * G, D, generator=r)).to(dev)
    pools = values(cache)
    at = torch.arange(longest)
    for most in (256, 257):
        mo, So = K.remax_attention_step(mq, Sq, cache, table, ln, scale=1 / math.sqrt(D), max_len=most)
        assert not mo[1].any() and not So[1].any()
        for b in (0, 2):
            n = int(ln[b])
            pg = table[b].cpu().long()[at[:n] // page]
            keys = [p[pg, :, at[:n] % page][None] for p in pools]
            ref = attention(mq[b, None, None], Sq[b, None, None], *keys, 1 / math.sqrt(D), causal=False, starts=[n - 1])
            within(mo[b, None, None], ref[0], f"mo {b} {most}"), within(So[b, None, None], ref[1], f"So {b} {most}")


@pytest.mark.parametrize("dtype", [F32, BF16, FP8])
def test_step_of_many_long_sequences(dtype, dev):
    """Enough sequences for the longest stretch of keys to a wave; all read the same few pages."""
    from triton_tagi_amd import kernels as K

    B, G, R, D, page, longest = 64, 8, 2, 32, 64, 4095
    cache = cache_of(dev, 9, G, page, D, dtype)
    fill = torch.arange(9, device=dev, dtype=torch.int32)[None]
    K.cache_write(cache, *rows_of(1, 9 * page, G, D, 3, dev), fill)
    r = torch.Generator().manual_seed(8)
    table = torch.randint(0, 9, (B, 64), generator=r).int().to(dev)
    lengths = torch.randint(0, longest, (B,), generator=r)
    lengths[:4] = torch.tensor([longest, 0, 2048, 2049])
    mq, Sq = torch.randn(B, G * R, D, generator=r).to(dev), (0.05 * torch.rand(B, G * R, D, generator=r)).to(dev)
    mo, So = K.remax_attention_step(mq, Sq, cache, table, lengths.to(dev), scale=1 / math.sqrt(D))
    assert not mo[1].any() and not So[1].any()
    pools = values(cache)
    for b in (0, 2, 3, 63):
        n = int(lengths[b])
        at = torch.arange(n)
        pg = table[b].cpu().long()[at // page]
        for g in (0, 5):
            keys = [p[pg, g, at % page][None, :, None] for p in pools]
            h = slice(g * R, g * R + R)
            ref = attention(mq[b, None, None, h], Sq[b, None, None, h], *keys, 1 / math.sqrt(D), causal=False,
                            starts=[n - 1])
            within(mo[b, None, None, h], ref[0], f"mo {b} {g}"), within(So[b, None, None, h], ref[1], f"So {b} {g}")


def test_tokens_behind_every_page(dev):
    """Positions that 32 bits do not hold are behind every table: nothing is written."""
    from triton_tagi_amd import kernels as K

    cache = cache_of(dev, 3, 1, 4, 8, FP8)
    before = [t.clone() for t in cache]
    table = torch.arange(3, device=dev, dtype=torch.int32)[None]
    for start in (12, 2**31 - 1, 2**31, 2**40, -(2**40), -3):
        K.cache_write(cache, *rows_of(1, 3, 1, 8, 1, dev), table, torch.tensor([start], device=dev))
    for a, b in zip(cache, before):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("D,pairs", [(80, 33), (8, 1), (128, 63), (24, 10)])
def test_neighbouring_pairs_in_whole_rows(D, pairs, dev):
    """Pairs of neighbours turn the same way whether four of them end inside a lane or not."""
    from triton_tagi_amd import kernels as K

    r = torch.Generator().manual_seed(D)
    x = [torch.randn(2, 5, h, D, generator=r).to(dev) for h in (3, 1)]
    S = [(0.1 * torch.rand(2, 5, h, D, generator=r)).to(dev) for h in (3, 1)]
    pos = torch.randint(0, 5000, (2, 5), generator=r).to(dev)
    freq = K.rotary_frequencies(pairs, device=dev)
    oq, oqS, ok, okS, _ = K.qk_norm_rotary(x[0], S[0], x[1], S[1], pos, freq, interleaved=True)
    t = (pos.double()[..., None, None] * freq).remainder(2 * math.pi)
    for m, v, om, ov in ((x[0], S[0], oq, oqS), (x[1], S[1], ok, okS)):
        a, b, A, B = (y[..., i:2 * pairs:2].double() for y in (m, v) for i in (0, 1))
        c, s = t.cos(), t.sin()
        # a turn to 2^-22, two products and a sum: under 8 roundings of |a| + |b|
        e = 2.0**-21
        assert ((om[..., 0:2 * pairs:2] - (a * c - b * s)).abs() <= e * (a.abs() + b.abs())).all()
        assert ((om[..., 1:2 * pairs:2] - (a * s + b * c)).abs() <= e * (a.abs() + b.abs())).all()
        assert ((ov[..., 0:2 * pairs:2] - (A * c * c + B * s * s)).abs() <= 2 * e * (A + B)).all()
        assert ((ov[..., 1:2 * pairs:2] - (A * s * s + B * c * c)).abs() <= 2 * e * (A + B)).all()
        assert torch.equal(om[..., 2 * pairs:], m[..., 2 * pairs:]) and torch.equal(ov[..., 2 * pairs:], v[..., 2 * pairs:])
