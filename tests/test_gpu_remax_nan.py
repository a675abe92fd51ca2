"""A NaN that a query sees is not lost: outputs of a query with one are NaN, and a key with one reaches
every query that sees it. Sequences and heads that do not see it are finite."""

from __future__ import annotations

import math

import pytest
import torch

from test_gpu_remax_attention import inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [16, 64, 80, 128])
def test_a_nan_is_not_lost(D, dev):
    """In a query's mean or variance, a key's, a value's: the outputs that see it are NaN, and those of
    sequences and heads that do not are finite."""
    from triton_tagi_amd import kernels as K

    B, T, H, G = 2, 40, 4, 2
    x, d = inputs(B, T, T, H, G, D, 13, dev)
    for i in range(6):
        for at in (0, 17):
            y = [t.clone() for t in x]
            y[i][0, at, 1, D // 2] = float("nan")
            mo, So, rows = K.remax_attention(*y, scale=1 / math.sqrt(D), return_rows=True)
            if i < 2:  # query (0, at, 1) alone
                hit = torch.zeros(B, T, H, dtype=torch.bool, device=dev)
                hit[0, at, 1] = True
                assert torch.equal(mo.isnan().all(-1), hit) and torch.equal(So.isnan().all(-1), hit), (i, at)
                assert torch.equal(mo.isnan().any(-1), hit) and torch.equal(So.isnan().any(-1), hit), (i, at)
                dmq = K.remax_attention_backward(*y[:5], *d, rows, scale=1 / math.sqrt(D))[0]
                assert dmq[0, at, 1].isnan().all() and torch.isfinite(dmq[1]).all()
            else:  # key head 1 of sequence 0: its queries from `at` on
                seen = So if i == 5 else mo
                nan = seen.isnan().all(-1) if i < 4 else seen[..., D // 2].isnan()
                assert nan[0, at:, 2:].all(), (i, at)
                assert torch.isfinite(mo[1]).all() and torch.isfinite(So[1]).all() and torch.isfinite(mo[0, :, :2]).all()


@pytest.mark.parametrize("R", [1, 4, 6])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("D,N", [(32, 40), (64, 700), (128, 40)])
def test_a_nan_is_not_lost_in_a_cache(R, dtype, D, N, dev):
    from triton_tagi_amd import kernels as K

    B, G, page = 2, 2, 16
    r = torch.Generator().manual_seed(14)
    width = -(-N // page)
    table = torch.arange(B * width, device=dev, dtype=torch.int32).view(B, width)
    k = [torch.randn(B, N, G, D, generator=r).to(dev) if i % 2 == 0 else torch.rand(B, N, G, D, generator=r).to(dev)
         for i in range(4)]
    q = [torch.randn(B, G * R, D, generator=r).to(dev), torch.rand(B, G * R, D, generator=r).to(dev)]
    lengths = torch.full((B,), N, device=dev)
    for i in range(6):
        kk, qq = [t.clone() for t in k], [t.clone() for t in q]
        if i < 4:
            kk[i][0, N - 3, 1, D // 2] = float("nan")
        else:
            qq[i - 4][0, R, D // 2] = float("nan")
        cache = K.new_kv_cache(B * width, G, page, D, dtype, dev)
        K.cache_write(cache, *kk, table)
        mo, So = K.remax_attention_step(*qq, cache, table, lengths, scale=1 / math.sqrt(D))
        assert torch.isfinite(mo[1]).all() and torch.isfinite(So[1]).all()
        assert torch.isfinite(mo[0, :R]).all() and torch.isfinite(So[0, :R]).all()
        if i < 2:
            assert mo[0, R:].isnan().all() and So[0, R:].isnan().all(), i
        elif i < 4:
            assert (mo if i == 2 else So)[0, R:, D // 2].isnan().all(), i
        else:
            hit = torch.zeros(G * R, dtype=torch.bool, device=dev)
            hit[R] = True
            assert torch.equal(mo[0].isnan().all(-1), hit) and torch.equal(mo[0].isnan().any(-1), hit), i
