"""Attention over so many keys (or rows) and heads that it takes several launches.

The workspace holds the sums of 8192 blocks of 128 rows (or keys); chunks of 1024 keys (2048 rows) beyond
them are another launch's, whose sums are added to those before. Outputs and deltas stay within
the bounds of short walks (remax_reference), and are the same bits in every run.
"""

from __future__ import annotations

import math

import pytest
import torch

from remax_reference import attention, within
from test_gpu_remax_attention import NAMES, run

pytestmark = pytest.mark.gpu


def inputs(B, T, N, H, G, D, dev):
    r = torch.Generator(device=dev).manual_seed(B + T + N + D)
    x = []
    for n, heads in ((T, H), (N, G), (N, G)):
        x += [torch.randn(B, n, heads, D, generator=r, device=dev),
              0.005 + 0.1 * torch.rand(B, n, heads, D, generator=r, device=dev)]
    d = [0.1 * torch.randn(B, T, H, D, generator=r, device=dev),
         -1e-4 - 0.02 * torch.rand(B, T, H, D, generator=r, device=dev)]
    return x, d


# B, T, N, H, G, D, causal
CASES = [
    (4100, 40, 1100, 2, 2, 16, True),    # 8200 blocks: one chunk a launch, two of keys
    (1500, 40, 3200, 4, 2, 24, True),    # 3000 blocks: two chunks a launch, four of keys
    (128, 2200, 2200, 4, 2, 16, True),   # three chunks of keys, three of 4400 rows
    (180, 1500, 1500, 6, 2, 80, False),
    (220, 1200, 1200, 8, 2, 128, True),
    (300, 1300, 1300, 3, 3, 33, False),
    (200, 40, 4100, 4, 2, 33, True),     # one launch of five chunks
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c[:6]) + ("c" if c[6] else "f"))
def test_several_launches(case, dev):
    B, T, N, H, G, D, causal = case
    x, d = inputs(B, T, N, H, G, D, dev)
    lengths = torch.full((B,), N, device=dev)
    lengths[-1] = N // 2 + 1
    starts = torch.full((B,), N - T, device=dev)
    starts[-1] = max(0, N // 2 + 1 - T)
    kw = dict(scale=1 / math.sqrt(D), causal=causal, lengths=lengths, starts=starts)
    got = run(x, d, **kw)
    again = run(x, d, **kw)
    for a, b, n in zip(got, again, NAMES):
        assert torch.equal(a, b), n
    for b in (0, B - 1):
        one = [t[b:b + 1] for t in x]
        ref = attention(*one, kw["scale"], causal, [int(lengths[b])], [int(starts[b])], deltas=[t[b:b + 1] for t in d])
        for g, r, n in zip(got, ref, NAMES):
            within(g[b:b + 1], r, f"{n} of {b}")
