"""One call over long sequences: some of its queries, and the keys that only they see, against float64.

The reference takes a few queries at their positions over all keys; deltas of keys come from all queries
that see them, so the last keys' are compared, which the last queries alone see.
"""

from __future__ import annotations

import math

import pytest
import torch

from remax_reference import attention, within
from test_gpu_remax_attention import NAMES, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,T,N,H,G,D", [(1, 9001, 9001, 2, 1, 32), (2, 6000, 6000, 4, 2, 64), (1, 4500, 4500, 2, 2, 128),
                                         (1, 3, 70001, 4, 2, 64), (1, 1, 300000, 2, 1, 80), (1, 40, 20011, 8, 1, 21)])
def test_long_sequences(B, T, N, H, G, D, dev):
    r = torch.Generator(device=dev).manual_seed(N + D)
    x = []
    for n, heads in ((T, H), (N, G), (N, G)):
        x += [torch.randn(B, n, heads, D, generator=r, device=dev),
              0.005 + 0.1 * torch.rand(B, n, heads, D, generator=r, device=dev)]
    d = [0.1 * torch.randn(B, T, H, D, generator=r, device=dev),
         -1e-4 - 0.02 * torch.rand(B, T, H, D, generator=r, device=dev)]
    c, start = 1 / math.sqrt(D), N - T
    got = run(x, d, scale=c, starts=torch.full((B,), start, device=dev))
    for a, b in zip(got, run(x, d, scale=c, starts=torch.full((B,), start, device=dev))):
        assert torch.equal(a, b)
    b = B - 1
    for first in sorted({0, T // 2, max(0, T - 7)}):
        last = min(T, first + 7)
        q = [t[b:b + 1, first:last] for t in (x[0], x[1], *d)]
        ref = attention(*q[:2], *(t[b:b + 1] for t in x[2:]), c, True, None, [start + first], deltas=q[2:])
        for g, w, n in zip(got[:4], ref, NAMES):
            within(g[b:b + 1, first:last], w, f"{n} of {first}")
        if last == T:
            for g, w, n in zip(got[4:], ref[4:], NAMES[4:]):
                within(g[b:b + 1, start + first:], (w[0][:, start + first:], w[1][:, start + first:]), n)
