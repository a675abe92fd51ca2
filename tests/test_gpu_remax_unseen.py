"""Keys that no query sees: in no sum, whatever they hold, also where they share a block with keys that are
seen; their own deltas are zeros."""

from __future__ import annotations

import pytest
import torch

from remax_reference import attention, within
from test_gpu_remax_attention import NAMES, inputs, run

pytestmark = pytest.mark.gpu

BAD = [float("nan"), float("inf"), -float("inf"), -torch.finfo(torch.float32).max]


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("D", [32, 80, 128])
def test_keys_after_the_last_query(bad, D, dev):
    """Causal queries end before the keys do: the later keys belong to nobody."""
    B, T, N, H, G = 2, 21, 45, 4, 2
    x, d = inputs(B, T, N, H, G, D, 12, dev)
    starts = [0, 13]
    ref = attention(*x, 0.2, True, None, starts, deltas=d)
    for t in x[2:]:
        for b, s in enumerate(starts):
            t[b, s + T:] = bad
    got = run(x, d, scale=0.2, starts=torch.tensor(starts, device=dev))
    for g, r, n in zip(got, ref, NAMES):
        within(g, r, n)
    for g in got[4:]:
        for b, s in enumerate(starts):
            assert not g[b, s + T:].any()
