"""Weight deltas of very many rows: what one thread adds up in float32 stays short.

2^30 rows of one feature whose terms are all 1 + 2^-13 - 2^-20. From a sum of 2048 on a float32 has
steps of 2^-12 and loses half of one with every such term; up to 512 its steps are 2^-15 and less, so
a thread's sum of that many terms is off by 512 x 2^-16 at most, 2^-16 of itself. The block's 256 sums
are joined in float32 (256 steps of half a last place at most, 2^-16 of the whole), the blocks' in float64.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_weight_deltas_of_many_rows(dev):
    from triton_tagi_amd import kernels as K

    T, x = 1 << 29, 1 + 2.0**-13 - 2.0**-20
    one = torch.ones(1, 1, 1, 1, device=dev).expand(1, T, 1, 1)
    d = torch.full((1, 1, 1, 1), x, device=dev).expand(1, T, 1, 1)
    inv = torch.ones(1, T, 2, device=dev)
    w = torch.ones(1, device=dev)
    out = K.qk_norm_rotary_backward(d, d, d, d, one, one, inv, weights=(w, w, w, w))
    for t in out[:4]:
        assert (t == x).all()
    for t in out[4:]:
        assert abs(t.item() / (T * x) - 1) <= 2 * 2.0**-16
