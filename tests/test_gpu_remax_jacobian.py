"""The scores' deltas with a Jacobian that is formed another way.

``oracle.remax_moments`` has the covariance of weight and score through logarithms of the log-normal
stage, as the reference's Remax does; ``remax_reference`` has it multiplied out, as the kernels do. The
two agree in float64 here, and the kernels' deltas with products of the oracle's own.
"""

from __future__ import annotations

import math

import pytest
import torch

from oracle import tagi_oracle as O
from remax_reference import Row, attention, d64, seen_mask
from test_gpu_remax_attention import inputs, run

pytestmark = pytest.mark.gpu


def moments(x, b, h, g, n, c):
    q, S = (d64(t)[b, :, h] for t in x[:2])
    k, K = (d64(t)[b, :n, g] for t in x[2:4])
    return c * (q @ k.T), c * c * (S @ (k * k + K).T + (q * q) @ K.T)


@pytest.mark.parametrize("spread", [0.3, 1.0, 2.0])
@pytest.mark.parametrize("B,T,H,G,D", [(2, 9, 4, 2, 16), (1, 40, 2, 1, 64), (1, 33, 3, 3, 80)])
def test_score_deltas_with_the_oracles_jacobian(B, T, H, G, D, spread, dev):
    x, d = inputs(B, T, T, H, G, D, 21, dev, spread)
    c, R = 1 / math.sqrt(D), H // G
    got = run(x, d, scale=c)[2:6]
    bounds = [b for _, b in attention(*x, c, deltas=d)[2:6]]
    want, slack = ([torch.zeros(t.shape, dtype=torch.float64) for t in got] for _ in range(2))
    for b in range(B):
        for h in range(H):
            g = h // R
            m, v = moments(x, b, h, g, T, c)
            q, k, val = d64(x[0])[b, :, h], d64(x[2])[b, :, g], d64(x[4])[b, :, g]
            J = torch.zeros(T, T, dtype=torch.float64)
            for t in range(T):  # a row of the keys that the query sees
                J[t, :t + 1] = O.remax_moments(m[t:t + 1, :t + 1], v[t:t + 1, :t + 1])[2]
            row = Row(q, d64(x[1])[b, :, h], k, d64(x[3])[b, :, g], val, d64(x[5])[b, :, g],
                      seen_mask(T, T, True, T, 0), c)
            # the logarithms of 1 + small lose 2^-53 / small of it, down to variances of a millionth of the score's
            assert ((row.J - J).abs() <= 1e-6 * J).all()
            e = c * J * (d64(d[0])[b, :, h] @ val.T)
            E = c * c * J * J * (d64(d[1])[b, :, h] @ (val * val).T)
            want[0][b, :, h] = e @ k
            want[1][b, :, h] = E @ (k * k)
            want[2][b, :, g] += e.T @ q
            want[3][b, :, g] += E.T @ (q * q)
            slack[0][b, :, h] = 1e-6 * e.abs() @ k.abs()
            slack[1][b, :, h] = 2e-6 * E.abs() @ (k * k)
            slack[2][b, :, g] += 1e-6 * e.abs().T @ q.abs()
            slack[3][b, :, g] += 2e-6 * E.abs().T @ (q * q)
    for a, w, s, bound, n in zip(got, want, slack, bounds, ("dmq", "dSq", "dmk", "dSk")):
        over = (d64(a) - w).abs() - bound - s
        assert (over <= 0).all(), f"{n}: over by {over.max().item():.3g}"
