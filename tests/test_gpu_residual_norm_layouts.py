"""Sum and RMSNorm in every layout of its kernels (threads and chunks of a row), with batches
large enough for the nontemporal policy (256 MB of traffic), against float64 on the GPU with the
bounds of test_gpu_sequence_ops."""

from __future__ import annotations

import pytest
import torch

from test_gpu_sequence_ops import U, close

pytestmark = pytest.mark.gpu

# rows, D: threads of a row x chunks of four values a thread
SMALL = [(9, 250), (4100, 510), (4100, 1022), (300, 1021), (513, 2046), (600, 4095), (520, 8190),
         (100, 3001), (100, 8191), (40, 16381), (20, 32766)]
LARGE = [(50000, 201), (20000, 510), (10000, 1022), (5000, 2046), (2500, 4095), (1200, 8190), (600, 16381), (600, 32766)]


@pytest.mark.parametrize("rows,D", SMALL + LARGE)
def test_layout(dev, rows, D):
    from triton_tagi_amd.kernels import add_rms_norm, add_rms_norm_backward

    r = torch.Generator(device=dev).manual_seed(rows + D)
    normal = lambda *s: torch.randn(*s, generator=r, device=dev)  # noqa: E731
    ma, mr, dm, ds = (normal(rows, D) for _ in range(4))
    Sa, Sr, dS = normal(rows, D).abs(), normal(rows, D).abs(), -normal(rows, D).abs()
    w, Sw = normal(D), 0.01 + normal(D).abs()
    mz, Sz, ms, Ss, inv = add_rms_norm(ma, Sa, mr, Sr, w, Sw, 1e-5)
    out = add_rms_norm_backward(dm, dS, ms, inv, w, Sw, ds, dS)
    k = (D / 256 + 28) * U
    m, S, g, gS = ma.double() + mr.double(), Sa.double() + Sr.double(), w.double(), Sw.double()
    i = ((m * m + S).mean(1, keepdim=True) + 1e-5).rsqrt()
    d, e, s = dm.double(), dS.double(), ds.double()

    def check(got, ref, bound, what):
        assert torch.isfinite(got).all(), what
        over = ((got.double() - ref).abs() - bound).max().item()
        assert over <= 0, f"{what}: over by {over:.3g}"

    check(ms, m, U * m.abs(), "ms"), check(Ss, S, U * S, "Ss"), check(inv, i, k * i, "inv")
    check(mz, m * i * g, k * (m * i * g).abs(), "mz")
    ref = i * i * (S * (g * g + gS) + gS * m * m)
    check(Sz, ref, 2 * k * ref, "Sz")
    check(out[0], d * i * g + s, k * ((d * i * g).abs() + s.abs()), "delta_m")
    ref = e * (i * g) ** 2 + e
    check(out[1], ref, 2 * k * ref.abs(), "delta_S")
    kc = k + 42 * U
    x = m * i
    close(out[2], gS * (d * x).sum(0), (kc * gS * (d * x).abs().sum(0)).cpu(), "delta_mw")
    ref = gS * gS * (e * x * x).sum(0)
    close(out[3], ref, (2 * kc * ref.abs()).cpu(), "delta_Sw")
