"""Long sums of the sequence-model operators: inputs whose roundings all go one way, so that an
error that grows with a sum's length shows (random ones average it out).

U is a float32 rounding, at most 2^-24 of the value.
"""

from __future__ import annotations

import pytest
import torch

from test_gpu_sequence_ops import U, close, d64, g

pytestmark = pytest.mark.gpu


# ======================================================================== residual norm
@pytest.mark.parametrize("rows,D", [(65536, 8192), (512, 1 << 20), (8191, 65536), ((1 << 27) + 11, 3)])
def test_gamma_deltas_of_many_values(dev, rows, D):
    """Column sums of the constant 1 + 2^-16, which a float sum of 256 or more of them rounds down
    by half a step every time (512 of them: 128 U short). A float sum holds at most 32 terms
    before it is added in float64: 32 U, and 10 U for the products, the partial sums and the
    weight, of sums without cancellation."""
    from triton_tagi_amd.kernels import add_rms_norm_backward

    if torch.cuda.get_device_properties(dev).total_memory < 40 << 30:
        pytest.skip("needs 40 GB of GPU memory")
    c = 1.0 + 2.0**-16
    dz, ms = torch.full((rows, D), c, device=dev), torch.ones(rows, D, device=dev)
    inv, w, Sw = torch.ones(rows, 1, device=dev), torch.ones(D, device=dev), torch.full((D,), 0.5, device=dev)
    _, _, dmw, dSw = add_rms_norm_backward(dz, dz, ms, inv, w, Sw)
    del dz, ms
    want = torch.full((D,), rows * c, dtype=torch.float64)
    close(dmw, 0.5 * want, 42 * U * 0.5 * want, "delta_mw")
    close(dSw, 0.25 * want, 42 * U * 0.25 * want, "delta_Sw")


@pytest.mark.parametrize("rows,D,stream", [(9001, 8190, True), (8193, 8192, False), (40000, 2049, True), (33 * 1024, 4096, True),
                                           (70000, 5, False)])
def test_gamma_deltas_of_row_ranges_past_a_partial_sum(dev, rows, D, stream):
    """Random rows whose ranges end inside a partial sum, against float64 on the GPU."""
    from triton_tagi_amd.kernels import add_rms_norm_backward

    r = torch.Generator(device=dev).manual_seed(rows + D)
    draw = lambda *s: torch.randn(*s, generator=r, device=dev)  # noqa: E731
    dm, ms, ds = draw(rows, D), draw(rows, D), draw(rows, D)
    dS = -draw(rows, D).abs()
    inv, w, Sw = 0.5 + draw(rows, 1).abs(), draw(D), 0.01 + draw(D).abs()
    got = add_rms_norm_backward(dm, dS, ms, inv, w, Sw, *((ds, ds) if stream else ()))
    S = d64(Sw)
    x = ms.double() * inv.double()
    t = dm.double() * x
    close(got[2], S * d64(t.sum(0)), 42 * U * S * d64(t.abs().sum(0)), "delta_mw")
    t = dS.double() * x * x
    close(got[3], S * S * d64(t.sum(0)), 46 * U * S * S * d64(t.abs().sum(0)), "delta_Sw")
    del t, x
    for a, b, p in ((got[0], dm, 1), (got[1], dS, 2)):  # the rows' own deltas at the ranges' ends
        at = torch.tensor([0, 1, rows // 2, rows - 2, rows - 1], device=dev)
        k = (d64(inv[at]) * d64(w)) ** p
        e = d64(ds[at]) if stream else torch.zeros(5, D, dtype=torch.float64)
        close(a[at], d64(b[at]) * k + e, 6 * U * ((d64(b[at]) * k).abs() + e.abs()), "deltas at the sum")
