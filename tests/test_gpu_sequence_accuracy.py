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


# ==================================================================== linear attention
# g^8 of this float32 rounds to exactly 1/2 and is 0.82 U above it: the state of a token long ago
# is then multiplied without a rounding, and what rounding g^8 lost is the only error that grows.
HALF_IN_8 = 0.9170040488243103


def aged(T, dev):
    """g^a and g^(2a) of the ages a = 0 .. T - 1, in float64; the means compared reach 2^-119."""
    a = torch.arange(T, device=dev, dtype=torch.float64)
    return HALF_IN_8**a, HALF_IN_8 ** (2 * a)


def near_powers(got, want, roundings, what):
    """got (B, T, H) against want (T,), where that is a normal float."""
    on = want > 2.0**-118
    err = ((got.double() / want[None, :, None] - 1.0).abs())[:, on].max().item()
    assert err <= roundings * U, f"{what}: off by {err / U:.2f} U"


def test_what_an_uncorrected_decay_would_lose():
    """In float64: the powers without the correction miss the bounds of the tests below."""
    groups = 118  # 2^-118
    assert abs(0.5**groups / HALF_IN_8 ** (8 * groups) - 1.0) > 10 * 6 * U
    g16 = float(torch.tensor(HALF_IN_8**16, dtype=torch.float32))
    assert abs((g16 / HALF_IN_8**16) ** (groups // 2) - 1.0) > 4 * 5 * U


@pytest.mark.parametrize("B,H,D", [(256, 8, 16), (128, 8, 40), (64, 8, 128), (1, 2, 40), (2, 1, 128)])
def test_decay_powers_of_one_token(dev, B, H, D):
    """One token's contribution of ones, read by every later token (backward: by every earlier
    one): powers of the decay. Heads enough that no chunks are made: 3 roundings of a mean (the
    staged power, the operand's product with it, the product with the state), 4 of a variance
    with its weight, 6 of a squared mean. Few heads: the time axis is split, and each of at most
    T/32 chunks adds a rounding (two of a squared mean) and the state's way into it 4."""
    from triton_tagi_amd.kernels import linear_attention, linear_attention_backward

    T = 960
    dec = torch.full((H,), HALF_IN_8, device=dev)
    assert dec[0].item() == HALF_IN_8
    more = 0 if B * H >= 512 else T // 32 + 4
    g1, g2 = aged(T, dev)
    zeros = lambda: torch.zeros(B, T, H, D, device=dev)  # noqa: E731
    q, k, v, one = zeros(), zeros(), zeros(), zeros()
    q[..., 0] = 1.0
    k[:, 0, :, 0], v[:, 0] = 1.0, 1.0
    one[:, 0] = 1.0
    z = zeros()
    # variances of the values alone: So = P; variances of the queries alone: So = M^2
    mo, So, (M, P) = linear_attention(q, z, k, z, v, one, dec, return_state=True)
    near_powers(mo[..., 0], g1, 3 + more, "mo"), near_powers(mo[..., D - 1], g1, 3 + more, "mo")
    near_powers(So[..., 0], g2, 4 + more, "So of P"), near_powers(So[..., D - 1], g2, 4 + more, "So of P")
    last = M[:, :, 0].double() / g1[-1]
    assert g1[-1] > 2.0**-126 and (last - 1.0).abs().max().item() <= (3 + more) * U
    short = 400  # whose variances are normal floats
    P = linear_attention(q[:, :short], z[:, :short], k[:, :short], z[:, :short], v[:, :short], one[:, :short], dec,
                         return_state=True)[2][1]
    assert (P[:, :, 0].double() / g2[short - 1] - 1.0).abs().max().item() <= (3 + more) * U
    _, So = linear_attention(q, q, k, z, v, z, dec)
    near_powers(So[..., 0], g2, 6 + 2 * more, "So of M^2")
    # queries: the first token's key and value, deltas everywhere
    d = zeros()
    d[..., 0] = 1.0
    out = linear_attention_backward(q, k, v, d, -d, dec)
    near_powers(out[0][..., 0], g1, 3 + more, "dmq"), near_powers(-out[1][..., 0], g2, 6 + 2 * more, "dSq")
    # keys and values: the last token's deltas, keys and values everywhere
    d.zero_(), k.zero_(), v.zero_()
    d[:, -1] = 1.0
    k[..., 0], v[..., 0] = 1.0, 1.0
    out = linear_attention_backward(q, k, v, d, -d, dec)
    for i, what in ((2, "dk"), (4, "dv")):
        near_powers(out[i].flip(1)[..., 0], g1, 3 + more, what + " mean")
        near_powers(-out[i + 1].flip(1)[..., 0], g2, 4 + more, what + " variance")


class Scan:
    """A state's values, sums of magnitudes and rounding bounds (in U), token by token: a
    contribution is rounded ``first`` times when it enters and, with the sum it is in, ``per``
    times a token from then on, so errors count by the age of what the decay has left."""

    def __init__(self, g, first, per, init=None, like=None):
        self.g, self.ga, self.first, self.per = g, g.abs(), first, per
        self.val = torch.zeros_like(like) if init is None else init
        self.mag, self.err = self.val.abs(), 2 * self.val.abs()

    def add(self, x, mag, on):
        new = (self.g * self.val + x, self.ga * self.mag + mag,
               self.ga * (self.err + self.per * self.mag) + self.first * mag)
        self.val, self.mag, self.err = (torch.where(on, a, b) for a, b in zip(new, (self.val, self.mag, self.err)))


def check_by_age(dev, B, T, H, D, decay, lengths=None, state=False, signs=True, seed=0):
    """Forward, end state and backward against float64 scans on the GPU with bounds by age.

    Means: 8 roundings of a staged contribution and 2.25 a token (the sum; the decay of a group
    of 8, or of every token below a quarter; a chunk's carry of 3 in 32). Variances: twice the
    operands, two sums and a rounded squared decay a token: 16 and 4.25. Reading: D + 24, twice
    that where the operand is squared."""
    from triton_tagi_amd.kernels import linear_attention, linear_attention_backward

    r = torch.Generator(device=dev).manual_seed(seed + 7 * T + D)
    c = 0.4
    shape = (B, T, H, D)

    def mean(std):
        x = std * torch.randn(shape, generator=r, device=dev)
        return x if signs else x.abs()

    def var(lo=0.01, hi=0.11):
        return lo + (hi - lo) * torch.rand(shape, generator=r, device=dev)

    mq, Sq, mk, Sk, mv, Sv = mean(1.0), var(), mean(0.5), var(), mean(1.0), var()
    dm, dS = mean(0.3), -var(0.0, 1.0)
    st = None
    if state:
        st = (torch.randn(B, H, D, D, generator=r, device=dev), torch.rand(B, H, D, D, generator=r, device=dev))
    dec = decay.to(dev)
    ln = None if lengths is None else lengths.to(dev)
    mo, So, ends = linear_attention(mq, Sq, mk, Sk, mv, Sv, dec, scale=c, lengths=ln, state=st, return_state=True)
    got = linear_attention_backward(mq, mk, mv, dm, dS, dec, scale=c, lengths=ln)

    g = dec.double()[None, :, None, None]
    like = torch.zeros(B, H, D, D, device=dev, dtype=torch.float64)
    init = (None, None) if st is None else tuple(t.double() for t in st)
    read = D + 24
    col, row = (lambda x: x.double()[..., :, None]), (lambda x: x.double()[..., None, :])
    live = torch.ones(B, T, dtype=torch.bool, device=dev) if ln is None else torch.arange(T, device=dev) < ln[:, None]

    def compare(t, got, ref, bound, what, dim):
        on = live[:, t][:, None, None]
        ref, bound = (torch.where(on, x.sum(dim), 0.0) for x in (ref, bound))
        over = ((got[:, t].double() - ref).abs() - U * bound - 1e-37).max().item()
        assert over <= 0, f"{what} of token {t}: over by {over:.3g}"

    M, P = Scan(g, 8, 2.25, init[0], like), Scan(g * g, 16, 4.25, init[1], like)
    Z = M if st is None else Scan(g, 8, 2.25, None, like)  # the backward's, from zeros
    for t in range(T):
        on = live[:, t][:, None, None, None]
        k, v, vk, vv = col(mk[:, t]), row(mv[:, t]), col(Sk[:, t]), row(Sv[:, t])
        for s in (M,) if Z is M else (M, Z):
            s.add(k * v, (k * v).abs(), on)
        new = vk * (v * v + vv) + k * k * vv
        P.add(new, new, on)
        q, vq = col(mq[:, t]), col(Sq[:, t])
        compare(t, mo, c * q * M.val, c * q.abs() * (M.err + read * M.mag), "mo", 2)
        w = vq + q * q
        compare(t, So, c * c * (w * P.val + vq * M.val**2),
                c * c * (w * (P.err + 2 * read * P.mag) + vq * M.mag * 2 * (M.err + read * M.mag)), "So", 2)
        d, e = c * row(dm[:, t]), c * c * row(dS[:, t])
        compare(t, got[0], d * Z.val, d.abs() * (Z.err + read * Z.mag), "dmq", 3)
        compare(t, got[1], e * Z.val**2, e.abs() * Z.mag * 2 * (Z.err + read * Z.mag), "dSq", 3)
    for end, s, what in ((ends[0], M, "M"), (ends[1], P, "P")):
        over = ((end.double() - s.val).abs() - U * (s.err + 4 * s.mag) - 1e-37).max().item()
        assert over <= 0, f"{what}: over by {over:.3g}"
    G, N = Scan(g, 8, 2.25, None, like), Scan(g * g, 16, 4.25, None, like)
    for t in reversed(range(T)):
        on = live[:, t][:, None, None, None]
        q, d, e = col(mq[:, t]), c * row(dm[:, t]), c * c * row(dS[:, t])
        G.add(q * d, (q * d).abs(), on)
        N.add(q * q * e, (q * q * e).abs(), on)
        k, v = col(mk[:, t]), row(mv[:, t])
        compare(t, got[2], G.val * v, (G.err + read * G.mag) * v.abs(), "dmk", 3)
        compare(t, got[3], N.val * v * v, (N.err + 2 * read * N.mag) * v * v, "dSk", 3)
        compare(t, got[4], G.val * k, (G.err + read * G.mag) * k.abs(), "dmv", 2)
        compare(t, got[5], N.val * k * k, (N.err + 2 * read * N.mag) * k * k, "dSv", 2)


@pytest.mark.parametrize("signs", [True, False])
@pytest.mark.parametrize("B,T,H,D,decay", [(1, 2100, 3, 24, (0.996, 0.8, 0.26)), (2, 1111, 1, 65, (0.99,)),
                                           (1, 2100, 2, 128, (0.9, 0.24)), (256, 300, 8, 16, (0.97, 0.9, 0.5, 0.99) * 2)])
def test_errors_follow_the_memory_not_the_length(dev, B, T, H, D, decay, signs):
    """Slow decays over many tokens, with operands of one sign too, whose roundings do not cancel."""
    check_by_age(dev, B, T, H, D, torch.tensor(decay), signs=signs, state=T == 1111)
