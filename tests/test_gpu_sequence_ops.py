"""Sequence-model operators against plain float64 forms on the CPU.

Tolerances count roundings (a float32 rounding is off by at most 2^-24 of the value):

* embedding sums: a piece's running sum rounds at most 64 times, partial sums are joined in
  float64, and the weights add 6 more: (64 + 6) 2^-24 of c Sw sum|delta|.
* norm: a row's mean of squares is summed with at most D/256 + 16 roundings of positive terms
  (a thread's share, then the threads'), its root halves that, and 12 more follow:
  (D/256 + 28) 2^-24 of the value. Column sums round once per row of a block's range, at most
  rows/512 + 32, and 10 times more.
* linear attention: a contribution to the state is rounded when staged (up to 8 times with
  its power of the decay) and then at most once per token and twice per 8 tokens; chunks add
  two roundings each 32 or more tokens; reading it adds D: (1.5 T + D + 32) 2^-24 of the same sums over
  absolute values, twice that where the state enters squared.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24


def g(seed):
    return torch.Generator().manual_seed(seed)


def d64(t):
    return t.detach().to("cpu", torch.float64)


def close(got, ref, bound, what):
    got, ref = d64(got), d64(ref)
    assert got.shape == ref.shape, f"{what}: {tuple(got.shape)} vs {tuple(ref.shape)}"
    over = (got - ref).abs() - bound
    assert torch.isfinite(got).all(), f"{what}: not finite"
    i = int(over.reshape(-1).argmax()) if over.numel() else 0
    assert over.numel() == 0 or over.reshape(-1)[i] <= 0, (
        f"{what}: got {got.reshape(-1)[i].item():.9g} ref {ref.reshape(-1)[i].item():.9g}, over by {over.reshape(-1)[i].item():.3g}")


# =========================================================================== embedding
def emb_inputs(n, V, D, kind, dtype, seed):
    r = g(seed)
    if kind == "uniform":
        ids = torch.randint(0, V, (n,), generator=r)
    elif kind == "one":  # one category takes every token: its run crosses every piece
        ids = torch.full((n,), V // 2)
    elif kind == "runs":  # runs of 64 end exactly at the pieces' borders
        ids = (torch.arange(n) // 64) % V
    else:  # half of them one category, the others spread
        ids = torch.where(torch.rand(n, generator=r) < 0.5, V - 1, torch.randint(0, V, (n,), generator=r))
    mw, Sw = torch.randn(V, D, generator=r), 0.01 + torch.rand(V, D, generator=r)
    dm, dS = torch.randn(n, D, generator=r), -torch.rand(n, D, generator=r)
    return ids.to(dtype), mw, Sw, dm, dS


def emb_reference(ids, dm, dS, Sw, c, pad):
    V = Sw.shape[0]
    real = (ids != pad) & (ids >= 0) & (ids < V)
    at = ids[real].long()
    S = d64(Sw)
    out = []
    for x, w in ((dm, c * S), (dS, (c * S) ** 2)):
        x = d64(x)[real]
        out += [w * torch.zeros_like(S).index_add_(0, at, x), w * torch.zeros_like(S).index_add_(0, at, x.abs())]
    return out  # deltas, their absolute sums, variance deltas, theirs


EMB = [
    (0, 5, 8, "uniform", torch.float32, -1, 1.0),
    (1, 1, 1, "uniform", torch.float32, -1, 3.0),
    (1, 40, 256, "uniform", torch.int64, -1, 16.0),
    (63, 7, 3, "uniform", torch.int32, 0, 0.5),
    (64, 2, 130, "one", torch.int64, -1, 2.0),
    (129, 300, 260, "mixed", torch.float32, 3, 1.0),
    (1000, 1023, 33, "mixed", torch.int64, 1022, 1.7),
    (1024, 1024, 64, "runs", torch.int32, -1, 1.0),
    (4097, 17, 8, "one", torch.float32, -1, 4.0),
    (5000, 3, 516, "uniform", torch.int32, 1, 2.0),
    (30011, 70001, 12, "mixed", torch.int64, -1, 8.0),
]


@pytest.mark.parametrize("n,V,D,kind,dtype,pad,c", EMB)
def test_embedding_lookup_deltas_update(dev, n, V, D, kind, dtype, pad, c):
    from triton_tagi_amd.kernels import embedding_lookup, embedding_param_deltas, embedding_update
    from triton_tagi_amd.update import update_parameters

    ids, mw, Sw, dm, dS = emb_inputs(n, V, D, kind, dtype, 7 * n + V + D)
    gi, gm, gS, gdm, gdS = (t.to(dev) for t in (ids, mw, Sw, dm, dS))
    mz, Sz = embedding_lookup(gi, gm, gS, scale=c, padding_idx=pad)
    real = (ids != pad)[:, None]
    rm, rS = torch.where(real, c * d64(mw)[ids.long()], 0.0), torch.where(real, c * c * d64(Sw)[ids.long()], 0.0)
    close(mz, rm, 2 * U * rm.abs(), "mz")
    close(Sz, rS, 2 * U * rS.abs(), "Sz")
    dmw, dSw = embedding_param_deltas(gi, gdm, gdS, gS, scale=c, padding_idx=pad)
    rm, am, rS, aS = emb_reference(ids, dm, dS, Sw, c, pad)
    close(dmw, rm, 70 * U * am, "delta_mw")
    close(dSw, rS, 70 * U * aS, "delta_Sw")
    again = embedding_param_deltas(gi, gdm, gdS, gS, scale=c, padding_idx=pad)
    assert torch.equal(dmw, again[0]) and torch.equal(dSw, again[1])
    # in place: the bits of the deltas and the update kernel after them
    m1, S1, m2, S2, m3, S3 = gm.clone(), gS.clone(), gm.clone(), gS.clone(), gm.clone(), gS.clone()
    update_parameters(m1, S1, dmw, dSw, 2.0)
    kept = embedding_update(gi, gdm, gdS, m2, S2, 2.0, scale=c, padding_idx=pad, keep_deltas=True)
    assert embedding_update(gi, gdm, gdS, m3, S3, 2.0, scale=c, padding_idx=pad) == (None, None)
    assert torch.equal(kept[0], dmw) and torch.equal(kept[1], dSw)
    for a, b, x in ((m1, m2, m3), (S1, S2, S3)):
        assert torch.equal(a, b) and torch.equal(a, x)


@pytest.mark.parametrize("n,V", [((1 << 20) + 77, 1), (1 << 20, 7), (32769, 1), (32768, 500), (32700, 511), (20000, 70000)])
def test_embedding_tables_and_batches_of_unlike_size(dev, n, V):
    """Many tokens of few categories, and batches at the borders of the sort's forms."""
    test_embedding_lookup_deltas_update(dev, n, V, 2, "uniform", torch.int32, -1, 1.5)


def test_embedding_ids_outside_the_table(dev):
    from triton_tagi_amd.kernels import embedding_lookup, embedding_param_deltas

    V, D = 9, 5
    r = g(3)
    mw, Sw = torch.randn(V, D, generator=r), torch.rand(V, D, generator=r)
    for ids in (torch.tensor([-7.0, 3.9, math.nan, math.inf, -math.inf, 8.0, 9.0, 1e30, -0.5, -1.0]),
                torch.tensor([-7, 3, 2**31 - 1, -2**31, 9, 8, -1, 10, 0, 9], dtype=torch.int32),
                torch.tensor([-7, 3, 2**62, -2**62, 2**32 + 1, 8, -1, 9, 0, 2**33], dtype=torch.int64)):
        ok = (ids > -1) & (ids < V)
        at = torch.where(ok, ids, 0).long()  # toward zero: 3.9 is 3 and -0.5 is 0
        dm, dS = torch.randn(10, D, generator=r), torch.randn(10, D, generator=r)
        mz, Sz = embedding_lookup(ids.to(dev), mw.to(dev), Sw.to(dev))
        assert torch.equal(mz.cpu(), torch.where(ok[:, None], mw[at], 0.0))
        assert torch.equal(Sz.cpu(), torch.where(ok[:, None], Sw[at], 0.0))
        dmw, dSw = embedding_param_deltas(ids.to(dev), dm.to(dev), dS.to(dev), Sw.to(dev))
        rm, am, rS, aS = emb_reference(torch.where(ok, at, -1), dm, dS, Sw, 1.0, -1)
        close(dmw, rm, 70 * U * am, "delta_mw")
        close(dSw, rS, 70 * U * aS, "delta_Sw")


def test_embedding_strides_and_shapes(dev):
    """ids of any shape, strided ids, deltas and tables."""
    from triton_tagi_amd.kernels import embedding_lookup, embedding_param_deltas

    r = g(11)
    ids = torch.randint(0, 6, (4, 10), generator=r).to(dev)
    wide, wideS = torch.randn(6, 14, generator=r).to(dev), torch.rand(6, 14, generator=r).to(dev)
    mw, Sw = wide[:, 3:11], wideS[:, 3:11]
    mz, Sz = embedding_lookup(ids.t(), mw, Sw, scale=2.0)
    assert mz.shape == (10, 4, 8) and torch.equal(mz, 2.0 * mw[ids.t()]) and torch.equal(Sz, 4.0 * Sw[ids.t()])
    dm, dS = torch.randn(4, 10, 8, generator=r).to(dev), torch.randn(4, 10, 8, generator=r).to(dev)
    a = embedding_param_deltas(ids.t(), dm.transpose(0, 1), dS.transpose(0, 1), Sw)
    rm, am, rS, aS = emb_reference(ids.cpu().reshape(-1), dm.cpu().reshape(-1, 8), dS.cpu().reshape(-1, 8), Sw.cpu(), 1.0, -1)
    close(a[0], rm, 70 * U * am, "delta_mw")
    close(a[1], rS, 70 * U * aS, "delta_Sw")


# ======================================================================== residual norm
@pytest.mark.parametrize("rows,D", [(1, 1), (3, 2), (1, 63), (64, 64), (257, 257), (33, 256), (1031, 100), (5, 1024),
                                    (2, 4097), (7, 8192), (1, 20000), (40000, 4)])
@pytest.mark.parametrize("stream", [True, False])
def test_add_rms_norm(dev, rows, D, stream):
    from triton_tagi_amd.kernels import add_rms_norm, add_rms_norm_backward

    r = g(rows * 13 + D)
    ma, mr = torch.randn(rows, D, generator=r), 2.0 * torch.randn(rows, D, generator=r)
    Sa, Sr = torch.rand(rows, D, generator=r), torch.rand(rows, D, generator=r)
    mw, Sw = 1.0 + 0.1 * torch.randn(D, generator=r), 0.01 + 0.01 * torch.rand(D, generator=r)
    dm, dS = torch.randn(rows, D, generator=r), -torch.rand(rows, D, generator=r)
    ds, dSs = torch.randn(rows, D, generator=r), -torch.rand(rows, D, generator=r)
    dv = lambda *ts: [t.to(dev) for t in ts]  # noqa: E731
    mz, Sz, ms, Ss, inv = add_rms_norm(*dv(ma, Sa, mr, Sr, mw, Sw), 1e-5, need_sum_var=stream)
    m, S, gm, gS = d64(ma) + d64(mr), d64(Sa) + d64(Sr), d64(mw), d64(Sw)
    i = ((m * m + S).mean(1, keepdim=True) + 1e-5).rsqrt()
    k = (D / 256 + 28) * U
    close(ms, m, U * m.abs(), "ms")
    if stream:
        close(Ss, S, U * S, "Ss")
    else:
        assert Ss is None
    assert inv.shape == (rows, 1)
    close(inv, i, k * i, "inv")
    close(mz, m * i * gm, k * (m * i * gm).abs(), "mz")
    rS = i * i * (S * (gm * gm + gS) + gS * m * m)
    close(Sz, rS, 2 * k * rS, "Sz")
    out = add_rms_norm_backward(*dv(dm, dS), ms, inv, *dv(mw, Sw), *(dv(ds, dSs) if stream else ()))
    dm, dS, ds, dSs = (d64(t) for t in (dm, dS, ds, dSs))
    if not stream:
        ds, dSs = torch.zeros_like(ds), torch.zeros_like(dSs)
    w, x = i * gm, m * i
    close(out[0], dm * w + ds, k * ((dm * w).abs() + ds.abs()), "delta_m")
    close(out[1], dS * w * w + dSs, 2 * k * (dS * w * w + dSs).abs(), "delta_S")
    kc = k + (rows / 512 + 42) * U
    close(out[2], gS * (dm * x).sum(0), kc * gS * (dm * x).abs().sum(0), "delta_mw")
    close(out[3], gS * gS * (dS * x * x).sum(0), 2 * kc * gS * gS * (dS * x * x).sum(0).abs(), "delta_Sw")


@pytest.mark.parametrize("rows,D", [(3, 32768), (3, 32769), (2, 40003)])
def test_add_rms_norm_of_the_longest_rows(dev, rows, D):
    """The longest rows that stay in registers, and longer ones."""
    test_add_rms_norm(dev, rows, D, True)


def test_add_rms_norm_is_add_then_norm(dev):
    """The container layers' path equals Add followed by RMSNorm within both forms' roundings."""
    from triton_tagi_amd import Add, RMSNorm
    from triton_tagi_amd.kernels import add_rms_norm

    r = g(5)
    ma, mr = (torch.randn(6, 9, 48, generator=r).to(dev) for _ in range(2))
    Sa, Sr = (torch.rand(6, 9, 48, generator=r).to(dev) for _ in range(2))
    norm = RMSNorm(48)
    ms, Ss = Add().forward(ma, Sa, mr, Sr)
    rz, rS = norm.forward(ms, Ss)
    mz, Sz, m2, S2, _ = add_rms_norm(ma, Sa, mr, Sr, norm.mw, norm.Sw, norm.eps)
    assert torch.equal(m2, ms) and torch.equal(S2, Ss)
    close(mz, rz, 60 * U * d64(rz).abs(), "mz")
    close(Sz, rS, 120 * U * d64(rS).abs(), "Sz")


def test_add_rms_norm_infinities_stay_in_their_rows(dev):
    from triton_tagi_amd.kernels import add_rms_norm

    ma, Sa = torch.ones(5, 70, device=dev), torch.ones(5, 70, device=dev)
    bad = ma.clone()
    bad[1, 3], bad[3, 69] = math.inf, math.nan
    mw, Sw = torch.ones(70, device=dev), torch.full((70,), 0.1, device=dev)
    want = add_rms_norm(ma, Sa, ma, Sa, mw, Sw)
    got = add_rms_norm(bad, Sa, ma, Sa, mw, Sw)
    for a, b in zip(got, want):
        assert torch.equal(a[[0, 2, 4]], b[[0, 2, 4]])
    assert got[0][3].isnan().all() and not got[0][1].isfinite().all()


# ==================================================================== linear attention
def lin_inputs(B, T, H, D, seed, dtype=torch.float32):
    r = g(seed)
    out = []
    for std in (1.0, 0.5, 1.0):
        out += [std * torch.randn(B, T, H, D, generator=r), 0.01 + 0.1 * torch.rand(B, T, H, D, generator=r)]
    return [t.to(dtype) for t in out]


def lin_reference(mq, Sq, mk, Sk, mv, Sv, decay, c, lengths=None, state=None):
    """Token by token in the inputs' type: outputs and the end state."""
    B, T, H, D = mq.shape
    M, P = (torch.zeros(B, H, D, D, dtype=mq.dtype) for _ in range(2)) if state is None else state
    gd = decay.to(mq.dtype)[None, :, None, None]
    mo, So = [], []
    for t in range(T):
        k, v = mk[:, t, :, :, None], mv[:, t, :, None, :]
        M1 = gd * M + k * v
        P1 = gd * gd * P + Sk[:, t, :, :, None] * (v * v + Sv[:, t, :, None, :]) + k * k * Sv[:, t, :, None, :]
        if lengths is not None:
            on = (t < lengths)[:, None, None, None]
            M, P = torch.where(on, M1, M), torch.where(on, P1, P)
        else:
            on, M, P = torch.ones(B, 1, 1, 1, dtype=torch.bool), M1, P1
        q, s = mq[:, t, :, :, None], Sq[:, t, :, :, None]
        mo.append(torch.where(on[..., 0], c * (q * M).sum(2), 0.0))
        So.append(torch.where(on[..., 0], c * c * ((s + q * q) * P + s * M * M).sum(2), 0.0))
    empty = torch.zeros(B, 0, H, D, dtype=mq.dtype)
    return (torch.stack(mo, 1) if T else empty), (torch.stack(So, 1) if T else empty), M, P


def lin_backward_reference(mq, mk, mv, dm, dS, decay, c, lengths=None):
    B, T, H, D = mq.shape
    if lengths is not None:
        on = (torch.arange(T) < lengths[:, None])[:, :, None, None]
        mq, mk, mv, dm, dS = (torch.where(on, x, 0.0) for x in (mq, mk, mv, dm, dS))
    gd = decay.to(mq.dtype)[None, :, None, None]
    z = torch.zeros(B, H, D, D, dtype=mq.dtype)
    d, e = c * dm, c * c * dS
    out = [torch.zeros_like(mq) for _ in range(6)]
    M = z
    for t in range(T):
        M = gd * M + mk[:, t, :, :, None] * mv[:, t, :, None, :]
        out[0][:, t] = (M * d[:, t, :, None, :]).sum(-1)
        out[1][:, t] = (M * M * e[:, t, :, None, :]).sum(-1)
    G = N = z
    for t in reversed(range(T)):
        G = gd * G + mq[:, t, :, :, None] * d[:, t, :, None, :]
        N = gd * gd * N + (mq[:, t] ** 2)[:, :, :, None] * e[:, t, :, None, :]
        out[2][:, t] = (G * mv[:, t, :, None, :]).sum(-1)
        out[3][:, t] = (N * (mv[:, t] ** 2)[:, :, None, :]).sum(-1)
        out[4][:, t] = (G * mk[:, t, :, :, None]).sum(-2)
        out[5][:, t] = (N * (mk[:, t] ** 2)[:, :, :, None]).sum(-2)
    return out


def decays(H):
    return torch.tensor([0.97, 0.0, 1.0, 0.03, 0.5, 0.999, 0.06, 0.9])[torch.arange(H) % 8]


def check_lin(dev, B, T, H, D, lengths=None, state=False, seed=0, decay=None, backward=True):
    from triton_tagi_amd.kernels import linear_attention, linear_attention_backward

    x = lin_inputs(B, T, H, D, seed + 31 * T + D)
    decay = decays(H) if decay is None else decay
    c = 1.0 / math.sqrt(D)
    r = g(seed + 1)
    st = (torch.randn(B, H, D, D, generator=r), torch.rand(B, H, D, D, generator=r)) if state else None
    ln = None if lengths is None else torch.tensor(lengths)
    gst = None if st is None else tuple(t.to(dev) for t in st)
    gx = [t.to(dev) for t in x]
    gl = None if ln is None else ln.to(dev)
    mo, So, (M, P) = linear_attention(*gx, decay.to(dev), scale=c, lengths=gl, state=gst, return_state=True)
    x64 = [d64(t) for t in x]
    ab = [t.abs() for t in x64]
    s64 = None if st is None else tuple(d64(t) for t in st)
    nn = None if ln is None else ln.clamp(0, T)
    ref = lin_reference(*x64, d64(decay), c, nn, s64)
    # sums over absolute values: of the decay's powers too (a negative decay alternates)
    mag = lin_reference(*ab, d64(decay).abs(), c, nn, None if s64 is None else tuple(t.abs() for t in s64))
    k = (1.5 * T + D + 32) * U
    for got, rf, mg, f, what in zip((mo, So, M, P), ref, mag, (1, 2, 1, 2), ("mo", "So", "M", "P")):
        close(got, rf, f * k * mg + 1e-37, what)
    if gst is not None:
        assert torch.equal(gst[0].cpu(), st[0]) and torch.equal(gst[1].cpu(), st[1])
    # without the state asked for, and on a second run: the same bits
    mo2, So2 = linear_attention(*gx, decay.to(dev), scale=c, lengths=gl, state=gst)
    assert torch.equal(mo, mo2) and torch.equal(So, So2)
    if not backward:
        return
    dm, dS = 0.3 * torch.randn(B, T, H, D, generator=r), -torch.rand(B, T, H, D, generator=r)
    got = linear_attention_backward(gx[0], gx[2], gx[4], dm.to(dev), dS.to(dev), decay.to(dev), scale=c, lengths=gl)
    ref = lin_backward_reference(x64[0], x64[2], x64[4], d64(dm), d64(dS), d64(decay), c, nn)
    mag = lin_backward_reference(ab[0], ab[2], ab[4], d64(dm).abs(), d64(dS).abs(), d64(decay).abs(), c, nn)
    for gt, rf, mg, what in zip(got, ref, mag, ("dmq", "dSq", "dmk", "dSk", "dmv", "dSv")):
        close(gt, rf, (2 if what[1] == "S" else 1) * k * mg + 1e-37, what)


@pytest.mark.parametrize("D", [1, 3, 15, 16, 17, 31, 32, 33, 48, 64, 65, 80, 96, 100, 127, 128])
def test_linear_attention_head_dims(dev, D):
    check_lin(dev, 2, 21, 3, D, seed=D)


@pytest.mark.parametrize("T", [0, 1, 2, 7, 8, 9, 15, 16, 17, 63, 64, 65, 130, 300])
@pytest.mark.parametrize("B,H,D", [(1, 8, 20), (3, 2, 64)])
def test_linear_attention_lengths_of_time(dev, T, B, H, D):
    check_lin(dev, B, T, H, D, seed=T, state=T % 2 == 0)


@pytest.mark.parametrize("T", [520, 1111, 4200])
def test_linear_attention_long(dev, T):
    """Few heads and long sequences: the time axis is split where that pays."""
    check_lin(dev, 1, T, 2, 24, seed=T, decay=torch.tensor([0.996, 0.8]))
    check_lin(dev, 2, T, 1, 65, seed=T, lengths=[T - 77, 300], state=True, decay=torch.tensor([0.99]))


# enough heads (or, split along time, enough chunks) that a wavefront takes 32 columns of the
# state, half as many that it takes 16; one for each padded head dimension
WIDE = [(1024, 3, 2, 30), (512, 3, 2, 30), (1024, 9, 2, 16), (512, 9, 2, 61), (256, 9, 2, 64), (342, 9, 2, 90),
        (171, 10, 2, 96), (256, 9, 2, 128), (128, 17, 2, 125), (32, 256, 8, 32), (8, 512, 8, 64), (6, 600, 7, 72),
        (4, 512, 8, 128), (3, 700, 8, 57), (33, 130, 3, 100)]


@pytest.mark.parametrize("B,T,H,D", WIDE)
def test_linear_attention_many_heads(dev, B, T, H, D):
    """As ``check_lin``, the float64 reference on the GPU (products and sums of tensors only)."""
    from triton_tagi_amd.kernels import linear_attention, linear_attention_backward

    x = [t.to(dev) for t in lin_inputs(B, T, H, D, B + T + D)]
    dec, c = decays(H).to(dev), 0.4
    r = g(B)
    ln = torch.randint(0, T + 1, (B,), generator=r).to(dev) if B % 2 else None
    dm, dS = torch.randn(B, T, H, D, generator=r).to(dev), -torch.rand(B, T, H, D, generator=r).to(dev)
    mo, So, (M, P) = linear_attention(*x, dec, scale=c, lengths=ln, return_state=True)
    bwd = linear_attention_backward(x[0], x[2], x[4], dm, dS, dec, scale=c, lengths=ln)
    x64 = [t.double() for t in x]
    ab = [t.abs() for t in x64]
    k = (1.5 * T + D + 32) * U

    with torch.device(dev):
        ref = lin_reference(*x64, dec.double(), c, ln)
        mag = lin_reference(*ab, dec.double(), c, ln)
        refb = lin_backward_reference(x64[0], x64[2], x64[4], dm.double(), dS.double(), dec.double(), c, ln)
        magb = lin_backward_reference(ab[0], ab[2], ab[4], dm.double().abs(), dS.double().abs(), dec.double(), c, ln)
    for got, rf, mg, f, what in zip((mo, So, M, P), ref, mag, (1, 2, 1, 2), ("mo", "So", "M", "P")):
        close(got, rf, f * k * d64(mg) + 1e-37, what)
    for got, rf, mg, what in zip(bwd, refb, magb, ("dmq", "dSq", "dmk", "dSk", "dmv", "dSv")):
        close(got, rf, (2 if what[1] == "S" else 1) * k * d64(mg) + 1e-37, what)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("state", [False, True])
def test_linear_attention_ragged(dev, dtype, state):
    """Lengths 0, 1, at and beside the stages' borders, and outside [0, T]."""
    T = 150
    lengths = [0, 1, 7, 8, 9, 64, 65, 149, 150, 999, -3]
    check_lin(dev, len(lengths), T, 2, 36, lengths=lengths, state=state, seed=5)
    from triton_tagi_amd.kernels import linear_attention, linear_attention_backward

    # what lies past a sequence's end is not read
    x = [t.to(dev) for t in lin_inputs(3, 40, 2, 16, 9)]
    ln = torch.tensor([0, 13, 40], dtype=dtype, device=dev)
    dec = decays(2).to(dev)
    dm, dS = x[0].clone(), x[1].clone()
    want = linear_attention(*x, dec, lengths=ln, return_state=True)
    wantb = linear_attention_backward(x[0], x[2], x[4], dm, dS, dec, lengths=ln)
    dead = torch.arange(40, device=dev) >= ln[:, None]
    for t in (*x, dm, dS):
        t[dead] = math.nan
    got = linear_attention(*x, dec, lengths=ln, return_state=True)
    gotb = linear_attention_backward(x[0], x[2], x[4], dm, dS, dec, lengths=ln)
    for a, b in zip((*got[:2], *got[2], *gotb), (*want[:2], *want[2], *wantb)):
        assert torch.equal(a, b)
    for a in (*got[:2], *gotb):
        assert (a[dead] == 0).all()


def test_linear_attention_negative_and_growing_decay(dev):
    check_lin(dev, 1, 50, 3, 8, decay=torch.tensor([-0.7, 1.05, -0.01]))


def test_linear_attention_strided_operands(dev):
    """Heads read in place from one (B, T, 3 H D) projection buffer, whatever its alignment,
    and expanded operands (one key head for all)."""
    from triton_tagi_amd.kernels import linear_attention, linear_attention_backward

    B, T, H, D = 2, 37, 3, 20
    dec = decays(H).to(dev)
    for pad in (0, 1, 4):  # 4 floats keep 16-byte alignment, 1 does not
        r = g(pad)
        bm, bS = torch.randn(B, T, 3 * H * D + pad, generator=r).to(dev), torch.rand(B, T, 3 * H * D + pad, generator=r).to(dev)
        cut = lambda b, i: b[:, :, pad + i * H * D:pad + (i + 1) * H * D].view(B, T, H, D)  # noqa: E731
        ops = [f for i in range(3) for f in (cut(bm, i), cut(bS, i))]
        packed = [t.contiguous() for t in ops]
        assert not ops[0].is_contiguous()
        for a, b in zip(linear_attention(*ops, dec), linear_attention(*packed, dec)):
            assert torch.equal(a, b)
        dm, dS = cut(bm, 2), cut(bS, 2)
        for a, b in zip(linear_attention_backward(ops[0], ops[2], ops[4], dm, dS, dec),
                        linear_attention_backward(packed[0], packed[2], packed[4], packed[4], packed[5], dec)):
            assert torch.equal(a, b)
    x = [t.to(dev) for t in lin_inputs(B, T, H, D, 4)]
    k1, S1 = x[2][:, :, :1].expand(B, T, H, D), x[3][:, :, :1].expand(B, T, H, D)
    for a, b in zip(linear_attention(x[0], x[1], k1, S1, x[4], x[5], dec),
                    linear_attention(x[0], x[1], k1.contiguous(), S1.contiguous(), x[4], x[5], dec)):
        assert torch.equal(a, b)
    t = [y.transpose(1, 2).contiguous().transpose(1, 2) for y in x]  # (B, H, T, D) storage
    for a, b in zip(linear_attention(*t, dec), linear_attention(*x, dec)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("D", [1, 7, 16, 33, 64, 100, 128])
def test_linear_attention_step(dev, D):
    """Tokens one by one from a state: the whole sequence's values, and the formula's."""
    from triton_tagi_amd.kernels import linear_attention, linear_attention_step

    B, T, H = 3, 9, 4
    x = lin_inputs(B, T, H, D, D)
    dec, c = decays(H), 0.3
    r = g(D)
    st = (torch.randn(B, H, D, D, generator=r), torch.rand(B, H, D, D, generator=r))
    ref = lin_reference(*(d64(t) for t in x), d64(dec), c, None, tuple(d64(t) for t in st))
    mag = lin_reference(*(d64(t).abs() for t in x), d64(dec), c, None, tuple(d64(t).abs() for t in st))
    gx = [t.to(dev) for t in x]
    first = linear_attention(*(t[:, :4] for t in gx), dec.to(dev), scale=c, state=tuple(t.to(dev) for t in st),
                             return_state=True)
    state, outs = first[2], [first[:2]]
    for t in range(4, T):
        outs.append(tuple(o[:, None] for o in linear_attention_step(*(y[:, t] for y in gx), state, dec.to(dev), scale=c)))
    k = (1.5 * T + D + 32) * U
    for i, (what, f) in enumerate((("mo", 1), ("So", 2))):
        close(torch.cat([o[i] for o in outs], 1), ref[i], f * k * mag[i], what)
        close(state[i], ref[2 + i], f * k * mag[2 + i], "state")


def test_linear_attention_step_inactive_sequences(dev):
    from triton_tagi_amd.kernels import linear_attention_step

    B, H, D = 4, 2, 24
    x = [t[:, 0].to(dev) for t in lin_inputs(B, 1, H, D, 2)]
    M, P = torch.randn(B, H, D, D, device=dev), torch.rand(B, H, D, D, device=dev)
    dec = decays(H).to(dev)
    for dtype in (torch.bool, torch.uint8):
        on = torch.tensor([1, 0, 1, 0], device=dev).to(dtype)
        a, b, want = (M.clone(), P.clone()), (M.clone(), P.clone()), None
        want = linear_attention_step(*x, a, dec)
        x2 = [t.clone() for t in x]
        for t in x2:
            t[[1, 3]] = math.nan
        got = linear_attention_step(*x2, b, dec, active=on)
        for i in range(2):
            assert torch.equal(got[i][[0, 2]], want[i][[0, 2]]) and (got[i][[1, 3]] == 0).all()
            assert torch.equal(b[i][[0, 2]], a[i][[0, 2]]) and torch.equal(b[i][[1, 3]], (M, P)[i][[1, 3]])


def test_linear_attention_backward_against_jacobians_and_differences(dev):
    """Mean deltas are J^T d of the output means. Variance deltas pass through the state's
    elements, each a Gaussian of its own: sum over the key features i of (J_i.J_i)^T e, J_i
    the Jacobian of c q_i M[i, :] (summing J_i first would correlate the elements). J from
    autograd, and from central differences, of the float64 forward."""
    from triton_tagi_amd.kernels import linear_attention_backward

    B, T, H, D = 1, 6, 2, 3
    x = lin_inputs(B, T, H, D, 77)
    dec, c = torch.tensor([0.9, 0.4]), 0.7
    r = g(8)
    dm, dS = torch.randn(B, T, H, D, generator=r), -torch.rand(B, T, H, D, generator=r)
    got = linear_attention_backward(x[0].to(dev), x[2].to(dev), x[4].to(dev), dm.to(dev), dS.to(dev), dec.to(dev), scale=c)
    x64 = [d64(t) for t in x]

    def parts(q, k, v):  # (D, B, T, H, D): feature i's share of the output means
        one = torch.eye(D, dtype=torch.float64)[:, None, None, None]
        return torch.stack([lin_reference(q * one[i], x64[1], k, x64[3], v, x64[5], d64(dec), c)[0] for i in range(D)])

    ops = (x64[0], x64[2], x64[4])
    jac = torch.autograd.functional.jacobian(parts, ops)
    n = dm.numel()
    k = (1.5 * T + D + 32) * U
    mags = lin_backward_reference(*(o.abs() for o in ops), d64(dm).abs(), d64(dS).abs(), d64(dec), c)
    for i, J in enumerate(jac):
        J = J.reshape(D, n, n)
        h = 1e-4
        for j in range(n):
            e = torch.zeros(n, dtype=torch.float64)
            e[j] = h
            hi, lo = ([o + (s * e.view_as(o) if a == i else 0.0) for a, o in enumerate(ops)] for s in (1, -1))
            # the output means are linear in each operand: differences carry rounding only
            assert torch.allclose((parts(*hi) - parts(*lo)).reshape(D, n) / (2 * h), J[:, :, j], rtol=0, atol=1e-9)
        close(got[2 * i].cpu().reshape(-1), J.sum(0).T @ d64(dm).reshape(-1), k * mags[2 * i].reshape(-1), "qkv"[i] + " mean")
        close(got[2 * i + 1].cpu().reshape(-1), (J * J).sum(0).T @ d64(dS).reshape(-1), 2 * k * mags[2 * i + 1].reshape(-1),
              "qkv"[i] + " variance")


# ============================================================================ large offsets
def test_offsets_past_32_bits(dev):
    """Tables, rows and strides whose element offsets pass 2^32."""
    from triton_tagi_amd.kernels import (add_rms_norm, add_rms_norm_backward, embedding_lookup, embedding_param_deltas,
                                         embedding_update, linear_attention, linear_attention_backward)

    if torch.cuda.get_device_properties(dev).total_memory < 150 << 30:
        pytest.skip("needs 150 GB of GPU memory")
    r = g(1)
    V, D = (1 << 21) + 3, 2052  # 4.3e9 elements
    mw, Sw = torch.full((V, D), 0.5, device=dev), torch.full((V, D), 0.25, device=dev)
    ids = torch.tensor([V - 1, 5, V - 1, 1 << 21, V], device=dev)
    mw[V - 1] = torch.arange(D, device=dev, dtype=torch.float32)
    mz, Sz = embedding_lookup(ids, mw, Sw, scale=2.0)
    assert torch.equal(mz[0], 2.0 * mw[V - 1]) and torch.equal(mz[3], 2.0 * mw[1 << 21]) and (mz[4] == 0).all()
    dm = torch.randn(5, D, generator=r).to(dev)
    dmw, dSw = embedding_param_deltas(ids, dm, dm, Sw, scale=2.0)
    close(dmw[V - 1], 0.5 * (d64(dm[0]) + d64(dm[2])), 70 * U * 0.5 * (d64(dm[0]).abs() + d64(dm[2]).abs()), "last row")
    assert torch.equal(dmw[5], 0.5 * dm[1]) and (dmw[V - 2] == 0).all() and (dSw[V - 2] == 0).all()
    assert int((dmw != 0).any(1).sum()) == 3
    del dmw, dSw
    before = mw[V - 1].clone()
    embedding_update(ids, dm, dm, mw, Sw, 3.0, scale=2.0)
    assert not torch.equal(mw[V - 1], before) and (mw[V - 2] == 0.5).all()
    del mw, Sw
    rows, D = (1 << 20) + 1, 2056  # 2.2e9 elements
    m, S = torch.full((rows, D), 0.5, device=dev), torch.full((rows, D), 0.25, device=dev)
    m[rows - 1] = torch.randn(D, generator=r).to(dev)
    w, Sg = torch.ones(D, device=dev), torch.full((D,), 0.01, device=dev)
    mz, Sz, ms, _, inv = add_rms_norm(m, S, m, S, w, Sg, need_sum_var=False)
    want = add_rms_norm(m[-3:], S[-3:], m[-3:], S[-3:], w, Sg)
    assert torch.equal(mz[-3:], want[0]) and torch.equal(Sz[-3:], want[1]) and torch.equal(inv[-3:], want[4])
    del Sz
    out = add_rms_norm_backward(mz, S, ms, inv, w, Sg)
    tail = add_rms_norm_backward(mz[-3:], S[-3:], ms[-3:], inv[-3:], w, Sg)
    assert torch.equal(out[0][-3:], tail[0]) and torch.equal(out[1][-3:], tail[1])
    del m, S, mz, ms, inv, out
    T, H, D = 20, 2, 24
    buf = torch.empty((T - 1) * (1 << 28) + 2 * H * D, device=dev)  # 5.1e9 elements
    x = [t.to(dev) for t in lin_inputs(1, T, H, D, 3)]
    far = buf.as_strided((1, T, H, D), (0, 1 << 28, D, 1))
    farS = buf.as_strided((1, T, H, D), (0, 1 << 28, D, 1), H * D)
    far.copy_(x[2]), farS.copy_(x[3])
    dec = decays(H).to(dev)
    for a, b in zip(linear_attention(x[0], x[1], far, farS, x[4], x[5], dec), linear_attention(*x, dec)):
        assert torch.equal(a, b)
    for a, b in zip(linear_attention_backward(x[0], far, x[4], far, farS, dec),
                    linear_attention_backward(x[0], x[2], x[4], x[2], x[3], dec)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("rows,D", [((1 << 22) + 5, 3), ((1 << 26) + 3, 5)])
def test_norm_of_more_rows_than_one_grid_dimension(dev, rows, D):
    """The last rows of a batch whose blocks pass 2^32 threads: the same bits as by themselves."""
    from triton_tagi_amd.kernels import add_rms_norm, add_rms_norm_backward

    r = g(4)
    m, S = torch.full((rows, D), 0.5, device=dev), torch.full((rows, D), 0.25, device=dev)
    m[-3:], S[-3:] = torch.randn(3, D, generator=r).to(dev), torch.rand(3, D, generator=r).to(dev)
    w, Sg = torch.randn(D, generator=r).to(dev), torch.rand(D, generator=r).to(dev)
    got, want = add_rms_norm(m, S, m, S, w, Sg), add_rms_norm(m[-3:], S[-3:], m[-3:], S[-3:], w, Sg)
    for a, b in zip(got, want):
        assert torch.equal(a[-3:], b)
    assert torch.equal(got[0][1], got[0][rows - 4]) and torch.equal(got[1][1], got[1][rows - 4])
    out = add_rms_norm_backward(m, S, got[2], got[4], w, Sg)
    tail = add_rms_norm_backward(m[-3:], S[-3:], got[2][-3:], got[4][-3:], w, Sg)
    assert torch.equal(out[0][-3:], tail[0]) and torch.equal(out[1][-3:], tail[1])


def test_lookup_of_more_tokens_than_one_grid(dev):
    """2^23 + 9 tokens of rows that take a block each."""
    from triton_tagi_amd.kernels import embedding_lookup

    n, V, D = (1 << 23) + 9, 7, 516
    if torch.cuda.get_device_properties(dev).total_memory < 60 << 30:
        pytest.skip("needs 60 GB of GPU memory")
    r = g(5)
    mw, Sw = torch.randn(V, D, generator=r).to(dev), torch.rand(V, D, generator=r).to(dev)
    ids = (torch.arange(n, device=dev) % V).to(torch.int32)
    mz, Sz = embedding_lookup(ids, mw, Sw)
    for t in (0, (1 << 23) - 1, 1 << 23, n - 1):
        assert torch.equal(mz[t], mw[t % V]) and torch.equal(Sz[t], Sw[t % V])


def test_overlapping_tensors_are_not_updated(dev):
    from triton_tagi_amd.kernels import embedding_update, linear_attention_step

    buf = torch.zeros(40, device=dev)
    d = torch.zeros(2, 4, device=dev)
    with pytest.raises(ValueError, match="share memory"):
        embedding_update(torch.zeros(2, device=dev), d, d, buf[:20].view(5, 4), buf[16:36].view(5, 4), 2.0)
    q = torch.zeros(1, 1, 4, device=dev)
    with pytest.raises(ValueError, match="share memory"):
        linear_attention_step(*([q] * 6), (buf[:16].view(1, 1, 4, 4), buf[12:28].view(1, 1, 4, 4)),
                              torch.ones(1, device=dev))


def test_float_ids_at_the_end_of_the_exact_range(dev):
    """2^24 is the last float every id below which is exact: it is a row of a table of 2^24 + 1."""
    from triton_tagi_amd.kernels import embedding_lookup

    V = (1 << 24) + 1
    mw = torch.arange(V, device=dev, dtype=torch.float32)[:, None].contiguous()
    ids = torch.tensor([float(1 << 24), float((1 << 24) - 1), float((1 << 24) + 2)], device=dev)
    mz, _ = embedding_lookup(ids, mw, torch.ones_like(mw))
    assert mz[:, 0].tolist() == [float(1 << 24), float((1 << 24) - 1), 0.0]


def test_calls_from_two_threads(dev):
    """Calls at the same time on streams of their own give each its own answers."""
    import threading

    from triton_tagi_amd.kernels import embedding_param_deltas, linear_attention

    r = g(4)
    jobs = []
    for s in range(2):
        x = [t.to(dev) for t in lin_inputs(1, 400, 2, 40, s)]
        ids, dm = torch.randint(0, 60, (9000,), generator=r).to(dev), torch.randn(9000, 36, generator=r).to(dev)
        Sw = torch.rand(60, 36, generator=r).to(dev)
        dec = decays(2).to(dev)

        def work(x=x, dec=dec, ids=ids, dm=dm, Sw=Sw):
            return (*linear_attention(*x, dec), *embedding_param_deltas(ids, dm, dm, Sw))

        jobs.append((work, [t.clone() for t in work()], [], []))
    torch.cuda.synchronize()

    def thread(work, want, got, failed):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[:] = work()
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001  (reported by the test's own thread)
            failed.append(e)

    threads = [threading.Thread(target=thread, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for _, want, got, failed in jobs:
        assert not failed
        for a, b in zip(got, want):
            assert torch.equal(a, b)


# =============================================================================== refusals
def test_refusals(dev):
    from triton_tagi_amd import kernels as K

    z = lambda *s, **k: torch.zeros(*s, device=dev, **k)  # noqa: E731
    ids, tab = z(5, dtype=torch.int64), z(4, 3)
    for bad, err in (((z(5, dtype=torch.float16), tab, tab), TypeError), (([1, 2], tab, tab), TypeError),
                     ((ids.cpu(), tab, tab), ValueError), ((ids, tab.double(), tab), TypeError),
                     ((ids, tab, z(4, 4)), ValueError), ((ids, z(3), z(3)), ValueError), ((ids, z(0, 3), z(0, 3)), ValueError)):
        with pytest.raises(err):
            K.embedding_lookup(*bad)
    with pytest.raises(ValueError):
        K.embedding_lookup(ids, tab, tab, scale=math.inf)
    with pytest.raises(ValueError, match="delta_mz"):
        K.embedding_param_deltas(ids, z(5, 4), z(5, 3), tab)
    with pytest.raises(ValueError, match="delta_Sz"):
        K.embedding_param_deltas(ids, z(5, 3), z(4, 3), tab)
    with pytest.raises(ValueError, match="contiguous"):
        K.embedding_update(ids, z(5, 3), z(5, 3), z(3, 4).t(), z(4, 3), 2.0)
    with pytest.raises(ValueError, match="share"):
        K.embedding_update(ids, z(5, 3), z(5, 3), tab, tab, 2.0)
    for cap in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="cap_factor"):
            K.embedding_update(ids, z(5, 3), z(5, 3), tab, z(4, 3), cap)
    x, w = z(2, 6), z(6)
    with pytest.raises(ValueError):
        K.add_rms_norm(x, x, z(2, 5), x, w, w)
    with pytest.raises(ValueError):
        K.add_rms_norm(x, x, x, x, z(5), w)
    with pytest.raises(TypeError):
        K.add_rms_norm(x, x.half(), x, x, w, w)
    with pytest.raises(ValueError, match="together"):
        K.add_rms_norm_backward(x, x, x, z(2, 1), w, w, x)
    with pytest.raises(ValueError, match="inv_rms"):
        K.add_rms_norm_backward(x, x, x, z(3, 1), w, w)
    q, dec = z(1, 4, 2, 8), z(2)
    with pytest.raises(ValueError):
        K.linear_attention(q, q, q, q, z(1, 4, 2, 7), q, dec)
    with pytest.raises(ValueError):
        K.linear_attention(q, q, q, q, q, q, z(3))
    with pytest.raises(ValueError):
        K.linear_attention(q[0], *([q[0]] * 5), dec)
    with pytest.raises(TypeError, match="lengths"):
        K.linear_attention(q, q, q, q, q, q, dec, lengths=z(1))
    with pytest.raises(ValueError, match="lengths"):
        K.linear_attention(q, q, q, q, q, q, dec, lengths=z(2, dtype=torch.int32))
    with pytest.raises(TypeError, match="state"):
        K.linear_attention(q, q, q, q, q, q, dec, state=3)
    with pytest.raises(ValueError, match="state"):
        K.linear_attention(q, q, q, q, q, q, dec, state=(z(1, 2, 8, 8), z(1, 2, 8, 4)))
    big = z(1, 1, 1, 129)
    with pytest.raises(RuntimeError, match="head dimension"):
        K.linear_attention(big, *([big] * 5), z(1))
    s, st = z(1, 2, 8), (z(1, 2, 8, 8), z(1, 2, 8, 8))
    with pytest.raises(ValueError, match="contiguous"):
        K.linear_attention_step(s, s, s, s, s, s, (st[0].transpose(2, 3), st[1]), dec)
    with pytest.raises(ValueError, match="share"):
        K.linear_attention_step(s, s, s, s, s, s, (st[0], st[0]), dec)
    with pytest.raises(TypeError, match="active"):
        K.linear_attention_step(s, s, s, s, s, s, st, dec, active=z(1))
    with pytest.raises(ValueError, match="active"):
        K.linear_attention_step(s, s, s, s, s, s, st, dec, active=z(2, dtype=torch.bool))
