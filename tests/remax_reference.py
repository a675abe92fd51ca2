"""Remax attention in float64 and how far a float32 evaluation may be off, to first order.

Roundings are 2^-24 of a value (U). A score's mean is a sum of D products, off by (D + 4) U of the
sum of their magnitudes; its variance a sum of 2 D positive terms, (2 D + 8) U of itself. From there
the bounds follow the formulas: with z ~ N(m, v), mean and var the moments of max(z, 0),

    d mean = Phi dm + phi / (2 sd) dv,   d var = 2 mean (1 - Phi) dm + Phi dv

plus 2e-6 of the mean and of Phi and 1e-5 of the variance for the tail's polynomials and the
subtraction in them (kernels' figures: 4e-7 for R, 7e-7 for 1 - x R, x^2 / 2 of R's for the variance
up to x = 5.5; beyond, the floor of 1e-6 holds the variance for the scales used here). Weights,
their variances and the Jacobian are rational in these; a row's sums over n keys are off by n / 4 U
at most (a lane adds every fourth key) plus their terms' errors. Every bound is doubled for the
second order.
"""

from __future__ import annotations

import math

import torch

U = 2.0**-24
EPS = 1e-6


def d64(t):
    return t.detach().to("cpu", torch.float64)


def rect(m, v):
    """mean, var, cdf, pdf of max(z, 0), without cancellation."""
    sd = v.sqrt()
    a = m / sd
    x = a.abs()
    pdf = torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)
    R = torch.special.erfcx(x / math.sqrt(2.0)) * math.sqrt(math.pi / 2)
    u = torch.where(x < 1e4, 1 - x * R, 0.0)
    f, q = pdf * u, pdf * torch.where(x < 1e4, R - x * u, 0.0)
    up = a >= 0
    mean = sd * f + m.clamp_min(0)
    var = v * torch.where(up, 1 - q - 2 * torch.where(pdf > 0, x * f, 0.0) - f * f, q - f * f)
    return mean, var, torch.where(up, 1 - pdf * R, pdf * R), pdf


class Row:
    """One head's attention: queries (T, D), keys (N, D), seen (T, N)."""

    def __init__(self, mq, Sq, mk, Sk, mv, Sv, seen, c):
        D, n = mq.shape[1], mk.shape[0]
        self.c, self.seen = c, seen.double()
        self.q, self.k, self.vm, self.vS = (mq, Sq), (mk, Sk), mv, Sv
        m = c * (mq @ mk.T)
        v = (c * c * (Sq @ (mk * mk + Sk).T + (mq * mq) @ Sk.T)).clamp_min(1e-20)
        dm = (D + 4) * U * abs(c) * (mq.abs() @ mk.abs().T)
        dv = (2 * D + 8) * U * v
        mean, var, cdf, pdf = rect(m, v)
        sd = v.sqrt()
        live = mean > EPS
        mm = mean.clamp_min(EPS)
        vraw = var + (mean - mm) * (mean + mm - 2 * m)
        vm = vraw.clamp_min(EPS)
        e_mm = torch.where(live, (cdf * dm + pdf / (2 * sd) * dv) / mm + 2e-6, 0.0)
        # where the floor lifts the mean: vraw = var + mean^2 - EPS^2 - 2 m (mean - EPS)
        d_v = (2 * mean * (1 - cdf) * dm + cdf * dv) + 1e-5 * var + 4 * U * v
        lift = torch.where(live, 0.0, 2 * EPS * dm + 2 * (m.abs() + EPS) * (cdf * dm + pdf / (2 * sd) * dv + 4 * U * EPS))
        e_vm = torch.where(vraw + d_v + lift > EPS, (d_v + lift) / vm, 0.0)
        e_cdf = (pdf / sd * (dm + m.abs() / (2 * v) * dv)) / cdf.clamp_min(EPS) + 2e-6
        s = self.seen
        mt, vt = ((x * s).sum(1, keepdim=True).clamp_min(EPS) for x in (mm, vm))
        e_mt = (mm * s * e_mm).sum(1, keepdim=True) / mt + (n / 4 + 8) * U
        e_vt = (vm * s * e_vm).sum(1, keepdim=True) / vt + (n / 4 + 8) * U
        y, x, w = vt / mt**2, vm / mm**2, vm / (mm * mt)
        e_y, e_x, e_w = e_vt + 2 * e_mt + 4 * U, e_vm + 2 * e_mm + 4 * U, e_vm + e_mm + e_mt + 4 * U
        raw = ((mm / mt) * (1 + y) / (1 + w)).clamp_min(EPS) * s
        e_raw = e_mm + e_mt + e_y * y / (1 + y) + e_w * w / (1 + w) + 8 * U
        total = raw.sum(1, keepdim=True).clamp_min(EPS)
        e_total = (raw * e_raw).sum(1, keepdim=True) / total + (n / 4 + 8) * U
        self.a = raw / total
        self.e_a = e_raw + e_total + 4 * U
        num = (x - w + y - w + x * y - w * w).clamp_min(0)
        self.k2 = num / (1 + w) ** 2
        d_num = x * e_x + 2 * w * e_w + y * e_y + x * y * (e_x + e_y) + 2 * w * w * e_w + 6 * U * (x + w + y + x * y + w * w)
        self.d_k2 = d_num / (1 + w) ** 2 + self.k2 * (2 * e_w + 4 * U)
        self.Sa = self.k2 * self.a**2
        self.d_Sa = self.d_k2 * self.a**2 + 2 * self.Sa * self.e_a
        cs, d_cs = (self.Sa * v).sqrt(), (self.d_Sa * v).sqrt()
        d_cs = torch.where(self.d_Sa < self.Sa, cs * self.d_Sa / self.Sa.clamp_min(1e-300), 2 * d_cs) + cs * 8 * U
        cov = (x - w).clamp_min(0) / (1 + w) * self.a * mm / cdf.clamp_min(EPS)
        d_cov = ((x * e_x + w * e_w + 2 * U * (x + w)) / (1 + w) * self.a * mm / cdf.clamp_min(EPS)
                 + cov * (e_w + self.e_a + e_mm + e_cdf + 8 * U))
        J = torch.minimum(cs, cov) / v * s
        self.J, self.d_J = J, (torch.maximum(d_cs, d_cov) / v + J * (dv / v + 4 * U)) * s

    def outputs(self):
        """(mo, So) and their bounds."""
        n = self.a.shape[1]
        r = (n / 4 + 8) * U
        mv, Sv, a, Sa = self.vm, self.vS, self.a, self.Sa
        mo, So = a @ mv, Sa @ (mv * mv + Sv) + (a * a) @ Sv
        b_mo = (a * (self.e_a + r)) @ mv.abs()
        b_So = (self.d_Sa + 2 * r * Sa) @ (mv * mv + Sv) + (a * a * (2 * self.e_a + 2 * r)) @ Sv
        return (mo, 2 * b_mo + 1e-30), (So, 2 * b_So + 1e-30)

    def deltas(self, dm, dS):
        """Six deltas and their bounds (keys' and values' of this head alone)."""
        c, (mq, _), (mk, _), mv = self.c, self.q, self.k, self.vm
        T, D = mq.shape
        n = mk.shape[0]
        x, X = dm @ mv.T, dS @ (mv * mv).T
        ax, aX = dm.abs() @ mv.abs().T, dS.abs() @ (mv * mv).T
        r = (D + 4) * U
        e, E = c * self.J * x, c * c * self.J**2 * X
        d_e = abs(c) * (self.d_J * x.abs() + self.J * ax * (r + 4 * U))
        d_E = c * c * (2 * self.J * self.d_J * X.abs() + self.d_J**2 * X.abs() + self.J**2 * aX * (r + 8 * U))
        out = []
        for p, d_p, w in ((e, d_e, mk), (E, d_E, mk * mk)):
            out.append((p @ w, 2 * ((d_p + (n / 4 + 8) * U * p.abs()) @ w.abs()) + 1e-30))
        for p, d_p, w in ((e, d_e, mq), (E, d_E, mq * mq), (self.a, self.a * self.e_a, dm),
                          (self.a**2, 2 * self.a**2 * self.e_a, dS)):
            out.append((p.T @ w, 2 * ((d_p + (T / 4 + 16) * U * p.abs()).T @ w.abs()) + 1e-30))
        return out


def seen_mask(T, N, causal, length, start):
    at = start + torch.arange(T)
    key = torch.arange(N)
    on = (at >= 0) & (at < length)
    seen = on[:, None] & (key < length)[None]
    return seen & (key[None] <= at[:, None]) if causal else seen


def attention(mq, Sq, mk, Sk, mv, Sv, c, causal=True, lengths=None, starts=None, deltas=None):
    """[(value, bound)] of (mo, So) and, with deltas (dm, dS), of the six deltas; float64 on the CPU."""
    t = [d64(x) for x in (mq, Sq, mk, Sk, mv, Sv)]
    B, T, H, D = t[0].shape
    N, G = t[2].shape[1:3]
    shapes = [(B, T, H, D)] * 2 + ([(B, T, H, D)] * 2 + [(B, N, G, D)] * 4 if deltas else [])
    out = [(torch.zeros(s, dtype=torch.float64), torch.zeros(s, dtype=torch.float64)) for s in shapes]
    R = H // G
    for b in range(B):
        length = N if lengths is None else min(max(int(lengths[b]), 0), N)
        start = 0 if starts is None else int(starts[b])
        seen = seen_mask(T, N, causal, length, start)
        rows = seen.any(1) if N else torch.zeros(T, dtype=torch.bool)
        if not rows.any():
            continue
        for h in range(H):
            g = h // R
            # what nothing sees is not read
            q = [x[b, rows, h] for x in t[:2]]
            k = [x[b, :length, g] for x in t[2:]]
            row = Row(*q, *k, seen[rows][:, :length], c)
            res = row.outputs()
            for i in range(2):
                for j in range(2):
                    out[i][j][b, rows, h] = res[i][j]
            if deltas:
                res = row.deltas(*(d64(x)[b, rows, h] for x in deltas))
                for i in range(2):
                    for j in range(2):
                        out[2 + i][j][b, rows, h] = res[i][j]
                for i in range(4):
                    for j in range(2):
                        out[4 + i][j][b, :length, g] += res[2 + i][j]
    return out


def within(got, ref, what):
    got = d64(got)
    value, bound = ref
    assert got.shape == value.shape, f"{what}: {tuple(got.shape)} vs {tuple(value.shape)}"
    if not got.numel():
        return
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - value).abs() - bound
    i = int(over.reshape(-1).argmax())
    assert over.reshape(-1)[i] <= 0, (
        f"{what}: got {got.reshape(-1)[i].item():.9g} ref {value.reshape(-1)[i].item():.9g}, bound "
        f"{bound.reshape(-1)[i].item():.3g}, over by {over.reshape(-1)[i].item():.3g} at {i}")
