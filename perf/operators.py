"""Performance cases of the sequence-model operators: token embedding, residual RMSNorm, decayed linear attention.

Each case is one pass through one operator of ``triton_tagi_amd.kernels`` on GPU tensors:

    lookup   embedding_lookup: moments of the token rows, scaled
    deltas   embedding_param_deltas: the parameter deltas of every row of the table
    update   embedding_update: the same sums applied to the rows that occur, in place
    norm     add_rms_norm: sum of two Gaussian streams and its RMSNorm
    normtr   add_rms_norm and add_rms_norm_backward
    attn     linear_attention over whole sequences: prompts, ragged batches, a state carried on
    attntr   linear_attention and linear_attention_backward
    step     linear_attention_step: one token of every sequence, the state advanced in place

``own`` false computes the same in elementary torch operations; ``exact`` from the definitions
in float64, token by token where the operator is a recurrence.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import numpy as np
import torch

_PKG = str(Path(__file__).resolve().parents[1] / "triton-tagi_amd")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

own = False

DEV = "cuda"
EPS = 1e-6
CAP = 3.0  # cap factor of batches of 256 and more
CHUNK = 32  # tokens per block of the plain form's two-level prefix sums


# ------------------------------------------------------------------------------ cases
def listed():
    return [
        # serving: the next token of 32 sequences in the transformer workload's embedding, latency
        {"name": "lookup_small", "kind": "lookup", "N": 32, "V": 64, "D": 256, "ids": "float32", "zipf": False, "pad": -1},
        # training, the transformer workload's table: 64 sequences of 256 tokens, few categories
        {"name": "deltas_workload", "kind": "deltas", "N": 16384, "V": 64, "D": 256, "ids": "float32", "zipf": False,
         "pad": -1},
        # training a language model's table, odd sizes, frequencies by Zipf's law, padding tokens
        {"name": "deltas_zipf_odd", "kind": "deltas", "N": 20001, "V": 50021, "D": 390, "ids": "int64", "zipf": True,
         "pad": 0},
        # a large table updated in place by a large batch: most rows do not occur
        {"name": "update_zipf", "kind": "update", "N": 65536, "V": 131071, "D": 1024, "ids": "int64", "zipf": True,
         "pad": -1},
        # serving: the residual norm of a few tokens, latency
        {"name": "norm_few", "kind": "norm", "N": 8, "D": 4096},
        # training, odd sizes on both axes
        {"name": "normtr_odd", "kind": "normtr", "N": 4099, "D": 771},
        # training, a large batch of wide rows
        {"name": "normtr_large", "kind": "normtr", "N": 16384, "D": 4096},
        # training, the transformer workload's attention sizes
        {"name": "attntr_workload", "kind": "attntr", "B": 64, "T": 256, "H": 8, "D": 32, "ragged": False},
        # training on long sequences
        {"name": "attntr_long", "kind": "attntr", "B": 2, "T": 4096, "H": 16, "D": 64, "ragged": False},
        # prompts of different lengths (an empty one among them) continued from a state; odd sizes
        {"name": "attn_ragged", "kind": "attn", "B": 7, "T": 777, "H": 6, "D": 80, "ragged": True, "state": True},
        # one long prompt: the time axis is all the parallelism there is
        {"name": "attn_prompt", "kind": "attn", "B": 1, "T": 32768, "H": 8, "D": 64, "ragged": False, "state": False},
        # serving: the next token of 32 sequences, bound by the states
        {"name": "step_batch", "kind": "step", "B": 32, "H": 16, "D": 128},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["lookup", "deltas", "update", "norm", "normtr", "attn", "attn", "attntr", "attntr", "step"])
    if kind in ("lookup", "deltas", "update"):
        N, V, D = _log(rng, 1, 65536), _log(rng, 32, 131071), _log(rng, 8, 1024)
        return {"kind": kind, "N": N, "V": V, "D": D, "ids": rng.choice(["float32", "int32", "int64"]),
                "zipf": rng.random() < 0.6, "pad": rng.choice([-1, 0])}
    if kind == "norm":
        return {"kind": kind, "N": _log(rng, 1, 512), "D": _log(rng, 16, 8192)}
    if kind == "normtr":
        D = _log(rng, 16, 8192)
        return {"kind": kind, "N": _log(rng, 1, min(16384, (1 << 26) // D)), "D": D}
    H, D = rng.randint(1, 16), rng.choice([rng.randint(8, 128), 16, 32, 64, 128])
    if kind == "step":
        return {"kind": kind, "B": _log(rng, 1, max(1, min(256, (1 << 23) // (H * D * D)))), "H": H, "D": D}
    room = (1 << 29) // (H * D * D)
    T = _log(rng, 1, min(32768 if kind == "attn" else 4096, room))
    case = {"kind": kind, "B": _log(rng, 1, max(1, min(64, room // T))), "T": T, "H": H, "D": D,
            "ragged": rng.random() < 0.4}
    if kind == "attn":
        case["state"] = rng.random() < 0.5
    return case


# ------------------------------------------------------------------------------ inputs
def _ids(case, gen):
    V, N = case["V"], case["N"]
    u = torch.rand(N, generator=gen, device=DEV, dtype=torch.float64)
    if not case["zipf"]:
        at = (u * V).long()
    else:  # rank r with probability log(1 + 1/r) / log(V + 1); the ranks in a shuffled order
        at = torch.exp(u * math.log(V + 1)).long() - 1
        at = torch.randperm(V, generator=gen, device=DEV)[at.clamp(0, V - 1)]
    return at.clamp(0, V - 1).to(getattr(torch, case["ids"]))


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=gen, device=DEV).mul_(std)

    def spread(*shape, lo, hi):
        return torch.rand(shape, generator=gen, device=DEV).mul_(hi - lo).add_(lo)

    kind, D = case["kind"], case["D"]
    s = {"case": case}
    if kind in ("lookup", "deltas", "update"):
        N, V = case["N"], case["V"]
        s["ids"], s["scale"], s["pad"] = _ids(case, gen), math.sqrt(D), case["pad"]
        s["mw"], s["Sw"] = normal(V, D, std=0.25), spread(V, D, lo=0.01, hi=0.07)
        if kind != "lookup":
            s["dm"], s["dS"] = normal(N, D, std=0.02), spread(N, D, lo=-1e-3, hi=-1e-5)
    elif kind in ("norm", "normtr"):
        N = case["N"]
        s["ma"], s["mr"] = normal(N, D), normal(N, D, std=2.0)
        s["Sa"], s["Sr"] = spread(N, D, lo=0.01, hi=0.1), spread(N, D, lo=0.02, hi=0.5)
        s["mw"], s["Sw"] = normal(D, std=0.1).add_(1.0), spread(D, lo=0.005, hi=0.02)
        if kind == "normtr":
            s["dm"], s["dms"] = normal(N, D, std=0.1), normal(N, D, std=0.1)
            s["dS"], s["dSs"] = spread(N, D, lo=-0.02, hi=-1e-4), spread(N, D, lo=-0.02, hi=-1e-4)
    else:
        B, H = case["B"], case["H"]
        lead = (B, H, D) if kind == "step" else (B, case["T"], H, D)
        for x, std in (("q", 1.0), ("k", 0.5), ("v", 1.0)):
            s["m" + x], s["S" + x] = normal(*lead, std=std), spread(*lead, lo=0.005, hi=0.1)
        # heads forget at different rates, from about 16 tokens to about 256
        s["decay"] = 1.0 - torch.exp2(-4.0 - 4.0 * torch.arange(H, device=DEV, dtype=torch.float32) / max(1, H - 1))
        s["scale"] = 1.0 / math.sqrt(D)
        s["lengths"] = s["state"] = None
        if case.get("ragged"):
            n = torch.randint(1, case["T"] + 1, (B,), generator=gen, device=DEV, dtype=torch.int32)
            n[0] = 0 if B > 1 else n[0]
            s["lengths"] = n
        if kind == "step" or case.get("state"):
            s["state"] = (normal(B, H, D, D), spread(B, H, D, D, lo=0.05, hi=0.5))
        if kind == "attntr":
            s["dm"], s["dS"] = normal(*lead, std=0.1), spread(*lead, lo=-0.02, hi=-1e-4)
    return s


# ------------------------------------------------------------------- the framework's calls
def _own(s):
    from triton_tagi_amd import kernels as K

    kind = s["case"]["kind"]
    if kind == "lookup":
        return K.embedding_lookup(s["ids"], s["mw"], s["Sw"], scale=s["scale"], padding_idx=s["pad"])
    if kind == "deltas":
        return K.embedding_param_deltas(s["ids"], s["dm"], s["dS"], s["Sw"], scale=s["scale"], padding_idx=s["pad"])
    if kind == "update":
        K.embedding_update(s["ids"], s["dm"], s["dS"], s["mw"], s["Sw"], CAP, scale=s["scale"], padding_idx=s["pad"])
        return s["mw"], s["Sw"]
    if kind in ("norm", "normtr"):
        mz, Sz, ms, Ss, inv = K.add_rms_norm(s["ma"], s["Sa"], s["mr"], s["Sr"], s["mw"], s["Sw"], EPS)
        if kind == "norm":
            return mz, Sz, ms, Ss
        return (mz, Sz, ms, Ss, *K.add_rms_norm_backward(s["dm"], s["dS"], ms, inv, s["mw"], s["Sw"], s["dms"],
                                                          s["dSs"]))
    qkv = [s[n] for n in ("mq", "Sq", "mk", "Sk", "mv", "Sv")]
    if kind == "step":
        mo, So = K.linear_attention_step(*qkv, s["state"], s["decay"], scale=s["scale"])
        return mo, So, s["state"][0], s["state"][1]
    if kind == "attn":
        mo, So, (M, P) = K.linear_attention(*qkv, s["decay"], scale=s["scale"], lengths=s["lengths"],
                                            state=s["state"], return_state=True)
        return mo, So, M, P
    mo, So = K.linear_attention(*qkv, s["decay"], scale=s["scale"], lengths=s["lengths"])
    return (mo, So, *K.linear_attention_backward(s["mq"], s["mk"], s["mv"], s["dm"], s["dS"], s["decay"],
                                                 scale=s["scale"], lengths=s["lengths"]))


# --------------------------------------------------------------------------- plain forms
def _plain_embedding(s):
    kind, c, D = s["case"]["kind"], s["scale"], s["case"]["D"]
    ids = s["ids"].long()
    real = (ids != s["pad"])[:, None]
    if kind == "lookup":
        return torch.where(real, s["mw"][ids] * c, 0.0), torch.where(real, s["Sw"][ids] * (c * c), 0.0)
    # long sums over the tokens of frequent categories: in 64 bits
    gm = torch.zeros(s["Sw"].shape, device=DEV, dtype=torch.float64)
    gS = torch.zeros_like(gm)
    gm.index_add_(0, ids, torch.where(real, s["dm"], 0.0).double())
    gS.index_add_(0, ids, torch.where(real, s["dS"], 0.0).double())
    dmw = (gm * c).float() * s["Sw"]
    dSw = (gS * (c * c)).float() * (s["Sw"] * s["Sw"])
    if kind == "deltas":
        return dmw, dSw
    bar = torch.sqrt(s["Sw"].clamp_min(1e-10)) / CAP
    s["mw"] += torch.sign(dmw) * torch.minimum(dmw.abs(), bar)
    new = s["Sw"] + torch.sign(dSw) * torch.minimum(dSw.abs(), bar)
    s["Sw"].copy_(torch.where(new <= 0.0, 1e-5, new))
    return s["mw"], s["Sw"]


def _plain_norm(s):
    ms, Ss = s["ma"] + s["mr"], s["Sa"] + s["Sr"]
    inv = torch.rsqrt((ms * ms + Ss).mean(-1, keepdim=True) + EPS)
    g, Sg = s["mw"], s["Sw"]
    mz, Sz = ms * inv * g, inv * inv * (Ss * (g * g + Sg) + Sg * (ms * ms))
    if s["case"]["kind"] == "norm":
        return mz, Sz, ms, Ss
    dm, dS, w = s["dm"], s["dS"], inv * g
    return (mz, Sz, ms, Ss, dm * w + s["dms"], dS * (w * w) + s["dSs"], Sg * (dm * (ms * inv)).sum(0),
            Sg * Sg * (dS * (ms * inv) ** 2).sum(0))


def _powers(decay, e):
    return decay.double()[:, None] ** e.double()  # (H, len(e)): high powers in 64 bits


def _scan(x, decay, init=None):
    """y_t = decay y_{t-1} + x_t along the second axis of x (B, H, T, X), y_{-1} = init: inside
    blocks of CHUNK tokens by a triangular matrix of powers, across blocks by another."""
    B, H, T, X = x.shape
    n = -(-T // CHUNK)
    if n * CHUNK != T:
        x = torch.cat([x, x.new_zeros(B, H, n * CHUNK - T, X)], 2)
    i = torch.arange(CHUNK, device=DEV)
    inside = torch.where(i[:, None] >= i, _powers(decay, (i[:, None] - i).clamp_min(0).reshape(-1)).view(H, CHUNK, CHUNK),
                         0.0).float()
    y = torch.matmul(inside[None, :, None], x.view(B, H, n, CHUNK, X))
    b = torch.arange(n, device=DEV)
    across = torch.where(b[:, None] > b, _powers(decay, ((b[:, None] - b - 1).clamp_min(0) * CHUNK).reshape(-1))
                         .view(H, n, n), 0.0).float()
    before = torch.matmul(across[None], y[:, :, :, -1])
    if init is not None:
        before += _powers(decay, b * CHUNK).float()[None, :, :, None] * init[:, :, None]
    y += _powers(decay, i + 1).float()[None, :, None, :, None] * before[:, :, :, None]
    return y.view(B, H, n * CHUNK, X)[:, :, :T]


def _plain_attention(s):
    case, scale, decay = s["case"], s["scale"], s["decay"]
    B, T, H, D = case["B"], case["T"], case["H"], case["D"]
    live = None
    if s["lengths"] is not None:
        live = (torch.arange(T, device=DEV) < s["lengths"][:, None]).view(B, 1, T, 1)

    def heads(x):  # (B, T, H, D) -> (B, H, T, D); zeros past a sequence's end, so its outputs there are zeros
        x = x.transpose(1, 2)
        return x if live is None else torch.where(live, x, 0.0)

    def outer(a, b):
        return (a.unsqueeze(-1) * b.unsqueeze(-2)).flatten(-2)

    mq, Sq, mk, Sk, mv, Sv = (heads(s[n]) for n in ("mq", "Sq", "mk", "Sk", "mv", "Sv"))
    M0, P0 = (None, None) if s["state"] is None else (x.flatten(-2) for x in s["state"])
    M = _scan(outer(mk, mv), decay, M0)
    P = _scan(outer(Sk, mv * mv + Sv) + outer(mk * mk, Sv), decay.double() ** 2, P0)
    if case["kind"] == "attn":
        last = torch.full((B,), T, device=DEV) if s["lengths"] is None else s["lengths"].long()
        at = (last - 1).clamp_min(0)
        rows = torch.arange(B, device=DEV)
        ends = []
        for y, y0 in ((M, M0), (P, P0)):
            end = y[rows, :, at]
            ends.append(torch.where((last > 0)[:, None, None], end, 0.0 if y0 is None else y0).view(B, H, D, D))
    M, P = M.view(B, H, T, D, D), P.view(B, H, T, D, D)
    mo = scale * (mq.unsqueeze(-1) * M).sum(-2)
    So = (scale * scale) * ((Sq + mq * mq).unsqueeze(-1) * P + Sq.unsqueeze(-1) * (M * M)).sum(-2)
    out = [mo.transpose(1, 2), So.transpose(1, 2)]
    if case["kind"] == "attn":
        return (*out, *ends)
    del P
    dm, dS = heads(s["dm"]) * scale, heads(s["dS"]) * (scale * scale)
    out += [(M * dm.unsqueeze(-2)).sum(-1).transpose(1, 2), (M * M * dS.unsqueeze(-2)).sum(-1).transpose(1, 2)]
    del M
    G = _scan(outer(mq, dm).flip(2), decay).flip(2).view(B, H, T, D, D)
    GS = _scan(outer(mq * mq, dS).flip(2), decay.double() ** 2).flip(2).view(B, H, T, D, D)
    dk = [(G * mv.unsqueeze(-2)).sum(-1), (GS * (mv * mv).unsqueeze(-2)).sum(-1)]
    dv = [(G * mk.unsqueeze(-1)).sum(-2), (GS * (mk * mk).unsqueeze(-1)).sum(-2)]
    out += [x.transpose(1, 2) for x in dk + dv]
    return tuple(out)


def _plain_step(s):
    M, P = s["state"]
    g, scale = s["decay"][None, :, None, None], s["scale"]
    col, row = (lambda x: x.unsqueeze(-1)), (lambda x: x.unsqueeze(-2))
    mq, Sq, mk, Sk, mv, Sv = (s[n] for n in ("mq", "Sq", "mk", "Sk", "mv", "Sv"))
    M.copy_(g * M + col(mk) * row(mv))
    P.copy_(g * g * P + (col(Sk) * row(mv * mv + Sv) + col(mk * mk) * row(Sv)))
    mo = scale * (col(mq) * M).sum(-2)
    So = (scale * scale) * (col(Sq + mq * mq) * P + col(Sq) * (M * M)).sum(-2)
    return mo, So, M, P


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    if kind in ("lookup", "deltas", "update"):
        return _plain_embedding(state)
    if kind in ("norm", "normtr"):
        return _plain_norm(state)
    return _plain_step(state) if kind == "step" else _plain_attention(state)


# ------------------------------------------------------------------------------- work
def _distinct(case):
    """Rows of the table that N tokens are expected to meet."""
    V, N = case["V"], case["N"]
    r = np.arange(1, V + 1, dtype=np.float64)
    p = np.log1p(1.0 / r) / math.log(V + 1) if case["zipf"] else np.full(V, 1.0 / V)
    return float((-np.expm1(N * np.log1p(-np.minimum(p, 1 - 1e-12)))).sum())


def work(case):
    kind, D = case["kind"], case["D"]
    if kind in ("lookup", "deltas", "update"):
        N, V, rows = case["N"], case["V"], _distinct(case)
        ids = N * (8 if case["ids"] == "int64" else 4)
        if kind == "lookup":
            return {"bytes": ids + 8 * D * (rows + N), "flops": 2 * N * D}
        if kind == "deltas":
            return {"bytes": ids + 8 * N * D + 4 * rows * D + 8 * V * D, "flops": 2 * N * D + 4 * rows * D}
        return {"bytes": ids + 8 * N * D + 16 * rows * D, "flops": 2 * N * D + 14 * rows * D}
    if kind in ("norm", "normtr"):
        n = case["N"] * D
        if kind == "norm":
            return {"bytes": 32 * n + 8 * D, "flops": 14 * n}
        # forward: 4 read, 4 written; backward: 4 deltas and the mean read, 2 written
        return {"bytes": 60 * n + 24 * D, "flops": 28 * n}
    if kind == "step":
        e = case["B"] * case["H"] * D
        return {"bytes": 16 * e * D + 32 * e, "flops": 15 * e * D}
    e = case["B"] * case["T"] * case["H"] * D
    ends = 8 * case["B"] * case["H"] * D * D
    # state element and token: 3 + 5 to advance the two moments, 2 + 2 + 3 for the outputs
    if kind == "attn":
        return {"bytes": 32 * e + ends * (2 if case["state"] else 1), "flops": 15 * e * D}
    # backward: the mean state again (3) with its two products (5), the adjoint states (6) with theirs (8)
    return {"bytes": 32 * e + 44 * e, "flops": 37 * e * D}


# ---------------------------------------------------------------------- values in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    s = {n: x.double() if isinstance(x, torch.Tensor) and n not in ("ids", "lengths") else x for n, x in s.items()}
    kind = case["kind"]
    if kind in ("lookup", "deltas", "update"):
        return _exact_embedding(s, kind)
    if kind in ("norm", "normtr"):
        return _exact_norm(s, kind)
    return _exact_attention(s, kind)


def _exact_embedding(s, kind):
    c, ids = s["scale"], s["ids"].long()
    keep = ids != s["pad"]
    if kind == "lookup":
        mz, Sz = c * s["mw"].index_select(0, ids), c * c * s["Sw"].index_select(0, ids)
        mz[~keep], Sz[~keep] = 0.0, 0.0
        return mz, Sz
    S = s["Sw"]
    dmw = torch.zeros_like(S).index_add_(0, ids[keep], c * s["dm"][keep] * S[ids[keep]])
    dSw = torch.zeros_like(S).index_add_(0, ids[keep], c * c * s["dS"][keep] * S[ids[keep]].square())
    if kind == "deltas":
        return dmw, dSw
    bar = S.clamp(min=1e-10).sqrt() / CAP
    m, S = s["mw"] + dmw.clamp(-bar, bar), S + dSw.clamp(-bar, bar)
    S[S <= 0] = 1e-5
    return m, S


def _exact_norm(s, kind):
    m, S = s["ma"] + s["mr"], s["Sa"] + s["Sr"]
    r = (m.square().sum(1, keepdim=True) + S.sum(1, keepdim=True)).div(m.shape[1]).add(EPS).sqrt()
    n = m / r
    mz, Sz = n * s["mw"], (S / r**2) * (s["mw"].square() + s["Sw"]) + n.square() * s["Sw"]
    if kind == "norm":
        return mz, Sz, m, S
    return (mz, Sz, m, S, s["dm"] * s["mw"] / r + s["dms"], s["dS"] * (s["mw"] / r).square() + s["dSs"],
            s["Sw"] * (n * s["dm"]).sum(0), s["Sw"].square() * (n.square() * s["dS"]).sum(0))


def _exact_attention(s, kind):
    one = kind == "step"
    seq = {n: (s[n][:, None] if one else s[n]) for n in ("mq", "Sq", "mk", "Sk", "mv", "Sv")}
    B, T, H, D = seq["mq"].shape
    g, c = s["decay"][None, :, None, None], s["scale"]
    zero = torch.zeros(B, H, D, D, device=DEV, dtype=torch.float64)
    M, P = (zero, zero) if s["state"] is None else (x.double() for x in s["state"])
    live = None
    if s["lengths"] is not None:
        live = torch.arange(T, device=DEV)[:, None] < s["lengths"][None, :]  # (T, B)
    train = kind == "attntr"
    outs = [torch.zeros(B, T, H, D, device=DEV, dtype=torch.float64) for _ in range(8 if train else 2)]

    def put(i, t, x):
        outs[i][:, t] = x if live is None else x * live[t][:, None, None]

    for t in range(T):
        mq, Sq, mk, Sk, mv, Sv = (seq[n][:, t] for n in ("mq", "Sq", "mk", "Sk", "mv", "Sv"))
        k, Sk = mk[..., :, None], Sk[..., :, None]
        v, Sv = mv[..., None, :], Sv[..., None, :]
        M1 = g * M + k * v
        P1 = g * g * P + Sk * v * v + Sk * Sv + k * k * Sv
        if live is not None:
            on = live[t][:, None, None, None]
            M1, P1 = torch.where(on, M1, M), torch.where(on, P1, P)
        M, P = M1, P1
        q, Sq = mq[..., None, :], Sq[..., None, :]
        put(0, t, c * (q @ M)[..., 0, :])
        put(1, t, c * c * (q * q @ P + Sq @ P + Sq @ (M * M))[..., 0, :])
        if train:
            put(2, t, c * (M @ s["dm"][:, t, :, :, None])[..., 0])
            put(3, t, c * c * (M.square() @ s["dS"][:, t, :, :, None])[..., 0])
    if not train:
        return (outs[0][:, 0], outs[1][:, 0], M, P) if one else (*outs, M, P)
    G, GS = zero, zero
    for t in reversed(range(T)):
        q, k, v = seq["mq"][:, t], seq["mk"][:, t], seq["mv"][:, t]
        G1 = g * G + c * q[..., :, None] * s["dm"][:, t, :, None, :]
        GS1 = g * g * GS + c * c * q.square()[..., :, None] * s["dS"][:, t, :, None, :]
        if live is not None:
            on = live[t][:, None, None, None]
            G1, GS1 = torch.where(on, G1, G), torch.where(on, GS1, GS)
        G, GS = G1, GS1
        put(4, t, (G @ v[..., None])[..., 0])
        put(5, t, (GS @ v.square()[..., None])[..., 0])
        put(6, t, (k[..., None, :] @ G)[..., 0, :])
        put(7, t, (k.square()[..., None, :] @ GS)[..., 0, :])
    return tuple(outs)
