"""Performance cases of Remax attention over long sequences and paged caches.

Each case is one pass through operators of ``triton_tagi_amd.kernels`` on GPU tensors:

    rot      qk_norm_rotary: RMSNorm of every query and key head, then the rotation by position
    rottr    qk_norm_rotary and qk_norm_rotary_backward
    attn     remax_attention: whole sequences, ragged batches, a chunk of queries on a long context
    attntr   remax_attention and remax_attention_backward, which forms the scores again
    write    cache_write: tokens' keys and values into the pages of a cache, rounded to its type
    read     cache_read: a cache's tokens as float32
    step     remax_attention_step: one query of every sequence over its pages

``own`` false computes the same in elementary torch operations; ``exact`` from the definitions
in float64, with the Remax by its logarithms.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

_PKG = str(Path(__file__).resolve().parents[1] / "triton-tagi_amd")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

own = False

DEV = "cuda"
EPS = 1e-6  # the norm's epsilon, and the Remax's floor
THETA = 10000.0
FP8 = "float8_e4m3fn"


# ------------------------------------------------------------------------------ cases
def listed():
    return [
        # serving: the next token of 32 sequences far along, latency
        {"name": "rot_token", "kind": "rot", "B": 32, "T": 1, "H": 16, "G": 4, "D": 128, "axes": 1, "pairs": 64,
         "interleaved": False, "far": 1000000},
        # training on video-like positions (time, height, width), odd sizes, part of each head rotated
        {"name": "rottr_axes", "kind": "rottr", "B": 4, "T": 1023, "H": 6, "G": 2, "D": 80, "axes": 3, "pairs": 33,
         "interleaved": True, "far": 1000},
        # training, a large batch of wide heads
        {"name": "rottr_large", "kind": "rottr", "B": 8, "T": 2048, "H": 16, "G": 16, "D": 128, "axes": 1, "pairs": 64,
         "interleaved": False, "far": 2048},
        # training, the transformer workload's attention: every token sees every other
        {"name": "attntr_workload", "kind": "attntr", "B": 64, "T": 256, "N": 256, "H": 8, "G": 8, "D": 32,
         "causal": False, "ragged": False},
        # training on long sequences, four query heads to a key head
        {"name": "attntr_long", "kind": "attntr", "B": 2, "T": 4096, "N": 4096, "H": 16, "G": 4, "D": 64,
         "causal": True, "ragged": False},
        # prompts of different lengths, an empty one among them; odd sizes
        {"name": "attn_ragged", "kind": "attn", "B": 7, "T": 777, "N": 777, "H": 6, "G": 3, "D": 80, "causal": True,
         "ragged": True},
        # serving: a chunk of a long prompt over what its earlier chunks left
        {"name": "attn_chunk", "kind": "attn", "B": 1, "T": 512, "N": 16384, "H": 16, "G": 4, "D": 128, "causal": True,
         "ragged": False},
        # serving: the newest token of 32 sequences into the cache, latency
        {"name": "write_token", "kind": "write", "B": 32, "T": 1, "N": 1024, "G": 4, "D": 128, "page": 16, "type": FP8},
        # serving: whole prompts into the cache
        {"name": "write_prompts", "kind": "write", "B": 16, "T": 2048, "N": 4096, "G": 8, "D": 128, "page": 64,
         "type": FP8},
        # serving: what a continued prompt reads back, odd page size
        {"name": "read_context", "kind": "read", "B": 5, "N": 6001, "G": 8, "D": 128, "page": 48, "type": "bfloat16"},
        # serving: short contexts of a small model, latency
        {"name": "step_small", "kind": "step", "B": 8, "N": 256, "H": 8, "G": 8, "D": 32, "page": 16,
         "type": "float32"},
        # serving: long contexts, bound by the cache
        {"name": "step_long", "kind": "step", "B": 16, "N": 32768, "H": 32, "G": 8, "D": 128, "page": 64, "type": FP8},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rot", "rottr", "attn", "attn", "attntr", "attntr", "write", "read", "step", "step", "step"])
    D = rng.choice([rng.randint(8, 128), 32, 64, 128])
    G = rng.choice([1, 2, 3, 4, 8])
    H = G * rng.choice([1, 1, 2, 3, 4, 8])
    if kind in ("rot", "rottr"):
        axes = rng.choice([1, 1, 2, 3])
        pairs = rng.choice([D // 2, rng.randint(max(1, axes), max(axes, D // 2))])
        tokens = _log(rng, 1, min(16384, (1 << 25) // (H * D)))
        T = _log(rng, 1, tokens)
        return {"kind": kind, "B": max(1, tokens // T), "T": T, "H": H, "G": G, "D": D, "axes": axes, "pairs": pairs,
                "interleaved": rng.random() < 0.5, "far": _log(rng, 100, 1000000)}
    if kind in ("attn", "attntr"):
        room = (1 << 29) // H
        N = _log(rng, 1, 4096 if kind == "attntr" else 16384)
        T = N if kind == "attntr" or N < 8 or rng.random() < 0.5 else _log(rng, 1, N // 2)
        T = max(1, min(T, room // N))
        N = T if kind == "attntr" else N
        return {"kind": kind, "B": _log(rng, 1, max(1, min(64, room // (T * N)))), "T": T, "N": N, "H": H, "G": G,
                "D": D, "causal": T != N or rng.random() < 0.7, "ragged": rng.random() < 0.4}
    case = {"kind": kind, "G": G, "D": D, "page": rng.choice([1, 7, 16, 48, 64, 128]),
            "type": rng.choice(["float32", "bfloat16", FP8, FP8])}
    if kind == "step":
        N = _log(rng, 1, 32768)
        return {**case, "B": _log(rng, 1, max(1, min(64, (1 << 27) // (N * G * D), (1 << 24) // (N * H)))), "N": N,
                "H": H}
    N = _log(rng, 1, 8192)
    case |= {"B": _log(rng, 1, max(1, min(64, (1 << 25) // (N * G * D)))), "N": N}
    if kind == "write":
        case["T"] = _log(rng, 1, N)
    return case


# ------------------------------------------------------------------------------ inputs
def _sections(case):
    a, p = case["axes"], case["pairs"]
    return tuple(p // a + (i < p % a) for i in range(a))


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=gen, device=DEV).mul_(std)

    def spread(*shape, lo=0.005, hi=0.1):
        return torch.rand(shape, generator=gen, device=DEV).mul_(hi - lo).add_(lo)

    def whole(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=gen, device=DEV, dtype=torch.int32)

    def pair(name, *shape, std=1.0):
        s["m" + name], s["S" + name] = normal(*shape, std=std), spread(*shape)

    def deltas(name, *shape):
        s["dm" + name], s["dS" + name] = normal(*shape, std=0.1), spread(*shape, lo=-0.02, hi=-1e-4)

    kind, B, G, D = case["kind"], case["B"], case["G"], case["D"]
    s = {"case": case, "scale": 1.0 / math.sqrt(D)}
    if kind in ("rot", "rottr"):
        T, H, A = case["T"], case["H"], case["axes"]
        pair("q", B, T, H, D, std=2.0), pair("k", B, T, G, D, std=2.0)
        first = whole(0, case["far"], B, 1, A)
        s["positions"] = first + torch.arange(T, device=DEV, dtype=torch.int32)[:, None] // (
            32 ** torch.arange(A, device=DEV, dtype=torch.int32))
        if A == 1:
            s["positions"] = s["positions"][..., 0].contiguous()
        n = torch.arange(case["pairs"], device=DEV, dtype=torch.float64)
        s["frequencies"] = THETA ** (-n / case["pairs"])
        s["sections"] = _sections(case)
        s["weights"] = tuple(x for _ in range(2) for x in (normal(D, std=0.1).add_(1.0), spread(D, hi=0.02)))
        if kind == "rottr":
            deltas("q", B, T, H, D), deltas("k", B, T, G, D)
        return s
    N = case["N"]
    if kind in ("attn", "attntr"):
        T, H = case["T"], case["H"]
        pair("q", B, T, H, D), pair("k", B, N, G, D), pair("v", B, N, G, D)
        s["lengths"] = s["starts"] = None
        if case["ragged"]:
            s["lengths"] = whole(1, N + 1, B)
            s["lengths"][0] = 0 if B > 1 else s["lengths"][0]
        if T != N:  # the queries are the newest tokens of the context
            s["starts"] = torch.full((B,), N - T, device=DEV, dtype=torch.int32)
            if case["ragged"]:
                s["starts"] = (s["lengths"] - T).clamp_min(0)
        if kind == "attntr":
            deltas("o", B, T, H, D)
        return s
    page = case["page"]
    room = -(-N // page)  # pages of a sequence
    pages = B * room + 3
    s["table"] = torch.randperm(pages, generator=gen, device=DEV)[:B * room].view(B, room).to(torch.int32)
    type_ = getattr(torch, case["type"])
    small = case["type"] == FP8
    shape = (pages, G, page, D)
    pools = []
    for i in range(4):
        x = normal(*shape) if i % 2 == 0 else spread(*shape)
        # means of a row reach about 4, variances 0.1: what its exponent brings near the type's 448
        pools.append((x.mul_(64.0 if i % 2 == 0 else 4096.0) if small else x).to(type_))
        del x
    scales = None
    if small:
        scales = torch.tensor([121, 115, 121, 115], device=DEV, dtype=torch.uint8).expand(pages, G, page, 4)
        scales = scales.contiguous()
    s["cache"] = (*pools, scales)
    if kind == "write":
        T = case["T"]
        pair("k", B, T, G, D), pair("v", B, T, G, D)
        s["starts"] = whole(0, N - T + 1, B)
    elif kind == "read":
        s["lengths"] = whole(0, N + 1, B)
        s["lengths"][0] = N
    else:
        pair("q", B, case["H"], D)
        s["lengths"] = whole(N - N // 4, N + 1, B)  # sequences of about one age
    return s


# ------------------------------------------------------------------- the framework's calls
def _own(s):
    from triton_tagi_amd import kernels as K

    kind = s["case"]["kind"]
    if kind in ("rot", "rottr"):
        kw = dict(sections=s["sections"], interleaved=s["case"]["interleaved"])
        *out, inv = K.qk_norm_rotary(s["mq"], s["Sq"], s["mk"], s["Sk"], s["positions"], s["frequencies"],
                                     s["weights"], eps=EPS, **kw)
        if kind == "rot":
            return out
        return (*out, *K.qk_norm_rotary_backward(s["dmq"], s["dSq"], s["dmk"], s["dSk"], s["mq"], s["mk"], inv,
                                                 s["positions"], s["frequencies"], s["weights"], **kw))
    if kind in ("attn", "attntr"):
        kw = dict(scale=s["scale"], causal=s["case"]["causal"], lengths=s["lengths"], starts=s["starts"])
        qk = (s["mq"], s["Sq"], s["mk"], s["Sk"], s["mv"])
        if kind == "attn":
            return K.remax_attention(*qk, s["Sv"], **kw)
        mo, So, rows = K.remax_attention(*qk, s["Sv"], return_rows=True, **kw)
        return (mo, So, *K.remax_attention_backward(*qk, s["dmo"], s["dSo"], rows, **kw))
    cache = K.KVCache(*s["cache"])
    if kind == "write":
        K.cache_write(cache, s["mk"], s["Sk"], s["mv"], s["Sv"], s["table"], s["starts"])
        return tuple(t for t in cache if t is not None)
    if kind == "read":
        return K.cache_read(cache, s["table"], s["lengths"], s["case"]["N"])
    return K.remax_attention_step(s["mq"], s["Sq"], cache, s["table"], s["lengths"], scale=s["scale"])


# --------------------------------------------------------------------------- plain forms
def _turns(s):
    """cos and sin of every token's pairs, (B, T, 1, pairs); angles of far positions in 64 bits."""
    pos = s["positions"].double()
    if pos.dim() == 3:
        axis = torch.repeat_interleave(torch.arange(len(s["sections"]), device=DEV),
                                       torch.tensor(s["sections"], device=DEV), output_size=s["case"]["pairs"])
        pos = pos[..., axis]
    else:
        pos = pos[..., None]
    a = (pos * s["frequencies"])[:, :, None]
    return torch.cos(a).float(), torch.sin(a).float()


def _split(s, x):
    """The two features of every pair, and the features that no pair holds."""
    n = 2 * s["case"]["pairs"]
    if s["case"]["interleaved"]:
        return x[..., 0:n:2], x[..., 1:n:2], x[..., n:]
    return x[..., :n // 2], x[..., n // 2:n], x[..., n:]


def _join(s, a, b, rest):
    if s["case"]["interleaved"]:
        return torch.cat([torch.stack([a, b], -1).flatten(-2), rest], -1)
    return torch.cat([a, b, rest], -1)


def _plain_rotary(s):
    c, n = _turns(s)
    out, back, gamma = [], [], []
    for x, mw, Sw in (("q", *s["weights"][:2]), ("k", *s["weights"][2:])):
        m, S = s["m" + x], s["S" + x]
        inv = torch.rsqrt((m * m + S).mean(-1, keepdim=True) + EPS)
        hat = m * inv
        a, b, rest = _split(s, hat * mw)
        out.append(_join(s, a * c - b * n, a * n + b * c, rest))
        a, b, rest = _split(s, inv * inv * (S * (mw * mw + Sw)) + Sw * (hat * hat))
        out.append(_join(s, a * (c * c) + b * (n * n), a * (n * n) + b * (c * c), rest))
        if s["case"]["kind"] == "rottr":
            a, b, rest = _split(s, s["dm" + x])
            dm = _join(s, a * c + b * n, b * c - a * n, rest)
            a, b, rest = _split(s, s["dS" + x])
            dS = _join(s, a * (c * c) + b * (n * n), a * (n * n) + b * (c * c), rest)
            w = inv * mw
            back += [dm * w, dS * (w * w)]
            gamma += [Sw * (dm * hat).sum((0, 1, 2)), Sw * Sw * (dS * (hat * hat)).sum((0, 1, 2))]
    return (*out, *back, *gamma)


def _remax(m, v, seen, jacobian):
    """Remax over the last axis of scores (m, v) where ``seen``, zeros elsewhere: mu_a, S_a (and J).
    The rectified moments through the scaled complementary error function, so that neither side cancels."""
    sd = v.sqrt()
    al = m / sd
    x = al.abs()
    pdf = torch.exp(-0.5 * x * x) * (1.0 / math.sqrt(2.0 * math.pi))
    # the lower tail's mean (over sd pdf) and square (over v pdf) are differences of near values: in 64 bits
    mills = torch.special.erfcx(x.double() * math.sqrt(0.5)) * math.sqrt(0.5 * math.pi)
    low = 1.0 - x * mills
    second = (mills - x * low).float()
    low, tail = low.float(), pdf * mills.float()
    del mills
    mean = sd * pdf * low
    var = pdf * second - (pdf * low) ** 2
    del second
    up = al >= 0
    raw = torch.where(up, mean + m, mean)
    var = v * torch.where(up, 1.0 - var - 2.0 * (pdf * low) * (pdf * low + x), var)
    cdf = torch.where(up, 1.0 - tail, tail)
    mm = raw.clamp_min(EPS)
    vm = (var + (raw - mm) * (raw + mm - 2.0 * m)).clamp_min(EPS)
    del raw, var, mean, tail, low, pdf, x, al, sd
    mt = torch.where(seen, mm, 0.0).sum(-1, keepdim=True).clamp_min(EPS)
    vt = torch.where(seen, vm, 0.0).sum(-1, keepdim=True).clamp_min(EPS)
    y = vt / (mt * mt)
    x, w = vm / (mm * mm), vm / (mm * mt)
    del vm
    mua = torch.where(seen, ((mm / mt) * ((1.0 + y) / (1.0 + w))).clamp_min(EPS), 0.0)
    mua = mua / mua.sum(-1, keepdim=True).clamp_min(EPS)
    vara = (((x - w) + (y - w)) + (x * y - w * w)).clamp_min(0.0) * (mua / (1.0 + w)) ** 2
    if not jacobian:
        return mua, vara
    cov = (x - w).clamp_min(0.0) / (1.0 + w) * mua * mm
    return mua, vara, torch.minimum((vara * v).sqrt(), cov / cdf.clamp_min(EPS)) / v


def _plain_attention(s):
    case, c = s["case"], s["scale"]
    B, T, N, H, G, D = (case[x] for x in ("B", "T", "N", "H", "G", "D"))
    R = H // G
    at = torch.arange(T, device=DEV)[None] + (0 if s["starts"] is None else s["starts"][:, None])  # (B or 1, T)
    key = torch.arange(N, device=DEV)
    length = torch.full((1,), N, device=DEV) if s["lengths"] is None else s["lengths"]
    seen = (key < length[:, None])[:, None] & (at < length[:, None])[..., None]
    if case["causal"]:
        seen = seen & (key <= at[..., None])
    seen = seen[:, None, None]  # (B or 1, 1, 1, T, N)

    def queries(x):  # (B, T, H, D) -> (B, G, R, T, D)
        return x.transpose(1, 2).reshape(B, G, R, T, D)

    def keys(x):  # (B, N, G, D) -> (B, G, 1, N, D)
        return x.transpose(1, 2).reshape(B, G, 1, N, D)

    def product(a, b):  # (B, G, R, T, X) with (B, G, 1, X, Y), the group's queries one under another
        return torch.matmul(a.reshape(B, G, R * T, -1), b[:, :, 0]).view(B, G, R, T, -1)

    def over_keys(a, b):  # the same with X the keys: long sums, in 64 bits
        return product(a.double(), b.double()).float()

    def heads(x):  # (B, G, R, T, D) -> (B, T, H, D)
        return x.reshape(B, H, T, D).transpose(1, 2)

    mq, Sq, mk, Sk, mv, Sv = queries(s["mq"]), queries(s["Sq"]), *(keys(s[n]) for n in ("mk", "Sk", "mv", "Sv"))
    flip = (lambda x: x.transpose(-1, -2).contiguous())
    m = product(mq, flip(mk)).mul_(c)
    v = product(Sq, flip(mk * mk + Sk)).add_(product(mq * mq, flip(Sk))).mul_(c * c)
    train = case["kind"] == "attntr"
    mua, vara, *J = _remax(m, v, seen, train)
    del m, v
    square = mua * mua
    out = [heads(over_keys(mua, mv)), heads(over_keys(vara, mv * mv + Sv).add_(over_keys(square, Sv)))]
    if not train:
        return tuple(out)
    del vara
    J = J[0]

    def back(p, x):  # p^T x, summed over the group's queries in 64 bits: (B, N, G, D)
        p, x = flip(p.view(B, G, R * T, N)).double(), x.reshape(B, G, R * T, D).double()
        return torch.matmul(p, x).float().transpose(1, 2)

    dm, dS = queries(s["dmo"]), queries(s["dSo"])
    dv = [back(mua, dm), back(square, dS)]
    del square, mua
    dsm = product(dm, flip(mv)).mul_(J).mul_(c)
    dsS = product(dS, flip(mv * mv)).mul_(J).mul_(J).mul_(c * c)
    dsm, dsS = torch.where(seen, dsm, 0.0), torch.where(seen, dsS, 0.0)
    del J
    out += [heads(over_keys(dsm, mk)), heads(over_keys(dsS, mk * mk))]
    return (*out, back(dsm, mq), back(dsS, mq * mq), *dv)


def _exponents(x):
    """Biased exponents (rows) that bring a row's largest magnitude to at most 448 = 0.875 * 2^9."""
    f, e = torch.frexp(x.abs().amax(-1))
    return torch.where(f > 0.875, e - 8, e - 9).add(127).clamp(1, 254)


def _plain_write(s):
    case = s["case"]
    B, T, G, page = case["B"], case["T"], case["G"], case["page"]
    at = (s["starts"][:, None] + torch.arange(T, device=DEV)).long()
    where = (s["table"].gather(1, at // page).long(), at % page)
    *pools, scales = s["cache"]
    for i, (pool, x) in enumerate(zip(pools, (s["mk"], s["Sk"], s["mv"], s["Sv"]))):
        if scales is not None:
            e = _exponents(x)
            scales[where[0], :, where[1], i] = e.to(torch.uint8)
            x = torch.ldexp(x, 127 - e[..., None])
            pool.view(torch.uint8)[where[0], :, where[1]] = x.to(pool.dtype).view(torch.uint8)
        else:
            pool[where[0], :, where[1]] = x.to(pool.dtype)
    return tuple(t for t in s["cache"] if t is not None)


def _tokens(s):
    """The cache's tokens as float32, (B, N, G, D) each, zeros from a sequence's length on."""
    case = s["case"]
    B, N, G, D = (case[x] for x in ("B", "N", "G", "D"))
    *pools, scales = s["cache"]
    table = s["table"].long()
    live = (torch.arange(N, device=DEV) < s["lengths"][:, None])[:, :, None, None]
    out = []
    for i, pool in enumerate(pools):
        small = pool.element_size() == 1
        x = (pool.view(torch.uint8) if small else pool)[table].transpose(2, 3).reshape(B, -1, G, D)[:, :N]
        x = x.contiguous().view(pool.dtype).float()
        if scales is not None:
            e = scales[..., i][table].transpose(2, 3).reshape(B, -1, G, 1)[:, :N]
            x = x * torch.exp2(e.float() - 127.0)
        out.append(torch.where(live, x, 0.0))
    return out


def _plain_step(s):
    case, c = s["case"], s["scale"]
    B, N, H, G, D = (case[x] for x in ("B", "N", "H", "G", "D"))
    R = H // G
    mk, Sk, mv, Sv = (x.transpose(1, 2).contiguous() for x in _tokens(s))  # (B, G, N, D)
    mq, Sq = s["mq"].view(B, G, R, D), s["Sq"].view(B, G, R, D)
    seen = (torch.arange(N, device=DEV) < s["lengths"][:, None])[:, None, None]
    flip = (lambda x: x.transpose(-1, -2).contiguous())
    m = torch.matmul(mq, flip(mk)) * c
    v = (torch.matmul(Sq, flip(mk * mk + Sk)) + torch.matmul(mq * mq, flip(Sk))) * (c * c)
    v = torch.where(seen, v, 1.0)
    mua, vara = _remax(m, v, seen, False)
    mo = torch.matmul(mua, mv)
    So = torch.matmul(vara, mv * mv + Sv) + torch.matmul(mua * mua, Sv)
    return mo.view(B, H, D), So.view(B, H, D)


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    if kind in ("rot", "rottr"):
        return _plain_rotary(state)
    if kind in ("attn", "attntr"):
        return _plain_attention(state)
    if kind == "write":
        return _plain_write(state)
    return tuple(_tokens(state)) if kind == "read" else _plain_step(state)


# ------------------------------------------------------------------------------- work
def work(case):
    kind, B, G, D = case["kind"], case["B"], case["G"], case["D"]
    if kind in ("rot", "rottr"):
        tokens = B * case["T"]
        n = tokens * (case["H"] + G) * D
        small = 4 * tokens * case["axes"] + 8 * case["pairs"] + 16 * D
        if kind == "rot":
            return {"bytes": 16 * n + small, "flops": 20 * n}
        # backward: two deltas and the mean read, two written
        return {"bytes": 36 * n + small + 16 * D, "flops": 36 * n}
    N = case["N"]
    if kind in ("attn", "attntr"):
        T, H = case["T"], case["H"]
        live = 0.5 if case["ragged"] else 1.0  # expected share of a sequence's keys
        scores = B * H * T * N * live
        if case["causal"]:
            scores = B * H * T * (N * live - (0.5 * T if T < N else 0.5 * N * live))
        flops = scores * (12 * D + 60)  # three products each for the scores and the outputs, and the Remax
        moved = 8 * D * B * (2 * T * H + 2 * N * G)
        if kind == "attntr":  # the scores again (3), and two products each for V, the scores, Q and K
            flops += scores * (22 * D + 70)
            moved += 8 * D * B * (3 * T * H + 4 * N * G)
        return {"bytes": moved, "flops": flops}
    size = {"float32": 4, "bfloat16": 2, FP8: 1}[case["type"]]
    row = 4 * D * size + (4 if size == 1 else 0)  # a token's entry for one head
    if kind == "write":
        n = B * case["T"] * G
        return {"bytes": n * (16 * D + row), "flops": 8 * n * D}
    if kind == "read":
        live = (N + (B - 1) * N * 0.5) * G
        return {"bytes": live * row + 16 * D * B * N * G, "flops": 4 * live * D}
    live = B * N * 0.875
    return {"bytes": live * G * row + 16 * B * case["H"] * D, "flops": live * case["H"] * (12 * D + 60)}


# ---------------------------------------------------------------------- values in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("rot", "rottr"):
        return _exact_rotary(s)
    if kind in ("attn", "attntr"):
        return _exact_attention(s)
    if kind == "write":
        return _exact_write(s)
    if kind == "read":
        return _exact_read(s)
    return _exact_step(s)


def _exact_rotary(s):
    case, n = s["case"], s["case"]["pairs"]
    i = torch.arange(n, device=DEV)
    first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + n)
    axis = torch.tensor([a for a, k in enumerate(s["sections"]) for _ in range(k)], device=DEV)
    pos = s["positions"].double().reshape(*s["positions"].shape[:2], -1)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), pos[:, :, axis] * s["frequencies"])[:, :, None]
    square = torch.complex(turn.real**2, turn.imag**2)

    def mean(x, turn):  # each pair as a complex number
        z = torch.complex(x[..., first], x[..., second]) * turn
        x = x.clone()
        x[..., first], x[..., second] = z.real, z.imag
        return x

    def variance(x):
        a, b = x[..., first], x[..., second]
        x = x.clone()
        x[..., first], x[..., second] = a * square.real + b * square.imag, a * square.imag + b * square.real
        return x

    out, back, gamma = [], [], []
    for x, mw, Sw in (("q", *s["weights"][:2]), ("k", *s["weights"][2:])):
        m, S, mw, Sw = s["m" + x].double(), s["S" + x].double(), mw.double(), Sw.double()
        r = ((m.square() + S).mean(-1, keepdim=True) + EPS).sqrt()
        out += [mean(m / r * mw, turn), variance((S * (mw.square() + Sw) + Sw * m.square()) / r.square())]
        if case["kind"] == "rottr":
            dm, dS = mean(s["dm" + x].double(), turn.conj()), variance(s["dS" + x].double())
            back += [dm * mw / r, dS * (mw / r).square()]
            gamma += [Sw * (dm * m / r).sum((0, 1, 2)), Sw.square() * (dS * (m / r).square()).sum((0, 1, 2))]
    return (*out, *back, *gamma)


def _exact_remax(m, v, seen):
    """Remax of each row by its logarithms; rows that see nothing are zeros."""
    sd = v.sqrt()
    al = m / sd
    pdf, cdf = torch.exp(-0.5 * al.square()) / math.sqrt(2 * math.pi), 0.5 * torch.special.erfc(-al / math.sqrt(2.0))
    mm = (m * cdf + sd * pdf).clamp(min=EPS)
    vm = (-mm.square() + 2 * mm * m - m * sd * pdf + (v - m.square()) * cdf).clamp(min=EPS)
    mt = (mm * seen).sum(-1, keepdim=True).clamp(min=EPS)
    vt = (vm * seen).sum(-1, keepdim=True).clamp(min=EPS)
    lm, lt, lmt = torch.log1p(vm / mm.square()), torch.log1p(vt / mt.square()), torch.log1p(vm / (mm * mt))
    la = (lm + lt - 2 * lmt).clamp(min=0)
    mu = (mm.log() - 0.5 * lm) - (mt.log() - 0.5 * lt)
    mua = torch.exp(mu + 0.5 * (lm + lt - 2 * lmt)).clamp(min=EPS) * seen
    mua = mua / mua.sum(-1, keepdim=True).clamp(min=EPS)
    vara = torch.expm1(la) * mua.square()
    cov = torch.expm1((lm - lmt).clamp(min=0)) * mua * mm
    J = torch.minimum((vara * v).sqrt(), cov / cdf.clamp(min=EPS)) / v
    return mua, vara, J * seen


def _exact_attention(s):
    case, c = s["case"], s["scale"]
    B, T, N, H, G, D = (case[x] for x in ("B", "T", "N", "H", "G", "D"))
    train = case["kind"] == "attntr"
    names = ("mq", "Sq", "mk", "Sk", "mv", "Sv") + (("dmo", "dSo") if train else ())
    x = {n: s[n].double() for n in names}
    like = [x["mq"], x["mq"]] + ([x["mq"], x["mq"]] + [x["mk"]] * 4 if train else [])
    out = [torch.zeros_like(t) for t in like]
    key = torch.arange(N, device=DEV)
    for b in range(B):
        at = torch.arange(T, device=DEV) + (0 if s["starts"] is None else s["starts"][b].long())
        length = N if s["lengths"] is None else s["lengths"][b].long()
        seen = ((key < length)[None] & (at < length)[:, None] & ((key[None] <= at[:, None]) | (not case["causal"])))
        for h in range(H):
            g = h // (H // G)
            mq, Sq = x["mq"][b, :, h], x["Sq"][b, :, h]
            mk, Sk, mv, Sv = (x[n][b, :, g] for n in ("mk", "Sk", "mv", "Sv"))
            m = c * (mq @ mk.T)
            v = c * c * (Sq @ mk.square().T + Sq @ Sk.T + mq.square() @ Sk.T)
            a, Sa, J = _exact_remax(m, v, seen.double())
            out[0][b, :, h] = a @ mv
            out[1][b, :, h] = Sa @ mv.square() + Sa @ Sv + a.square() @ Sv
            if train:
                dm, dS = x["dmo"][b, :, h], x["dSo"][b, :, h]
                em, eS = c * J * (dm @ mv.T), c * c * J.square() * (dS @ mv.square().T)
                out[2][b, :, h], out[3][b, :, h] = em @ mk, eS @ mk.square()
                for i, d in enumerate((em.T @ mq, eS.T @ mq.square(), a.T @ dm, a.square().T @ dS)):
                    out[4 + i][b, :, g] += d
    return tuple(out)


def _exact_round(x, type_):
    """Nearest value of the type, ties to even: steps of 2^(e - 3) (e4m3), 2^(e - 7) (bfloat16)."""
    if type_ == "float32":
        return x
    bits, least = (3, -6) if type_ == FP8 else (7, -126)
    e = (torch.frexp(x)[1] - 1).clamp(min=least)
    step = torch.exp2((e - bits).double())
    return torch.round(x / step) * step


def _exact_write(s):
    case = s["case"]
    page, type_ = case["page"], case["type"]
    *pools, scales = s["cache"]
    pools = [p.double() for p in pools]
    start, table = s["starts"].tolist(), s["table"].tolist()
    for b in range(case["B"]):
        at = torch.arange(start[b], start[b] + case["T"], device=DEV)
        rows, slots = torch.tensor(table[b], device=DEV)[at // page], at % page
        for i, n in enumerate(("mk", "Sk", "mv", "Sv")):
            x = s[n][b].double()  # (T, G, D)
            if scales is not None:
                # the least power of two that brings the row under 448 (up to the type's ends)
                e = torch.ceil(torch.log2(x.abs().amax(-1) / 448.0)).clamp(-126, 127)
                x = x / torch.exp2(e)[..., None]
                scales[rows, :, slots, i] = (e + 127).to(torch.uint8)
            pools[i][rows, :, slots] = _exact_round(x, type_)
    return (*pools, scales) if scales is not None else tuple(pools)


def _exact_read(s):
    case = s["case"]
    B, N, G, D, page = (case[x] for x in ("B", "N", "G", "D", "page"))
    *pools, scales = s["cache"]
    outs = [torch.zeros(B, N, G, D, device=DEV, dtype=torch.float64) for _ in range(4)]
    for b, n in enumerate(s["lengths"].tolist()):
        at = torch.arange(n, device=DEV)
        rows, slots = s["table"][b].long()[at // page], at % page
        for i in range(4):
            x = pools[i].view(torch.uint8 if case["type"] == FP8 else pools[i].dtype)[rows, :, slots]
            x = x.view(pools[i].dtype).double()
            if scales is not None:
                x = x * torch.exp2(scales[rows, :, slots, i].double() - 127)[..., None]
            outs[i][b, :n] = x
    return tuple(outs)


def _exact_step(s):
    case, c = s["case"], s["scale"]
    B, H, G, D = (case[x] for x in ("B", "H", "G", "D"))
    mo = torch.zeros(B, H, D, device=DEV, dtype=torch.float64)
    So = torch.zeros_like(mo)
    everything = {**s}
    for b, n in enumerate(s["lengths"].tolist()):
        everything["case"] = {**case, "B": 1, "N": n}
        everything["lengths"], everything["table"] = s["lengths"][b:b + 1], s["table"][b:b + 1]
        mk, Sk, mv, Sv = (x[0] for x in _exact_read(everything))  # (n, G, D)
        for h in range(H):
            g = h // (H // G)
            q, Sq = s["mq"][b, h].double(), s["Sq"][b, h].double()
            m = c * (mk[:, g] @ q)
            v = c * c * (mk[:, g].square() @ Sq + Sk[:, g] @ Sq + Sk[:, g] @ q.square())
            a, Sa, _ = _exact_remax(m[None], v[None], torch.ones(1, n, device=DEV, dtype=torch.float64))
            mo[b, h] = (a @ mv[:, g])[0]
            So[b, h] = (Sa @ (mv[:, g].square() + Sv[:, g]) + a.square() @ Sv[:, g])[0]
    return mo, So
