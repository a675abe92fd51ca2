"""RMSNorm of every query and key head and its rotation by position, on Gaussian moments.

For a head's moments (m, S), its weight's (g, Sg) and a pair of features (a, b) that turns by
t = position * frequency:

    inv = 1 / sqrt(mean(m^2 + S) + eps)
    n = m inv g,  N = inv^2 (S (g^2 + Sg) + Sg m^2)
    (a, b) of n -> (a cos t - b sin t, a sin t + b cos t)
    (A, B) of N -> (A cos^2 t + B sin^2 t, A sin^2 t + B cos^2 t)

Queries (B, T, H, D) and keys (B, T, G, D) go through one launch, read in place with any strides
but the last dim's, which is 1. Features stay independent (a pair's covariance is dropped).
"""

from __future__ import annotations

import ctypes

import torch
from torch import Tensor

from .. import _lib
from ._operands import dense_like, heads, mean, pair, shape_of, written


def rotary_frequencies(pairs: int, base: float = 10000.0, device="cuda") -> Tensor:
    """base^(-u / pairs) radians a position, u < pairs: (pairs,) float64."""
    u = torch.arange(pairs, device=device, dtype=torch.float64)
    return float(base) ** (-u / max(1, pairs))


def _sizes(mq: Tensor, mk: Tensor):
    shape = shape_of(mq, "mq", 4)
    G = shape_of(mk, "mk", 4)[2]
    B, T, H, D = shape
    if D > 256:
        raise ValueError(f"qk_norm_rotary supports head dimensions up to 256, got {D}")
    return shape, torch.Size((B, T, G, D))


def _weights(weights, ref: Tensor, D: int):
    if weights is None:
        return (None,) * 4
    try:
        mwq, Swq, mwk, Swk = weights
    except (TypeError, ValueError):
        raise TypeError("weights: expected (mwq, Swq, mwk, Swk) or None") from None
    names = ("mwq", "Swq", "mwk", "Swk")
    return tuple(_lib.dense_with(w, n, ref, (D,)) for w, n in zip((mwq, Swq, mwk, Swk), names))


def _turns(positions, frequencies, sections, ref: Tensor, shape):
    """(positions, their bytes, axes, sections, frequencies, pairs); all empty without positions."""
    if positions is None:
        if frequencies is not None or sections is not None:
            raise ValueError("frequencies and sections belong to positions")
        return None, 4, 0, None, None, 0
    B, T, _, D = shape
    if not isinstance(positions, Tensor) or positions.dtype not in (torch.int32, torch.int64):
        raise TypeError("positions: expected an int32 or int64 tensor")
    axes = 1 if positions.dim() == 2 else (positions.shape[2] if positions.dim() == 3 else 0)
    if positions.device != ref.device or tuple(positions.shape[:2]) != (B, T) or not 1 <= axes <= 4:
        raise ValueError(f"positions: expected ({B}, {T}) or ({B}, {T}, 1 to 4 axes) on {ref.device}, "
                         f"got {tuple(positions.shape)} on {positions.device}")
    if not isinstance(frequencies, Tensor) or frequencies.dtype is not torch.float64:
        raise TypeError("frequencies: expected a float64 tensor")
    pairs = frequencies.numel()
    if frequencies.device != ref.device or frequencies.dim() != 1 or not 1 <= pairs <= D // 2:
        raise ValueError(f"frequencies: expected 1 to {D // 2} pairs on {ref.device}, "
                         f"got {tuple(frequencies.shape)} on {frequencies.device}")
    if sections is None:
        if axes != 1:
            raise ValueError(f"sections: needed for positions of {axes} axes")
        sections = (pairs,)
    sections = tuple(int(n) for n in sections)
    if len(sections) != axes or min(sections) < 0 or sum(sections) != pairs:
        raise ValueError(f"sections: expected {axes} counts that add up to {pairs} pairs, got {sections}")
    return (positions.contiguous(), positions.element_size(), axes, (ctypes.c_int64 * axes)(*sections),
            frequencies.contiguous(), pairs)


def qk_norm_rotary(mq: Tensor, Sq: Tensor, mk: Tensor, Sk: Tensor, positions: Tensor | None = None,
                   frequencies: Tensor | None = None, weights=None, sections=None, interleaved: bool = False,
                   eps: float = 1e-6):
    """(mq, Sq, mk, Sk, inv): the moments normed and turned, dense; inv (B, T, H + G), the norm's
    factors for the backward, is None without ``weights``.

    ``weights``: (mwq, Swq, mwk, Swk), each (D,), or None for no norm. ``positions`` (B, T) or
    (B, T, axes), int32 or int64, or None for no rotation; ``frequencies`` (pairs,) float64 radians a
    position, 2 pairs <= D (the features after them stay). With several axes the first
    ``sections[0]`` pairs turn by the first axis, and so on. A pair is features (u, u + pairs), or
    (2u, 2u + 1) if ``interleaved``."""
    qs, ks = _sizes(mq, mk)
    B, T, H, D = qs
    G = ks[2]
    mq, Sq = pair(mq, Sq, "q", mq, qs)
    mk, Sk = pair(mk, Sk, "k", mq, ks)
    w = _weights(weights, mq, D)
    pos, pos_bytes, axes, sec, freq, pairs = _turns(positions, frequencies, sections, mq, qs)
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    oqm, okm = dense_like(mq, qs), dense_like(mk, ks)
    oqS, okS = torch.empty_like(oqm), torch.empty_like(okm)
    inv = None if weights is None else mq.new_empty((B, T, H + G))
    _lib.call_on(mq, "tagi_qk_rotary_fwd", mq.data_ptr(), Sq.data_ptr(), heads(mq), mk.data_ptr(), Sk.data_ptr(),
                 heads(mk), *(_lib.ptr(x) for x in w), _lib.ptr(pos), pos_bytes, axes, sec, _lib.ptr(freq), pairs,
                 int(interleaved), float(eps), oqm.data_ptr(), oqS.data_ptr(), okm.data_ptr(), okS.data_ptr(),
                 _lib.ptr(inv), B, T, H, G, D, _lib.stream_of(mq))
    return oqm, oqS, okm, okS, inv


def qk_norm_rotary_backward(delta_mq: Tensor, delta_Sq: Tensor, delta_mk: Tensor, delta_Sk: Tensor, mq: Tensor,
                            mk: Tensor, inv: Tensor | None, positions: Tensor | None = None,
                            frequencies: Tensor | None = None, weights=None, sections=None,
                            interleaved: bool = False) -> tuple[Tensor, ...]:
    """(dmq, dSq, dmk, dSk) of ``qk_norm_rotary``, with ``weights`` also their deltas (dmwq, dSwq,
    dmwk, dSwk), each (D,). ``mq``, ``mk``: the forward's input means. The deltas turn back, then

        dm = d inv g, dS = D (inv g)^2;  dmw = Sg sum d inv m, dSw = Sg^2 sum D (inv m)^2."""
    oqm, okm = (dense_like(t, t.shape) for t in (mq, mk))
    out = (oqm, torch.empty_like(oqm), okm, torch.empty_like(okm))
    return (*out, *_backward(out, delta_mq, delta_Sq, delta_mk, delta_Sk, mq, mk, inv, positions, frequencies, weights,
                             sections, interleaved))


def qk_norm_rotary_backward_into(out, delta_mq: Tensor, delta_Sq: Tensor, delta_mk: Tensor, delta_Sk: Tensor,
                                 mq: Tensor, mk: Tensor, inv: Tensor | None, positions: Tensor | None = None,
                                 frequencies: Tensor | None = None, weights=None, sections=None,
                                 interleaved: bool = False) -> tuple[Tensor, ...]:
    """``qk_norm_rotary_backward`` into four tensors (a mean's and its variance's in one layout, unit
    last stride), which may be the four deltas themselves; returns the weights' deltas."""
    qs, ks = _sizes(mq, mk)
    oqm, oqS, okm, okS = out
    written((oqm, oqS), ("dmq", "dSq"), mq, qs)
    written((okm, okS), ("dmk", "dSk"), mq, ks)
    return _backward(out, delta_mq, delta_Sq, delta_mk, delta_Sk, mq, mk, inv, positions, frequencies, weights, sections,
                     interleaved)


def _backward(out, delta_mq: Tensor, delta_Sq: Tensor, delta_mk: Tensor, delta_Sk: Tensor, mq: Tensor, mk: Tensor,
              inv: Tensor | None, positions: Tensor | None, frequencies: Tensor | None, weights, sections,
              interleaved: bool) -> tuple[Tensor, ...]:
    qs, ks = _sizes(mq, mk)
    B, T, H, D = qs
    G = ks[2]
    mq, mk = mean(mq, "q", mq, qs), mean(mk, "k", mq, ks)
    dmq, dSq = pair(delta_mq, delta_Sq, "q (delta)", mq, qs)
    dmk, dSk = pair(delta_mk, delta_Sk, "k (delta)", mq, ks)
    w = _weights(weights, mq, D)
    if weights is not None:
        inv = _lib.dense_with(inv, "inv", mq, (B, T, H + G))
    pos, pos_bytes, axes, sec, freq, pairs = _turns(positions, frequencies, sections, mq, qs)
    oqm, oqS, okm, okS = out
    dw = ()
    ws = None
    if weights is not None:
        dw = mq.new_empty((4, D)).unbind()
        ws = _lib.workspace(_lib.query("tagi_qk_rotary_bwd_ws_bytes", B, T, H, G, D), mq.device)
    wp, wb = _lib.ws_args(ws)
    _lib.call_on(mq, "tagi_qk_rotary_bwd", dmq.data_ptr(), dSq.data_ptr(), heads(dmq), dmk.data_ptr(), dSk.data_ptr(),
                 heads(dmk), mq.data_ptr(), heads(mq), mk.data_ptr(), heads(mk), _lib.ptr(inv),
                 *(_lib.ptr(x) for x in w), _lib.ptr(pos), pos_bytes, axes, sec, _lib.ptr(freq), pairs,
                 int(interleaved), oqm.data_ptr(), oqS.data_ptr(), heads(oqm), okm.data_ptr(), okS.data_ptr(),
                 heads(okm), *((x.data_ptr() for x in dw) if dw else (None,) * 4), B, T, H, G, D, wp, wb,
                 _lib.stream_of(mq))
    return dw
