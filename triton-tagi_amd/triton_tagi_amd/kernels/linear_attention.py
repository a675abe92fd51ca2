"""Linear attention with a decay for each head, on Gaussian moments.

A head's state is a D x D matrix of independent Gaussians (means M, variances P). With its
decay g and the scale c, token t advances it and reads it:

    M_t = g M_{t-1} + k v^T,   P_t = g^2 P_{t-1} + Sk (v^2 + Sv)^T + (k^2) Sv^T
    mo  = c M_t^T q,           So  = c^2 [P_t^T (Sq + q^2) + (M_t.M_t)^T Sq]

Causal, in time linear in the sequence's length. ``linear_attention`` runs whole sequences
(split into chunks along time where the heads alone would not fill the GPU),
``linear_attention_step`` one token of each, its state in place; a sequence may change
between the two at any token. ``linear_attention_backward`` holds each product's other
operand at its mean, as the attention layer's backward does.

Operands are (B, T, H, D) (a step's (B, H, D)) with any strides but the last dim's, which
is 1: heads are read in place from a side-by-side projection buffer. A mean and its variance
share strides; other layouts are copied. D is at most 128, B H below 2^22. ``decay`` (H,) is meant to lie
in [0, 1]; it is not checked, as that would wait for the GPU.
"""

from __future__ import annotations

import math

import torch
from torch import Tensor

from .. import _lib


def _pair(m: Tensor, S: Tensor, name: str, ref: Tensor, shape) -> tuple[Tensor, Tensor]:
    """A mean and its variance in one layout with a unit last stride."""
    if (isinstance(m, Tensor) and isinstance(S, Tensor) and m.dtype is torch.float32 and S.dtype is torch.float32
            and m.get_device() == ref.get_device() == S.get_device() and m.shape == shape == S.shape):
        st = m.stride()
        if st == S.stride() and (st[-1] == 1 or shape[-1] == 1):
            return m, S
    _lib.check_with(m, "m" + name, ref, shape)
    _lib.check_with(S, "S" + name, ref, shape)
    if m.stride() != S.stride() or (m.stride(-1) != 1 and m.shape[-1] != 1):
        m, S = m.contiguous(), S.contiguous()
    return m, S


def _mean(m: Tensor, name: str, ref: Tensor, shape) -> Tensor:
    _lib.check_with(m, "m" + name, ref, shape)
    return m if m.stride(-1) == 1 or m.shape[-1] == 1 else m.contiguous()


def _heads(t: Tensor) -> _lib.Heads:
    st = t.stride()
    return _lib.Heads(st[0], st[1], st[2]) if t.dim() == 4 else _lib.Heads(st[0], 0, st[1])


def _shape(t: Tensor, dims: int) -> torch.Size:
    _lib.check(t, "mq", contiguous=False)
    if t.dim() != dims or min(t.shape[-2:]) == 0:
        what = "(B, T, H, D)" if dims == 4 else "(B, H, D)"
        raise ValueError(f"mq: expected {what} with heads and features, got {tuple(t.shape)}")
    return t.shape


def _decay(decay: Tensor, ref: Tensor, H: int) -> Tensor:
    return _lib.dense_with(decay, "decay", ref, (H,))


def _scale(scale: float) -> float:
    scale = float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    return scale


def _lengths(lengths: Tensor | None, ref: Tensor, B: int) -> tuple[Tensor | None, int]:
    if lengths is None:
        return None, 0
    if not isinstance(lengths, torch.Tensor) or lengths.dtype not in (torch.int32, torch.int64):
        raise TypeError("lengths: expected an int32 or int64 tensor")
    if lengths.device != ref.device or tuple(lengths.shape) != (B,):
        raise ValueError(f"lengths: expected ({B},) on {ref.device}, got {tuple(lengths.shape)} on {lengths.device}")
    return lengths.contiguous(), lengths.element_size()


def _state(state, ref: Tensor, shape) -> tuple[Tensor, Tensor]:
    try:
        M, P = state
    except (TypeError, ValueError):
        raise TypeError("state: expected a pair of tensors (means, variances)") from None
    return _lib.check_with(M, "state means", ref, shape), _lib.check_with(P, "state variances", ref, shape)


def linear_attention(mq: Tensor, Sq: Tensor, mk: Tensor, Sk: Tensor, mv: Tensor, Sv: Tensor, decay: Tensor,
                     scale: float = 1.0, lengths: Tensor | None = None, state=None, return_state: bool = False):
    """(mo, So), each (B, T, H, D); with ``return_state`` also the state after each
    sequence's last token, (M, P) each (B, H, D, D).

    ``lengths`` (B,): tokens from there on add nothing, are not read, and get zeros; values
    outside [0, T] count as the nearer end. ``state``: where the sequences start from
    (zeros by default); it is not written."""
    shape = _shape(mq, 4)
    B, T, H, D = shape
    mq, Sq = _pair(mq, Sq, "q", mq, shape)
    mk, Sk = _pair(mk, Sk, "k", mq, shape)
    mv, Sv = _pair(mv, Sv, "v", mq, shape)
    decay, scale = _decay(decay, mq, H), _scale(scale)
    lengths, len_bytes = _lengths(lengths, mq, B)
    M0 = P0 = M = P = None
    if state is not None:
        M0, P0 = (t.contiguous() for t in _state(state, mq, (B, H, D, D)))
    mo = torch.empty(shape, device=mq.device, dtype=torch.float32)
    So = torch.empty_like(mo)
    if return_state:
        M = torch.empty((B, H, D, D), device=mq.device, dtype=torch.float32)
        P = torch.empty_like(M)
    ws = _lib.workspace(_lib.query("tagi_linear_attention_fwd_ws_bytes", B, T, H, D), mq.device)
    wp, wb = _lib.ws_args(ws)
    _lib.call_on(mq, "tagi_linear_attention_fwd", mq.data_ptr(), Sq.data_ptr(), mk.data_ptr(), Sk.data_ptr(),
                 mv.data_ptr(), Sv.data_ptr(), _heads(mq), _heads(mk), _heads(mv), decay.data_ptr(),
                 _lib.ptr(lengths), len_bytes, _lib.ptr(M0), _lib.ptr(P0), mo.data_ptr(), So.data_ptr(), _heads(mo),
                 _lib.ptr(M), _lib.ptr(P), B, T, H, D, scale, wp, wb, _lib.stream_of(mq))
    return (mo, So, (M, P)) if return_state else (mo, So)


def linear_attention_backward_packed(mq: Tensor, mk: Tensor, mv: Tensor, delta_mo: Tensor, delta_So: Tensor,
                                     decay: Tensor, scale: float = 1.0,
                                     lengths: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """The deltas of ``linear_attention_backward`` side by side: means and variances, each
    (B, T, 3, H, D) with queries, keys and values in this order."""
    shape = _shape(mq, 4)
    B, T, H, D = shape
    mq, mk, mv = _mean(mq, "q", mq, shape), _mean(mk, "k", mq, shape), _mean(mv, "v", mq, shape)
    dm, dS = _pair(delta_mo, delta_So, "o (delta)", mq, shape)
    decay, scale = _decay(decay, mq, H), _scale(scale)
    lengths, len_bytes = _lengths(lengths, mq, B)
    om = torch.empty((B, T, 3, H, D), device=mq.device, dtype=torch.float32)
    oS = torch.empty_like(om)
    pm, pS = ([t.data_ptr() + i * H * D * 4 for i in range(3)] for t in (om, oS))
    ws = _lib.workspace(_lib.query("tagi_linear_attention_bwd_ws_bytes", B, T, H, D), mq.device)
    wp, wb = _lib.ws_args(ws)
    _lib.call_on(mq, "tagi_linear_attention_bwd", mq.data_ptr(), mk.data_ptr(), mv.data_ptr(), _heads(mq), _heads(mk),
                 _heads(mv), dm.data_ptr(), dS.data_ptr(), _heads(dm), decay.data_ptr(), _lib.ptr(lengths), len_bytes,
                 pm[0], pS[0], pm[1], pS[1], pm[2], pS[2], _lib.Heads(T * 3 * H * D, 3 * H * D, D), B, T, H, D, scale,
                 wp, wb, _lib.stream_of(mq))
    return om, oS


def linear_attention_backward(mq: Tensor, mk: Tensor, mv: Tensor, delta_mo: Tensor, delta_So: Tensor, decay: Tensor,
                              scale: float = 1.0, lengths: Tensor | None = None) -> tuple[Tensor, ...]:
    """(dmq, dSq, dmk, dSk, dmv, dSv) of a ``linear_attention`` that started from zeros.

        dq = M_t d, dSq = (M_t.M_t) e;   dk = G_t v, dSk = N_t (v^2);   dv = G_t^T k, dSv = N_t^T (k^2)
        G_t = g G_{t+1} + q d^T,  N_t = g^2 N_{t+1} + (q^2) e^T,  d = c delta_mo,  e = c^2 delta_So

    Tokens from ``lengths`` on get zeros, and their deltas are not read."""
    om, oS = linear_attention_backward_packed(mq, mk, mv, delta_mo, delta_So, decay, scale, lengths)
    return tuple(t[:, :, i] for i in range(3) for t in (om, oS))


def linear_attention_step(mq: Tensor, Sq: Tensor, mk: Tensor, Sk: Tensor, mv: Tensor, Sv: Tensor, state,
                          decay: Tensor, scale: float = 1.0, active: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """(mo, So), each (B, H, D), of one token of every sequence. ``state`` (M, P), each
    (B, H, D, D) and contiguous, is advanced in place. ``active`` (B,), bool or uint8: a
    sequence that is off keeps its state and gets zeros."""
    shape = _shape(mq, 3)
    B, H, D = shape
    mq, Sq = _pair(mq, Sq, "q", mq, shape)
    mk, Sk = _pair(mk, Sk, "k", mq, shape)
    mv, Sv = _pair(mv, Sv, "v", mq, shape)
    decay, scale = _decay(decay, mq, H), _scale(scale)
    M, P = _state(state, mq, (B, H, D, D))
    _lib.check_in_place(M, "state means"), _lib.check_in_place(P, "state variances")
    if _lib.overlap(M, P):
        raise ValueError("state: means and variances share memory")
    if active is not None:
        if not isinstance(active, torch.Tensor) or active.dtype not in (torch.bool, torch.uint8):
            raise TypeError("active: expected a bool or uint8 tensor")
        if active.device != mq.device or tuple(active.shape) != (B,):
            raise ValueError(f"active: expected ({B},) on {mq.device}, got {tuple(active.shape)} on {active.device}")
        active = active.contiguous()
    mo = torch.empty(shape, device=mq.device, dtype=torch.float32)
    So = torch.empty_like(mo)
    _lib.call_on(mq, "tagi_linear_attention_step", mq.data_ptr(), Sq.data_ptr(), mk.data_ptr(), Sk.data_ptr(),
                 mv.data_ptr(), Sv.data_ptr(), _heads(mq), _heads(mk), _heads(mv), decay.data_ptr(), _lib.ptr(active),
                 M.data_ptr(), P.data_ptr(), mo.data_ptr(), So.data_ptr(), _heads(mo), B, H, D, scale,
                 _lib.stream_of(mq))
    return mo, So
