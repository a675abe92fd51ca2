"""Attention with Remax scores over sequences of any length, on Gaussian moments.

With the scale c, for a query and the keys j that it sees:

    m_j = c q.k_j,  v_j = c^2 [Sq.(k_j^2 + Sk_j) + q^2.Sk_j]
    (a_j, Sa_j) = Remax of (m_j, v_j) over those keys,  J_j = cov(a_j, z_j) / v_j
    mo = sum a_j v_j,  So = sum Sa_j (v_j^2 + Sv_j) + a_j^2 Sv_j

No score is stored: the backward forms them again. Queries (B, T, H, D), keys and values
(B, N, G, D) with G dividing H: query head h reads key head h // (H // G). Any strides but the last
dim's, which is 1; a mean and its variance share strides; other layouts are copied. D is at most 128.

Query t of sequence b stands at position ``starts[b]`` + t (t without). It sees the keys j <
``lengths[b]`` (all without), with ``causal`` those up to its position. A query at or behind its
sequence's length, or before 0, sees nothing: zeros, and no deltas; such queries and the keys behind
a length may hold anything. A NaN that a query sees makes its outputs NaN; infinities and NaN inside a
sequence may reach any of its queries.

``remax_attention_step`` runs one query of every sequence over the pages of a cache (kv_cache.py).
"""

from __future__ import annotations

import torch
from torch import Tensor

from .. import _lib
from ._operands import counts, dense_like, finite_scale, heads, key_heads, mean, pair, shape_of, written
from .kv_cache import KVCache, cache_struct, check_table


def _sizes(mq: Tensor, mk: Tensor):
    qs = shape_of(mq, "mq", 4)
    ks = shape_of(mk, "mk", 4)
    if ks[0] != qs[0] or ks[3] != qs[3]:
        raise ValueError(f"mk: expected ({qs[0]}, keys, heads, {qs[3]}), got {tuple(ks)}")
    key_heads(ks[2], qs[2])
    if qs[3] > 128:
        raise ValueError(f"remax_attention supports head dimensions up to 128, got {qs[3]}")
    return qs, ks


def remax_attention(mq: Tensor, Sq: Tensor, mk: Tensor, Sk: Tensor, mv: Tensor, Sv: Tensor, scale: float = 1.0,
                    causal: bool = True, lengths: Tensor | None = None, starts: Tensor | None = None,
                    return_rows: bool = False):
    """(mo, So), each (B, T, H, D); with ``return_rows`` also the rows' sums (3, B, H, T), which
    ``remax_attention_backward`` reads."""
    qs, ks = _sizes(mq, mk)
    B, T, H, D = qs
    N, G = ks[1:3]
    mq, Sq = pair(mq, Sq, "q", mq, qs)
    mk, Sk = pair(mk, Sk, "k", mq, ks)
    mv, Sv = pair(mv, Sv, "v", mq, ks)
    scale = finite_scale(scale)
    lengths, len_bytes = counts(lengths, "lengths", mq, B)
    starts, start_bytes = counts(starts, "starts", mq, B)
    mo = dense_like(mq, qs)
    So = torch.empty_like(mo)
    rows = mq.new_empty((3, B, H, T))
    ws = _lib.workspace(_lib.query("tagi_remax_attention_fwd_ws_bytes", B, T, N, H, G, D), mq.device)
    wp, wb = _lib.ws_args(ws)
    _lib.call_on(mq, "tagi_remax_attention_fwd", mq.data_ptr(), Sq.data_ptr(), heads(mq), mk.data_ptr(), Sk.data_ptr(),
                 heads(mk), mv.data_ptr(), Sv.data_ptr(), heads(mv), _lib.ptr(lengths), len_bytes, _lib.ptr(starts),
                 start_bytes, int(causal), mo.data_ptr(), So.data_ptr(), rows.data_ptr(), B, T, N, H, G, D, scale, wp,
                 wb, _lib.stream_of(mq))
    return (mo, So, rows) if return_rows else (mo, So)


def remax_attention_backward(mq: Tensor, Sq: Tensor, mk: Tensor, Sk: Tensor, mv: Tensor, delta_mo: Tensor,
                             delta_So: Tensor, rows: Tensor, scale: float = 1.0, causal: bool = True,
                             lengths: Tensor | None = None, starts: Tensor | None = None) -> tuple[Tensor, ...]:
    """(dmq, dSq, dmk, dSk, dmv, dSv), each product's other operand held at its mean:

        e = c J (dm v^T),  E = c^2 J^2 (dS (v^2)^T)
        dq = e k, dSq = E k^2;  dk = e^T q, dSk = E^T q^2;  dv = a^T dm, dSv = (a^2)^T dS

    ``rows``: of a ``remax_attention`` of the same operands. Keys' deltas are summed over the query
    heads that share them."""
    dmq, dmk = (dense_like(t, t.shape) for t in (mq, mk))
    out = (dmq, torch.empty_like(dmq), dmk, *(torch.empty_like(dmk) for _ in range(3)))
    _backward(out, mq, Sq, mk, Sk, mv, delta_mo, delta_So, rows, scale, causal, lengths, starts)
    return out


def remax_attention_backward_into(out, mq: Tensor, Sq: Tensor, mk: Tensor, Sk: Tensor, mv: Tensor, delta_mo: Tensor,
                                  delta_So: Tensor, rows: Tensor, scale: float = 1.0, causal: bool = True,
                                  lengths: Tensor | None = None, starts: Tensor | None = None) -> None:
    """``remax_attention_backward`` into six tensors: the queries' two in one layout, the keys' and
    values' four in one, unit last strides."""
    qs, ks = _sizes(mq, mk)
    dmq, dSq, dmk, dSk, dmv, dSv = out
    written((dmq, dSq), ("dmq", "dSq"), mq, qs)
    written((dmk, dSk, dmv, dSv), ("dmk", "dSk", "dmv", "dSv"), mq, ks)
    _backward(out, mq, Sq, mk, Sk, mv, delta_mo, delta_So, rows, scale, causal, lengths, starts)


def _backward(out, mq: Tensor, Sq: Tensor, mk: Tensor, Sk: Tensor, mv: Tensor, delta_mo: Tensor, delta_So: Tensor,
              rows: Tensor, scale: float, causal: bool, lengths: Tensor | None, starts: Tensor | None) -> None:
    qs, ks = _sizes(mq, mk)
    B, T, H, D = qs
    N, G = ks[1:3]
    mq, Sq = pair(mq, Sq, "q", mq, qs)
    mk, Sk = pair(mk, Sk, "k", mq, ks)
    mv = mean(mv, "v", mq, ks)
    dm, dS = pair(delta_mo, delta_So, "o (delta)", mq, qs)
    rows = _lib.dense_with(rows, "rows", mq, (3, B, H, T))
    scale = finite_scale(scale)
    lengths, len_bytes = counts(lengths, "lengths", mq, B)
    starts, start_bytes = counts(starts, "starts", mq, B)
    ws = _lib.workspace(_lib.query("tagi_remax_attention_bwd_ws_bytes", B, T, N, H, G, D), mq.device)
    wp, wb = _lib.ws_args(ws)
    p = [t.data_ptr() for t in out]
    _lib.call_on(mq, "tagi_remax_attention_bwd", mq.data_ptr(), Sq.data_ptr(), heads(mq), mk.data_ptr(), Sk.data_ptr(),
                 heads(mk), mv.data_ptr(), heads(mv), dm.data_ptr(), dS.data_ptr(), heads(dm), rows.data_ptr(),
                 _lib.ptr(lengths), len_bytes, _lib.ptr(starts), start_bytes, int(causal), p[0], p[1],
                 heads(out[0]), p[2], p[3], p[4], p[5], heads(out[2]), B, T, N, H, G, D, scale, wp, wb, _lib.stream_of(mq))


def remax_attention_step(mq: Tensor, Sq: Tensor, cache: KVCache, table: Tensor, lengths: Tensor, scale: float = 1.0,
                         max_len: int | None = None) -> tuple[Tensor, Tensor]:
    """(mo, So), each (B, H, D), of one query of every sequence over the first ``lengths[b]`` tokens
    of its pages (its own token written before; a sequence of none gets zeros). ``max_len``: no
    length is above it (longer ones count as it); the table's room without. A bound near the lengths
    splits the work better."""
    shape = shape_of(mq, "mq", 3)
    B, H, D = shape
    mq, Sq = pair(mq, Sq, "q", mq, shape)
    c = cache_struct(cache, mq)
    if c.head_dim != D:
        raise ValueError(f"cache: holds heads of {c.head_dim}, got {D}")
    key_heads(c.heads, H)
    table = check_table(table, mq, B)
    scale = finite_scale(scale)
    if lengths is None:
        raise TypeError("lengths: expected an int32 or int64 tensor")
    lengths, len_bytes = counts(lengths, "lengths", mq, B)
    room = table.shape[1] * c.page_size
    most = room if max_len is None else min(int(max_len), room)
    if most < 0:
        raise ValueError(f"max_len must not be negative, got {max_len}")
    mo = dense_like(mq, shape)
    So = torch.empty_like(mo)
    ws = _lib.workspace(_lib.query("tagi_remax_attention_step_ws_bytes", B, H, c.heads, D, most), mq.device)
    wp, wb = _lib.ws_args(ws)
    _lib.call_on(mq, "tagi_remax_attention_step", mq.data_ptr(), Sq.data_ptr(), heads(mq), c, table.data_ptr(),
                 table.shape[1], lengths.data_ptr(), len_bytes, mo.data_ptr(), So.data_ptr(), B, H, most, scale, wp, wb,
                 _lib.stream_of(mq))
    return mo, So
