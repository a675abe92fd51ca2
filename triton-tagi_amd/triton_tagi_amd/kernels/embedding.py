"""Scaled embedding lookup and the table's deltas by sorted tokens.

    embedding_lookup:       mz = c mw[id],  Sz = c^2 Sw[id]
    embedding_param_deltas: dmw[v] = c Sw[v] sum_{id = v} dmz,  dSw[v] = (c Sw[v])^2 sum_{id = v} dSz
    embedding_update:       those deltas with the capped update, applied to the rows that occur

``ids`` holds whole numbers as float32 (what the Embedding layer takes, cast toward zero),
int32 or int64, in any shape. Ids equal to ``padding_idx`` or outside the table look up
zeros and add nothing. The tokens are sorted by id on the GPU and every row's sum runs over
its own tokens: the cost follows the tokens, not tokens times categories.
"""

from __future__ import annotations

import math

import torch
from torch import Tensor

from .. import _lib

_ID_TYPES = {torch.float32: 0, torch.int32: 1, torch.int64: 2}


def _check_ids(ids: Tensor, ref: Tensor) -> tuple[Tensor, int]:
    if not isinstance(ids, torch.Tensor):
        raise TypeError(f"ids: expected a torch.Tensor, got {type(ids).__name__}")
    kind = _ID_TYPES.get(ids.dtype)
    if kind is None:
        raise TypeError(f"ids: expected float32, int32 or int64, got {ids.dtype}")
    if ids.get_device() != ref.get_device():
        raise ValueError(f"ids: tensor is on {ids.device}, the table on {ref.device}")
    return ids.contiguous(), kind


def _check_table(t: Tensor, name: str) -> Tensor:
    _lib.check(t, name, contiguous=False)
    if t.dim() != 2 or t.numel() == 0:
        raise ValueError(f"{name}: expected a (categories, features) table, got {tuple(t.shape)}")
    return t


def _check_scale(scale: float) -> float:
    scale = float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    return scale


def _check_deltas(ids: Tensor, delta_mz: Tensor, delta_Sz: Tensor, ref: Tensor) -> tuple[Tensor, Tensor]:
    D = ref.shape[1]
    out = []
    for t, name in ((delta_mz, "delta_mz"), (delta_Sz, "delta_Sz")):
        _lib.check_with(t, name, ref)
        if t.numel() != ids.numel() * D or (t.dim() and t.shape[-1] != D):
            raise ValueError(f"{name}: expected {tuple(ids.shape)} ids x {D} features, got {tuple(t.shape)}")
        out.append(t.contiguous())
    return out[0], out[1]


def embedding_lookup(ids: Tensor, mw: Tensor, Sw: Tensor, scale: float = 1.0,
                     padding_idx: int = -1) -> tuple[Tensor, Tensor]:
    """Moments (*ids.shape, D) of the rows ``ids`` of the table (mw, Sw), scaled."""
    mw = _check_table(mw, "mw").contiguous()
    Sw = _lib.dense_with(Sw, "Sw", mw, mw.shape)
    ids, kind = _check_ids(ids, mw)
    scale = _check_scale(scale)
    V, D = mw.shape
    mz = torch.empty((*ids.shape, D), device=mw.device, dtype=torch.float32)
    Sz = torch.empty_like(mz)
    _lib.call_on(mw, "tagi_embedding_scaled_fwd", ids.data_ptr(), kind, mw.data_ptr(), Sw.data_ptr(), mz.data_ptr(),
                 Sz.data_ptr(), ids.numel(), V, D, int(padding_idx), scale, _lib.stream_of(mw))
    return mz, Sz


def _workspace(n: int, V: int, D: int, dev) -> tuple:
    ws = _lib.workspace(_lib.query("tagi_embedding_sorted_ws_bytes", n, V, D), dev)
    return (ws, *_lib.ws_args(ws))


def embedding_param_deltas(ids: Tensor, delta_mz: Tensor, delta_Sz: Tensor, Sw: Tensor, scale: float = 1.0,
                           padding_idx: int = -1) -> tuple[Tensor, Tensor]:
    """Parameter deltas (V, D) from the deltas at the lookup's output; zeros for rows that
    do not occur. Deterministic."""
    Sw = _check_table(Sw, "Sw").contiguous()
    ids, kind = _check_ids(ids, Sw)
    scale = _check_scale(scale)
    dm, dS = _check_deltas(ids, delta_mz, delta_Sz, Sw)
    n, (V, D) = ids.numel(), Sw.shape
    dmw, dSw = torch.empty_like(Sw), torch.empty_like(Sw)
    ws, wp, wb = _workspace(n, V, D, Sw.device)
    _lib.call_on(Sw, "tagi_embedding_sorted_bwd", ids.data_ptr(), kind, dm.data_ptr(), dS.data_ptr(), Sw.data_ptr(),
                 dmw.data_ptr(), dSw.data_ptr(), n, V, D, int(padding_idx), scale, wp, wb, _lib.stream_of(Sw))
    return dmw, dSw


def embedding_update(ids: Tensor, delta_mz: Tensor, delta_Sz: Tensor, mw: Tensor, Sw: Tensor, cap_factor: float,
                     scale: float = 1.0, padding_idx: int = -1,
                     keep_deltas: bool = False) -> tuple[Tensor, Tensor] | tuple[None, None]:
    """``embedding_param_deltas`` followed by ``update_parameters`` on (mw, Sw) in place, the
    same bits for a table of positive variances: rows that do not occur have no deltas and
    are neither read nor written. Returns the deltas with ``keep_deltas``, else (None, None)."""
    _check_table(mw, "mw")
    _lib.check_with(Sw, "Sw", mw, mw.shape)
    _lib.check_in_place(mw, "mw"), _lib.check_in_place(Sw, "Sw")
    if _lib.overlap(mw, Sw):
        raise ValueError("mw and Sw share memory")
    cap = float(cap_factor)
    if not 0.0 < cap <= 3.4e38:
        raise ValueError(f"cap_factor must be positive and finite, got {cap_factor}")
    ids, kind = _check_ids(ids, mw)
    scale = _check_scale(scale)
    dm, dS = _check_deltas(ids, delta_mz, delta_Sz, mw)
    n, (V, D) = ids.numel(), mw.shape
    dmw, dSw = (torch.empty_like(mw), torch.empty_like(Sw)) if keep_deltas else (None, None)
    ws, wp, wb = _workspace(n, V, D, mw.device)
    _lib.call_on(mw, "tagi_embedding_sorted_bwd_update", ids.data_ptr(), kind, dm.data_ptr(), dS.data_ptr(),
                 mw.data_ptr(), Sw.data_ptr(), _lib.ptr(dmw), _lib.ptr(dSw), cap, n, V, D, int(padding_idx), scale,
                 wp, wb, _lib.stream_of(mw))
    return dmw, dSw
