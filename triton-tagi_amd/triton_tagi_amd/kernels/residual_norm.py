"""Sum of two Gaussian streams and its RMSNorm in one pass.

    s = a + r (means and variances add),  inv = 1/sqrt(mean(ms^2 + Ss) + eps)
    mz = ms inv g,  Sz = inv^2 (Ss (g^2 + Sg) + Sg ms^2)

The same moments as ``Add`` followed by ``RMSNorm``, for rows of any length; the sum is
written on the way (the residual stream of the next block, and what the backward reads).
"""

from __future__ import annotations

import torch
from torch import Tensor

from .. import _lib


def _rows(t: Tensor) -> int:
    return t.numel() // t.shape[-1]


def add_rms_norm(ma: Tensor, Sa: Tensor, mr: Tensor, Sr: Tensor, mw: Tensor, Sw: Tensor, eps: float = 1e-6,
                 need_sum_var: bool = True) -> tuple[Tensor, Tensor, Tensor, Tensor | None, Tensor]:
    """(mz, Sz, ms, Ss, inv_rms) of (ma, Sa) + (mr, Sr), rows over the last dim; inv_rms is
    (rows, 1). Ss is None without ``need_sum_var``."""
    _lib.check(ma, "ma", contiguous=False)
    if ma.dim() < 1 or ma.shape[-1] == 0:
        raise ValueError(f"ma: rows must hold at least one feature, got {tuple(ma.shape)}")
    ma = ma.contiguous()
    shape = ma.shape
    D, rows = shape[-1], _rows(ma)
    Sa, mr, Sr = (_lib.dense_with(Sa, "Sa", ma, shape), _lib.dense_with(mr, "mr", ma, shape),
                  _lib.dense_with(Sr, "Sr", ma, shape))
    mw, Sw = _lib.dense_with(mw, "mw", ma, (D,)), _lib.dense_with(Sw, "Sw", ma, (D,))
    mz, Sz, ms = torch.empty_like(ma), torch.empty_like(ma), torch.empty_like(ma)
    Ss = torch.empty_like(ma) if need_sum_var else None
    inv = torch.empty(rows, 1, device=ma.device, dtype=torch.float32)
    _lib.call_on(ma, "tagi_add_rmsnorm_fwd", ma.data_ptr(), Sa.data_ptr(), mr.data_ptr(), Sr.data_ptr(),
                 mw.data_ptr(), Sw.data_ptr(), mz.data_ptr(), Sz.data_ptr(), ms.data_ptr(), _lib.ptr(Ss),
                 inv.data_ptr(), rows, D, float(eps), _lib.stream_of(ma))
    return mz, Sz, ms, Ss, inv


def add_rms_norm_backward(delta_mz: Tensor, delta_Sz: Tensor, ms: Tensor, inv_rms: Tensor, mw: Tensor, Sw: Tensor,
                          delta_ms: Tensor | None = None,
                          delta_Ss: Tensor | None = None) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """(delta_m, delta_S, delta_mw, delta_Sw): the deltas at the sum, which both inputs
    receive, and the gamma deltas. ``delta_ms`` / ``delta_Ss`` are the deltas that reach the
    sum on another way (the residual stream of a following block); both or neither."""
    _lib.check(ms, "ms", contiguous=False)
    if ms.dim() < 1 or ms.shape[-1] == 0:
        raise ValueError(f"ms: rows must hold at least one feature, got {tuple(ms.shape)}")
    if (delta_ms is None) != (delta_Ss is None):
        raise ValueError("delta_ms and delta_Ss must be given together")
    ms = ms.contiguous()
    D, rows = ms.shape[-1], _rows(ms)
    dm, dS = _lib.dense_with(delta_mz, "delta_mz", ms, ms.shape), _lib.dense_with(delta_Sz, "delta_Sz", ms, ms.shape)
    if delta_ms is not None:
        delta_ms = _lib.dense_with(delta_ms, "delta_ms", ms, ms.shape)
        delta_Ss = _lib.dense_with(delta_Ss, "delta_Ss", ms, ms.shape)
    inv = _lib.check_with(inv_rms, "inv_rms", ms).contiguous()
    if inv.numel() != rows:
        raise ValueError(f"inv_rms: expected {rows} rows, got {tuple(inv.shape)}")
    mw, Sw = _lib.dense_with(mw, "mw", ms, (D,)), _lib.dense_with(Sw, "Sw", ms, (D,))
    dma, dSa = torch.empty_like(ms), torch.empty_like(ms)
    dmw, dSw = torch.empty_like(mw), torch.empty_like(mw)
    ws = _lib.workspace(_lib.query("tagi_add_rmsnorm_bwd_ws_bytes", rows, D), ms.device)
    wp, wb = _lib.ws_args(ws)
    _lib.call_on(ms, "tagi_add_rmsnorm_bwd", dm.data_ptr(), dS.data_ptr(), _lib.ptr(delta_ms), _lib.ptr(delta_Ss),
                 ms.data_ptr(), inv.data_ptr(), mw.data_ptr(), Sw.data_ptr(), dma.data_ptr(), dSa.data_ptr(),
                 dmw.data_ptr(), dSw.data_ptr(), rows, D, wp, wb, _lib.stream_of(ms))
    return dma, dSa, dmw, dSw
