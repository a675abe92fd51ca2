"""Outputs that a caller hands to the backward forms: what the kernels would write elsewhere, or twice, is
refused before any launch. The tensors lie on the CPU and are said to lie on a GPU."""

from __future__ import annotations

import pytest
import torch


class OnGpu(torch.Tensor):
    """A CPU tensor that passes for one of cuda:0 where arguments are checked."""

    @property
    def is_cuda(self):
        return True

    def get_device(self):
        return 0


def gpu(*shape):
    return torch.zeros(*shape).as_subclass(OnGpu)


B, T, H, G, D = 2, 5, 4, 2, 8


def bad_outputs():
    q, k = (B, T, H, D), (B, T, G, D)
    yield "shape", (gpu(B, T, G, D), gpu(*q)), (gpu(*k), gpu(*k))
    yield "shape", (gpu(*q), gpu(*q)), (gpu(B, T - 1, G, D), gpu(*k))
    yield "layout", (gpu(*q), gpu(B, H, T, D).transpose(1, 2)), (gpu(*k), gpu(*k))
    yield "layout", (gpu(*q), gpu(*q)), tuple(gpu(B, T, D, G).transpose(2, 3) for _ in range(2))
    yield "share", tuple(gpu(B, 1, H, D).expand(q) for _ in range(2)), (gpu(*k), gpu(*k))
    yield "float32", (gpu(*q).double(), gpu(*q)), (gpu(*k), gpu(*k))
    yield "GPU only", (torch.zeros(q), gpu(*q)), (gpu(*k), gpu(*k))


@pytest.mark.parametrize("case", range(7))
def test_outputs_refused(case, monkeypatch):
    from triton_tagi_amd import _lib
    from triton_tagi_amd.kernels.remax_attention import remax_attention_backward_into
    from triton_tagi_amd.kernels.rotary import qk_norm_rotary_backward_into

    monkeypatch.setattr(_lib, "call_on", lambda *a: pytest.fail("launched"))
    monkeypatch.setattr(_lib, "stream_of", lambda t: 0)
    what, oq, ok = list(bad_outputs())[case]
    q, k = gpu(B, T, H, D), gpu(B, T, G, D)
    with pytest.raises((ValueError, TypeError), match=what):
        remax_attention_backward_into((*oq, *ok, *ok), q, q, k, k, k, q, q, gpu(3, B, H, T))
    with pytest.raises((ValueError, TypeError), match=what):
        qk_norm_rotary_backward_into((*oq, *ok), q, q, k, k, q, k, None)


def test_outputs_taken(monkeypatch):
    """Side by side in one buffer, as the layer has them."""
    from triton_tagi_amd import _lib
    from triton_tagi_amd.kernels.remax_attention import remax_attention_backward_into
    from triton_tagi_amd.kernels.rotary import qk_norm_rotary_backward_into

    calls = []
    monkeypatch.setattr(_lib, "call_on", lambda t, name, *a: calls.append(name))
    monkeypatch.setattr(_lib, "stream_of", lambda t: 0)
    monkeypatch.setattr(_lib, "workspace", lambda n, device: None)
    dm, dS = gpu(B, T, H + 2 * G, D), gpu(B, T, H + 2 * G, D)
    oq, ok, ov = ((dm[:, :, a:b], dS[:, :, a:b]) for a, b in ((0, H), (H, H + G), (H + G, H + 2 * G)))
    q, k = gpu(B, T, H, D), gpu(B, T, G, D)
    remax_attention_backward_into((*oq, *ok, *ov), q, q, k, k, k, q, q, gpu(3, B, H, T))
    qk_norm_rotary_backward_into((*oq, *ok), q, q, k, k, q, k, None)
    assert calls == ["tagi_remax_attention_bwd", "tagi_qk_rotary_bwd"]
