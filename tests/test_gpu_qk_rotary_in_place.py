"""The backward of norms and rotation over its own deltas: the same bits, and no buffers beside them."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("normed", [True, False])
@pytest.mark.parametrize("B,T,H,G,D,pairs,interleaved", [
    (2, 33, 4, 2, 128, 64, False),
    (3, 7, 6, 3, 80, 33, True),
    (1, 130, 3, 1, 80, 24, False),
    (2, 19, 2, 2, 21, 9, False),
    (2, 5, 1, 1, 7, 3, True),
    (1, 64, 8, 8, 32, 0, False),
])
def test_in_place(B, T, H, G, D, pairs, interleaved, normed, dev):
    from triton_tagi_amd import kernels as K
    from triton_tagi_amd.kernels.rotary import qk_norm_rotary_backward_into

    r = torch.Generator(device=dev).manual_seed(D + T)
    new = lambda *s: torch.randn(*s, generator=r, device=dev)  # noqa: E731
    q, k = (new(B, T, H, D), new(B, T, H, D).abs()), (new(B, T, G, D), new(B, T, G, D).abs())
    kw = {}
    if pairs:
        kw = dict(positions=torch.randint(0, 9999, (B, T), generator=r, device=dev),
                  frequencies=K.rotary_frequencies(pairs, device=dev), interleaved=interleaved)
    w = tuple(new(D).abs() for _ in range(4)) if normed else None
    inv = K.qk_norm_rotary(*q, *k, weights=w, **kw)[4]
    # deltas side by side in one buffer with a third part, as the layer has them
    d = [new(B, T, H + 2 * G, D) for _ in range(2)]
    dq, dk = ([t[:, :, a:b] for t in d] for a, b in ((0, H), (H, H + G)))
    rest = [t[:, :, H + G:].clone() for t in d]
    want = K.qk_norm_rotary_backward(*dq, *dk, q[0], k[0], inv, weights=w, **kw)
    dw = qk_norm_rotary_backward_into((*dq, *dk), *dq, *dk, q[0], k[0], inv, weights=w, **kw)
    for a, b in zip((*dq, *dk, *dw), want):
        assert torch.equal(a, b)
    for a, b in zip(d, rest):
        assert torch.equal(a[:, :, H + G:], b)


def test_the_layers_backward_has_one_set_of_deltas(dev):
    from triton_tagi_amd import RemaxAttention, _lib

    E, H, G, B, T = 512, 8, 2, 8, 1024
    D = E // H
    layer = RemaxAttention(E, H, G, device="cuda:0")
    r = torch.Generator(device=dev).manual_seed(1)
    m, S = torch.randn(B, T, E, generator=r, device=dev), torch.rand(B, T, E, generator=r, device=dev)
    out = layer.forward(m, S)
    layer.backward(m, S)  # parameters' deltas and whatever is allocated once
    layer.forward(m, S)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    layer.backward(m, S)
    peak = torch.cuda.max_memory_allocated() - before
    deltas = 4 * B * T * D * 2 * (H + 2 * G)
    ws = _lib.query("tagi_remax_attention_bwd_ws_bytes", B, T, T, H, G, D)
    inputs = 4 * B * T * E * 2
    # the projections' products: a second set of their parameters' deltas, and room to split them
    weights = 8 * 4 * E * (H + 2 * G) * D
    assert peak <= deltas + max(ws, inputs) + weights + inputs // 4
    assert out is not None
