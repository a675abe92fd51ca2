"""The decays that LinearAttention hands to its kernels follow its ``decay`` (CPU)."""

from __future__ import annotations

import torch

from triton_tagi_amd import LinearAttention


def test_decays_on_a_device_follow_the_attribute():
    layer = LinearAttention(8, 2, decay=[0.5, 0.25], device="cpu")
    cpu = torch.device("cpu")
    first = layer._decay_on(cpu)
    assert first.tolist() == [0.5, 0.25] and layer._decay_on(cpu) is first
    layer.decay = (0.75, 0.125)
    again = layer._decay_on(cpu)
    assert again.tolist() == [0.75, 0.125]
    assert again.data_ptr() == first.data_ptr()  # recorded graphs go on reading it
    assert layer._decay_on(cpu) is again
