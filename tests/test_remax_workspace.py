"""Workspaces of attention over long sequences: in proportion to the length, not to its square."""

from __future__ import annotations

import pytest


def most(name, B, T, H, G, D):
    """Sums of 8192 blocks of 128 rows or keys, and of each row and key once more (a last split's)."""
    if "fwd" in name:  # a row's two outputs, its weights' sum, two statistics
        return 4 * (2 * D + 3) * (8192 * 128 + B * H * T)
    return 4 * max(2 * D * (8192 * 128 + B * H * T), 4 * D * (8192 * 128 + B * G * T))


@pytest.mark.parametrize("H,G,D", [(32, 8, 128), (16, 4, 64), (8, 8, 96), (4, 1, 32)])
@pytest.mark.parametrize("B", [1, 4])
@pytest.mark.parametrize("name", ["tagi_remax_attention_fwd_ws_bytes", "tagi_remax_attention_bwd_ws_bytes"])
def test_workspace_grows_with_the_length(name, B, H, G, D):
    from triton_tagi_amd import _lib

    size = getattr(_lib.load(), name)
    for T in (1, 100, 1024, 8192, 16384, 32768, 131072):
        assert size(B, T, T, H, G, D) <= most(name, B, T, H, G, D), T


def test_a_long_context_for_few_queries():
    """The parts of a chunk's queries do not grow with the context."""
    from triton_tagi_amd import _lib

    name = "tagi_remax_attention_fwd_ws_bytes"
    assert getattr(_lib.load(), name)(1, 512, 1 << 20, 32, 8, 128) <= most(name, 1, 512, 32, 8, 128)
