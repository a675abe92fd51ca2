"""Cache calls whose last block would reach 2^32 threads are refused before the launch (without a GPU)."""

from __future__ import annotations

import pytest


@pytest.mark.parametrize("heads,head_dim,T", [(3, 4, 1431655765), (3, 8, 715827882), (5, 128, 26843545)])
def test_last_block_beyond_the_launch(heads, head_dim, T):
    from triton_tagi_amd import _lib

    lib = _lib.load()
    lanes = max(1, head_dim // 4)
    assert T * heads < 2**32 // lanes <= -(-T * heads // (256 // lanes)) * (256 // lanes)
    h = _lib.Heads(1, 1, 1)
    c = _lib.KvCache(16, 16, 16, 16, None, 0, 2, heads, 4, head_dim)
    assert lib.tagi_kv_cache_write(c, 16, 16, h, 16, 16, h, 16, 3, None, 0, None, 0, 1, T, None) != 0
    assert "too large" in _lib.last_error(), _lib.last_error()
    assert lib.tagi_kv_cache_read(c, 16, 3, 16, 4, 16, 16, 16, 16, 1, T, None) != 0
    assert "too large" in _lib.last_error(), _lib.last_error()
