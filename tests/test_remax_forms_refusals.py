"""Arguments of the cache's entry points that no kernel takes (without a GPU)."""

from __future__ import annotations

import pytest


@pytest.mark.parametrize("kw,T,match", [
    (dict(type=2, scales=2), 2, "aligned"),
    (dict(heads=1 << 19), 1 << 14, "too large"),
    (dict(head_dim=128), 1 << 27, "too large"),
])
def test_cache_writes_refused(kw, T, match):
    from triton_tagi_amd import _lib

    lib = _lib.load()
    h = _lib.Heads(1, 1, 1)
    shape = dict(type=0, pages=2, heads=1, page_size=4, head_dim=8, scales=None)
    c = _lib.KvCache(16, 16, 16, 16, **{**shape, **kw})
    assert lib.tagi_kv_cache_write(c, 16, 16, h, 16, 16, h, 16, 3, None, 0, None, 0, 1, T, None) != 0
    assert match in _lib.last_error(), _lib.last_error()
