"""Argument checks of the sequence-model operators that need no GPU."""

from __future__ import annotations

import pytest
import torch


def test_cpu_tensors_are_refused():
    from triton_tagi_amd import kernels as K

    t, w, q = torch.zeros(4, 3), torch.zeros(3), torch.zeros(1, 2, 1, 3)
    for call in (lambda: K.embedding_lookup(torch.zeros(2), t, t),
                 lambda: K.embedding_param_deltas(torch.zeros(2), t[:2], t[:2], t),
                 lambda: K.embedding_update(torch.zeros(2), t[:2], t[:2], t, t.clone(), 2.0),
                 lambda: K.add_rms_norm(t, t, t, t, w, w),
                 lambda: K.add_rms_norm_backward(t, t, t, torch.zeros(4, 1), w, w),
                 lambda: K.linear_attention(q, q, q, q, q, q, torch.zeros(1)),
                 lambda: K.linear_attention_backward(q, q, q, q, q, torch.zeros(1)),
                 lambda: K.linear_attention_step(*([q[:, 0]] * 6), (torch.zeros(1, 1, 3, 3),) * 2, torch.zeros(1))):
        with pytest.raises(ValueError, match="GPU only"):
            call()


def test_library_argument_errors():
    from triton_tagi_amd import _lib

    lib = _lib.load()
    h = _lib.Heads(1, 1, 1)

    def err(name, *args, match):
        assert getattr(lib, name)(*args) != 0, name
        assert match in _lib.last_error(), _lib.last_error()

    err("tagi_embedding_scaled_fwd", 1, 7, 1, 1, 1, 1, 4, 4, 4, -1, 1.0, None, match="id type")
    err("tagi_embedding_scaled_fwd", None, 0, 1, 1, 1, 1, 4, 4, 4, -1, 1.0, None, match="null pointer")
    err("tagi_embedding_scaled_fwd", 1, 0, 1, 1, 1, 1, 4, 0, 4, -1, 1.0, None, match="bad sizes")
    err("tagi_embedding_scaled_fwd", 1, 0, 1, 1, 1, 1, 1 << 31, 4, 4, -1, 1.0, None, match="too large")
    assert lib.tagi_embedding_scaled_fwd(None, 0, None, None, None, None, 0, 4, 4, -1, 1.0, None) == 0
    need = lib.tagi_embedding_sorted_ws_bytes(100, 50, 8)
    assert need > 0 and lib.tagi_embedding_sorted_ws_bytes(0, 50, 8) == 0
    err("tagi_embedding_sorted_bwd", 1, 0, 1, 1, 1, 1, 1, 100, 50, 8, -1, 1.0, 1, need - 1, None, match="workspace")
    err("tagi_embedding_sorted_bwd", 1, 0, 1, 1, 1, None, None, 100, 50, 8, -1, 1.0, 1, need, None, match="null pointer")
    err("tagi_embedding_sorted_bwd_update", 1, 0, 1, 1, 1, 1, 1, None, 2.0, 100, 50, 8, -1, 1.0, 1, need, None,
        match="null pointer")
    err("tagi_embedding_sorted_bwd_update", 1, 0, 1, 1, 1, 1, None, None, 0.0, 100, 50, 8, -1, 1.0, 1, need, None,
        match="cap_factor")
    err("tagi_add_rmsnorm_fwd", *([None] * 11), 4, 8, 1e-6, None, match="null pointer")
    err("tagi_add_rmsnorm_fwd", *([1] * 11), 4, 0, 1e-6, None, match="bad sizes")
    assert lib.tagi_add_rmsnorm_fwd(*([None] * 11), 0, 8, 1e-6, None) == 0
    err("tagi_add_rmsnorm_bwd", 1, 1, 1, None, *([1] * 8), 4, 8, 1, 1 << 20, None, match="together")
    err("tagi_add_rmsnorm_bwd", *([1] * 12), 4, 8, 1, 0, None, match="workspace")
    fwd = lambda B, T, H, D, lens=None, lb=0, i=None, e=(None, None): (  # noqa: E731
        *([1] * 6), h, h, h, 1, lens, lb, i, None, 1, 1, h, *e, B, T, H, D, 1.0, None, 0, None)
    err("tagi_linear_attention_fwd", *fwd(1, 4, 1, 129), match="head dimension")
    err("tagi_linear_attention_fwd", *fwd(1, 4, 0, 8), match="bad sizes")
    err("tagi_linear_attention_fwd", *fwd(1, 4, 1, 8, lens=1, lb=2), match="lengths")
    err("tagi_linear_attention_fwd", *fwd(1, 4, 1, 8, i=1), match="state")
    err("tagi_linear_attention_fwd", *fwd(1, 4, 1, 8, e=(1, None)), match="state")
    err("tagi_linear_attention_fwd", *fwd(1 << 20, 4, 1 << 20, 8), match="too large")
    err("tagi_linear_attention_fwd", *fwd(1 << 21, 4, 2, 8), match="too large")
    err("tagi_linear_attention_step", *([None] * 6), h, h, h, *([None] * 6), h, 1 << 21, 2, 8, 1.0, None,
        match="too large")
    err("tagi_embedding_sorted_bwd", 1, 0, 1, 1, 1, 1, 1, 1 << 30, 50, 8, -1, 1.0, 1, 1 << 50, None, match="too large")
    assert lib.tagi_linear_attention_fwd(*fwd(0, 4, 1, 8)) == 0
    err("tagi_linear_attention_bwd", *([None] * 3), h, h, h, None, None, h, None, None, 0, *([None] * 6), h, 1, 4, 1, 8,
        1.0, None, 0, None, match="null pointer")
    err("tagi_linear_attention_step", *([None] * 6), h, h, h, *([None] * 6), h, 1, 1, 8, 1.0, None, match="null pointer")


def test_token_counts_at_the_limit_of_a_launch():
    """2^30 - 64 tokens are the most whose joins (a block of 256 threads for every 64 tokens) stay
    below 2^32 threads; more are refused before anything is launched, so that no row is updated
    by a call that fails. The accepted count goes on to the next check (no workspace here)."""
    from triton_tagi_amd import _lib

    lib = _lib.load()
    for n, match in (((1 << 30) - 64, "workspace"), ((1 << 30) - 63, "too large"), ((1 << 30) - 1, "too large")):
        assert lib.tagi_embedding_sorted_bwd(1, 0, 1, 1, 1, 1, 1, n, 50, 1, -1, 1.0, None, 0, None) != 0
        assert match in _lib.last_error(), (n, _lib.last_error())
        assert lib.tagi_embedding_sorted_bwd_update(1, 0, 1, 1, 1, 1, None, None, 2.0, n, 50, 1, -1, 1.0, None, 0, None) != 0
        assert match in _lib.last_error(), (n, _lib.last_error())
