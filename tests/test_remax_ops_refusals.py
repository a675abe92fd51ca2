"""Argument checks of the Remax attention operators that need no GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch


def test_cpu_tensors_are_refused():
    from triton_tagi_amd import kernels as K

    q, n = torch.zeros(1, 2, 1, 4), torch.zeros(1, dtype=torch.int32)
    cache, table = K.new_kv_cache(1, 1, 2, 4, device="cpu"), torch.zeros(1, 1, dtype=torch.int32)
    for call in (lambda: K.qk_norm_rotary(q, q, q, q),
                 lambda: K.qk_norm_rotary_backward(q, q, q, q, q, q, None),
                 lambda: K.remax_attention(q, q, q, q, q, q),
                 lambda: K.remax_attention_backward(q, q, q, q, q, q, q, torch.zeros(3, 1, 1, 2)),
                 lambda: K.cache_write(cache, q, q, q, q, table),
                 lambda: K.cache_read(cache, table, n, 2),
                 lambda: K.remax_attention_step(q[:, 0], q[:, 0], cache, table, n)):
        with pytest.raises(ValueError, match="GPU only"):
            call()


def test_new_kv_cache_arguments():
    from triton_tagi_amd import kernels as K

    with pytest.raises(TypeError, match="float16"):
        K.new_kv_cache(1, 1, 1, 8, torch.float16, device="cpu")
    with pytest.raises(ValueError, match="bad sizes"):
        K.new_kv_cache(1, 1, 0, 8, device="cpu")
    c = K.new_kv_cache(3, 2, 5, 8, torch.float8_e4m3fn, device="cpu")
    assert c.km.shape == (3, 2, 5, 8) and c.km.dtype is torch.float8_e4m3fn and c.scales.shape == (3, 2, 5, 4)
    assert K.new_kv_cache(3, 2, 5, 8, torch.bfloat16, device="cpu").scales is None


def test_library_argument_errors():
    from triton_tagi_amd import _lib

    lib = _lib.load()
    h = _lib.Heads(1, 1, 1)

    def err(name, *args, match):
        assert getattr(lib, name)(*args) != 0, name
        assert match in _lib.last_error(), _lib.last_error()

    def sec(*n):
        return (ctypes.c_int64 * len(n))(*n)

    def rot(B=1, T=2, H=1, G=1, D=8, w=(None,) * 4, pos=1, pb=4, axes=1, s=None, freq=1, pairs=4, p=1):
        return (p, p, h, p, p, h, *w, pos, pb, axes, s or sec(4), freq, pairs, 0, 1e-6, p, p, p, p, p, B, T, H, G, D, None)

    err("tagi_qk_rotary_fwd", *rot(D=257), match="head dimension")
    err("tagi_qk_rotary_fwd", *rot(H=0), match="bad sizes")
    err("tagi_qk_rotary_fwd", *rot(pairs=5), match="pairs")
    err("tagi_qk_rotary_fwd", *rot(axes=5), match="axes")
    err("tagi_qk_rotary_fwd", *rot(pb=2), match="positions")
    err("tagi_qk_rotary_fwd", *rot(s=sec(3)), match="sections")
    err("tagi_qk_rotary_fwd", *rot(axes=2, s=sec(5, -1)), match="sections")
    err("tagi_qk_rotary_fwd", *rot(pos=None), match="null pointer")
    err("tagi_qk_rotary_fwd", *rot(w=(1, None, 1, 1)), match="norm")
    err("tagi_qk_rotary_fwd", *rot(p=None), match="null pointer")
    err("tagi_qk_rotary_fwd", *rot(B=1 << 20, T=1 << 20), match="too large")
    assert lib.tagi_qk_rotary_fwd(*rot(B=0, p=None)) == 0
    need = lib.tagi_qk_rotary_bwd_ws_bytes(2, 300, 4, 2, 64)
    assert need > 0

    def bwd(ws, n, dw=(1,) * 4):
        return (1, 1, h, 1, 1, h, 1, h, 1, h, 1, 1, 1, 1, 1, 1, 4, 1, sec(4), 1, 4, 0, 1, 1, h, 1, 1, h, *dw, 2, 300, 4, 2, 64,
                ws, n, None)

    err("tagi_qk_rotary_bwd", *bwd(1, need - 1), match="workspace")
    err("tagi_qk_rotary_bwd", *bwd(1, need, (1, None, 1, 1)), match="null pointer")

    def cache(kind=0, pages=2, heads=1, page=4, dim=8, p=1, scales=None):
        return _lib.KvCache(p, p, p, p, scales, kind, pages, heads, page, dim)

    write = lambda c, table=1, sb=0, st=None, p=1, T=2: (c, p, p, h, p, p, h, table, 3, st, sb, None, 0, 1, T, None)  # noqa: E731
    err("tagi_kv_cache_write", *write(cache(kind=3)), match="type")
    err("tagi_kv_cache_write", *write(cache(kind=2)), match="null pointer")
    err("tagi_kv_cache_write", *write(cache(dim=129)), match="head dimension")
    err("tagi_kv_cache_write", *write(cache(page=0)), match="bad sizes")
    err("tagi_kv_cache_write", *write(cache(), table=None), match="null pointer")
    err("tagi_kv_cache_write", *write(cache(), st=1, sb=2), match="starts")
    err("tagi_kv_cache_write", *write(cache(), p=None), match="null pointer")
    err("tagi_kv_cache_write", *write(cache(p=None)), match="null pointer")
    assert lib.tagi_kv_cache_write(*write(cache(), T=0, p=None)) == 0
    err("tagi_kv_cache_read", cache(), 1, 3, None, 4, 1, 1, 1, 1, 1, 2, None, match="lengths")
    err("tagi_kv_cache_read", cache(), 1, 3, 1, 4, 1, 1, None, 1, 1, 2, None, match="null pointer")

    def fwd(B=1, T=4, N=4, H=2, G=1, D=8, p=1, lens=None, lb=0, ws=None, n=0):
        return (p, p, h, p, p, h, p, p, h, lens, lb, None, 0, 1, p, p, p, B, T, N, H, G, D, 1.0, ws, n, None)

    err("tagi_remax_attention_fwd", *fwd(D=129), match="head dimension")
    err("tagi_remax_attention_fwd", *fwd(H=3, G=2), match="bad sizes")
    err("tagi_remax_attention_fwd", *fwd(B=1 << 12, G=1 << 6, H=1 << 6), match="too large")
    err("tagi_remax_attention_fwd", *fwd(lens=1, lb=3), match="lengths")
    err("tagi_remax_attention_fwd", *fwd(p=None), match="null pointer")
    err("tagi_remax_attention_fwd", *fwd(ws=1, n=1), match="workspace")
    assert lib.tagi_remax_attention_fwd(*fwd(T=0, p=None)) == 0

    def back(p=1, D=8):
        return (p, p, h, p, p, h, p, h, p, p, h, p, None, 0, None, 0, 1, p, p, h, p, p, p, p, h, 1, 4, 4, 2, 1, D, 1.0, None, 0,
                None)

    err("tagi_remax_attention_bwd", *back(D=200), match="head dimension")
    err("tagi_remax_attention_bwd", *back(p=None), match="null pointer")

    def step(c=None, H=2, ws=None, n=0, p=1, lens=1, lb=4):
        return (p, p, h, c or cache(), 1, 3, lens, lb, p, p, 1, H, 12, 1.0, ws, n, None)

    err("tagi_remax_attention_step", *step(cache(heads=2), H=3), match="bad sizes")
    err("tagi_remax_attention_step", *step(lens=None), match="lengths")
    err("tagi_remax_attention_step", *step(p=None), match="null pointer")
    err("tagi_remax_attention_step", *step(ws=1, n=8), match="workspace")
