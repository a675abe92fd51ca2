"""The paged cache: writes and reads bit for bit, and one query over its pages against float64."""

from __future__ import annotations

import math

import pytest
import torch

from remax_reference import attention, within

pytestmark = pytest.mark.gpu

F32, BF16, FP8 = torch.float32, torch.bfloat16, torch.float8_e4m3fn


def rounded(x, dtype):
    """What the cache holds of rows x (..., D), as float64, and the exponents of 8-bit rows. CPU."""
    x = x.detach().cpu().float()
    if dtype is not FP8:
        return x.to(dtype).double(), None
    ok = torch.isfinite(x)
    top = torch.where(ok, x.abs(), 0.0).amax(-1).double()
    e = torch.where(top > 0, torch.ceil(torch.log2(top.clamp_min(1e-300) / 448.0)), -126.0).clamp(-126, 127)
    code = torch.where(ok, x.double() / torch.exp2(e)[..., None], float("nan")).float().to(FP8).double()
    return code * torch.exp2(e)[..., None], (e + 127).to(torch.uint8)


def cache_of(dev, pages, G, page, D, dtype, seed=0):
    from triton_tagi_amd import kernels as K

    c = K.new_kv_cache(pages, G, page, D, dtype, dev)
    r = torch.Generator().manual_seed(seed)
    for p in c[:4]:  # marks, so that a stray write shows
        p.view(torch.uint8).copy_(torch.randint(0, 120, p.view(torch.uint8).shape, generator=r, dtype=torch.uint8))
    return c


def rows_of(B, T, G, D, seed, dev):
    r = torch.Generator().manual_seed(seed)
    x = [torch.randn(B, T, G, D, generator=r), 0.1 * torch.rand(B, T, G, D, generator=r),
         10 * torch.randn(B, T, G, D, generator=r), torch.rand(B, T, G, D, generator=r) ** 8]
    return [t.to(dev) for t in x]


def values(cache):
    """The pools as float64 on the CPU, by the definition."""
    out = []
    for i, p in enumerate(cache[:4]):
        x = p.view(torch.uint8).cpu().view(p.dtype).double() if p.dtype is FP8 else p.cpu().double()
        if cache.scales is not None:
            x = x * torch.exp2(cache.scales[..., i].cpu().double() - 127)[..., None]
        out.append(x)
    return out


WRITES = [(B, T, G, D, page, dtype) for dtype in (F32, BF16, FP8)
          for B, T, G, D, page in ((1, 1, 1, 1, 1), (2, 5, 2, 3, 7), (3, 9, 2, 80, 4), (2, 40, 3, 128, 16), (1, 7, 1, 6, 64))]


@pytest.mark.parametrize("case", WRITES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_write_and_read(case, dev):
    from triton_tagi_amd import kernels as K

    B, T, G, D, page, dtype = case
    width = -(-(T + 5) // page)
    pages = B * width + 2
    cache = cache_of(dev, pages, G, page, D, dtype)
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(1))[:B * width].view(B, width).int()
    starts = torch.arange(B) % 6
    x = rows_of(B, T, G, D, 2, dev)
    before = values(cache)
    K.cache_write(cache, *x, table.to(dev), starts.to(dev))
    after = values(cache)
    expect = [t.clone() for t in before]
    for i in range(4):
        v, e = rounded(x[i], dtype)
        for b in range(B):
            for t in range(T):
                at = int(starts[b]) + t
                expect[i][table[b, at // page], :, at % page] = v[b, t]
                if e is not None:
                    assert torch.equal(cache.scales[table[b, at // page], :, at % page, i].cpu(), e[b, t])
    for a, b in zip(after, expect):
        assert torch.equal(a, b)
    n = T + 3
    lengths = (starts + T).int()
    got = K.cache_read(cache, table.to(dev), lengths.to(dev), n)
    for i in range(4):
        for b in range(B):
            for t in range(n):
                at = expect[i][table[b, t // page], :, t % page] if t < lengths[b] else torch.zeros(G, D).double()
                assert torch.equal(got[i][b, t].cpu().double(), at)


def test_eight_bits_at_their_ends(dev):
    from triton_tagi_amd import kernels as K

    inf, nan = float("inf"), float("nan")
    rows = [[0.0] * 8, [448.0] * 8, [448.1, 1, 0, 0, 0, 0, 0, 0], [3.4e38, -3.4e38, 1e30, 0, 0, 0, 0, 0],
            [1e-45, 0, 0, 0, 0, 0, 0, 0], [1e-38, 2e-39, 0, 0, 0, 0, 0, 0], [inf, 1.0, -2.0, nan, 0, 0, 0, -inf],
            [nan] * 8, [1.0625, 1.1875, 1.3125, 17.0, 19.0, 21.0, 23.0, 448.0], [-0.0, 0.25, -448, 2**-9, 2**-10, 3 * 2**-10, 2**-11, 0]]
    x = torch.tensor(rows, device=dev).view(1, len(rows), 1, 8)
    cache = K.new_kv_cache(2, 1, 8, 8, FP8, dev)
    table = torch.tensor([[1, 0]], device=dev, dtype=torch.int32)
    K.cache_write(cache, x, x, x, x, table)
    want, e = rounded(x, FP8)
    got = values(cache)
    for i in range(4):
        v = torch.cat([got[i][1, 0], got[i][0, 0]])[:len(rows)]
        assert torch.equal(torch.nan_to_num(v, nan=12345.0), torch.nan_to_num(want[0, :, 0], nan=12345.0))
        s = torch.cat([cache.scales[1, 0, :, i], cache.scales[0, 0, :, i]])[:len(rows)].cpu()
        assert torch.equal(s, e[0, :, 0])


@pytest.mark.parametrize("dtype", [F32, BF16, FP8])
def test_pages_that_do_not_exist(dtype, dev):
    """Written nowhere, read as zeros, not seen; counts, starts and lengths outside the table alike."""
    from triton_tagi_amd import kernels as K

    B, T, G, D, page = 4, 12, 2, 16, 4
    cache = cache_of(dev, 6, G, page, D, dtype)
    table = torch.tensor([[0, -1, 2], [5, 6, 1], [2**31 - 1, -(2**31), 3], [4, 4, 4]], dtype=torch.int32, device=dev)
    x = rows_of(B, T, G, D, 3, dev)
    before = values(cache)
    starts = torch.tensor([0, 0, 0, -(1 << 62)], device=dev)
    K.cache_write(cache, *x, table, starts, counts=torch.tensor([12, 99, 11, 12], device=dev))
    after = values(cache)
    for i in range(4):
        v, _ = rounded(x[i], dtype)
        want = before[i].clone()
        for b in range(3):
            for t in range(12 if b < 2 else 11):
                p = int(table[b, t // page])
                if 0 <= p < 6:
                    want[p, :, t % page] = v[b, t]
        assert torch.equal(after[i], want)
    K.cache_write(cache, *x, table, torch.tensor([1 << 62, 12, 100, -12], device=dev),
                  counts=torch.tensor([12, 12, -3, 0], device=dev))
    for a, b in zip(values(cache), after):
        assert torch.equal(a, b)
    lengths = torch.tensor([9, 1 << 40, 12, -1], device=dev)
    got = K.cache_read(cache, table, lengths, 15)
    ok = torch.zeros(B, 15, dtype=torch.bool)
    for b, n in enumerate((9, 12, 12, 0)):
        for t in range(n):
            ok[b, t] = 0 <= int(table[b, t // page]) < 6
    for i in range(4):
        assert not got[i][~ok.to(dev)].any()
    # attention over the same pages: the tokens that exist, whichever they are
    r = torch.Generator().manual_seed(4)
    mq, Sq = torch.randn(B, 4, D, generator=r).to(dev), 0.1 * torch.rand(B, 4, D, generator=r).to(dev) + 0.01
    # (the marks in unwritten slots are random bits: as float32 up to 2^118, whose squares have no
    # float32 value; every page is written with tokens first)
    pages = torch.arange(6, dtype=torch.int32, device=dev).view(6, 1)
    K.cache_write(cache, *(t.view(-1, page, G, D)[:6] + (0.01 if i % 2 else 0.0)
                           for i, t in enumerate(rows_of(6, page, G, D, 12, dev))), pages)
    mo, So = K.remax_attention_step(mq, Sq, cache, table, lengths, scale=0.3)
    read = K.cache_read(cache, table, lengths, 12)
    for b in range(B):
        live = ok[b, :12].to(dev)
        k = [t[b, live][None] for t in read]
        ref = attention(mq[b, None, None], Sq[b, None, None], *k, 0.3, causal=False,
                        starts=[max(0, int(live.sum()) - 1)])
        within(mo[b, None, None], ref[0], f"mo {b}"), within(So[b, None, None], ref[1], f"So {b}")


# B, H, G, D, page, longest, dtype
STEPS = [
    (1, 1, 1, 1, 1, 1, F32),
    (3, 4, 4, 32, 16, 40, F32),
    (2, 8, 2, 64, 7, 300, F32),
    (2, 6, 2, 80, 48, 333, BF16),
    (5, 5, 1, 128, 16, 100, BF16),
    (2, 12, 2, 128, 64, 700, FP8),
    (3, 3, 3, 33, 5, 90, FP8),
    (1, 16, 1, 48, 128, 1500, FP8),
    (1, 9, 1, 64, 16, 2100, BF16),
    (2, 40, 2, 24, 32, 260, FP8),
]


@pytest.mark.parametrize("case", STEPS, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_step_against_float64(case, dev):
    from triton_tagi_amd import kernels as K

    B, H, G, D, page, longest, dtype = case
    width = -(-longest // page) + 1
    pages = B * width + 1
    cache = K.new_kv_cache(pages, G, page, D, dtype, dev)
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(5))[:B * width].view(B, width).int().to(dev)
    r = torch.Generator().manual_seed(6)
    x = [torch.randn(B, longest, G, D, generator=r), 0.005 + 0.1 * torch.rand(B, longest, G, D, generator=r),
         torch.randn(B, longest, G, D, generator=r), 0.005 + 0.1 * torch.rand(B, longest, G, D, generator=r)]
    K.cache_write(cache, *(t.to(dev) for t in x), table)
    lengths = [longest] + [max(0, longest - 13 * b - (longest if b == B - 1 else 0)) for b in range(1, B)]
    ln = torch.tensor(lengths, device=dev)
    # rows of a wider buffer
    buf = torch.randn(B, 2, H, D + 1, generator=r).to(dev)
    mq, Sq = buf[:, 0, :, :D], buf[:, 1, :, :D].abs_().mul_(0.05).add_(0.005)
    scale = 1 / math.sqrt(D)
    mo, So = K.remax_attention_step(mq, Sq, cache, table, ln, scale=scale)
    keys = K.cache_read(cache, table, ln, longest)
    for b in range(B):
        n = lengths[b]
        ref = attention(mq[b, None, None], Sq[b, None, None], *(t[b, None, :n] for t in keys), scale, causal=False,
                        starts=[max(0, n - 1)])
        within(mo[b, None, None], ref[0], f"mo {b}"), within(So[b, None, None], ref[1], f"So {b}")
    # a bound on the lengths splits the work otherwise
    m1, S1 = K.remax_attention_step(mq, Sq, cache, table, ln, scale=scale, max_len=longest)
    within(m1[0, None, None], attention(mq[0, None, None], Sq[0, None, None], *(t[0, None] for t in keys), scale,
                                        causal=False, starts=[longest - 1])[0], "bounded")
    short = K.remax_attention_step(mq, Sq, cache, table, ln, scale=scale, max_len=longest // 2)
    cut = K.remax_attention_step(mq, Sq, cache, table, ln.clamp_max(longest // 2), scale=scale, max_len=longest // 2)
    for a, b in zip(short, cut):
        assert torch.equal(a, b)
    none = K.remax_attention_step(mq, Sq, cache, table, torch.zeros_like(ln), scale=scale)
    assert not none[0].any() and not none[1].any()


def test_what_lies_behind_a_length_may_hold_anything(dev):
    from triton_tagi_amd import kernels as K

    for dtype in (F32, FP8):
        cache = K.new_kv_cache(4, 1, 8, 16, dtype, dev)
        table = torch.tensor([[2, 0, 3]], device=dev, dtype=torch.int32)
        x = rows_of(1, 11, 1, 16, 7, dev)
        K.cache_write(cache, *x, table)
        mq, Sq = x[0][:, 0].repeat(1, 2, 1), x[1][:, 0].repeat(1, 2, 1) + 0.01
        n = torch.tensor([11], device=dev)
        ref = K.remax_attention_step(mq, Sq, cache, table, n, scale=0.25)
        for p in cache[:4]:
            p.view(torch.uint8)[[1, 3]] = 0x7f  # NaN codes, large floats
            p.view(torch.uint8)[0, :, 3:] = 0xff  # NaN
        for a, b in zip(K.remax_attention_step(mq, Sq, cache, table, n, scale=0.25), ref):
            assert torch.equal(a, b)


def test_serving_captured(dev):
    """Write and attend in one graph whose lengths advance on the GPU; two graphs share nothing."""
    from triton_tagi_amd import kernels as K

    B, H, G, D, page = 2, 4, 2, 32, 4
    cache = K.new_kv_cache(20, G, page, D, FP8, dev)
    table = torch.randperm(20, generator=torch.Generator().manual_seed(8))[:20].view(2, 10).int().to(dev)
    lengths = torch.tensor([3, 9], device=dev)
    K.cache_write(cache, *rows_of(B, 9, G, D, 9, dev), table, counts=lengths)
    new = [t + 0.01 for t in rows_of(B, 1, G, D, 10, dev)]
    mq, Sq = rows_of(B, H, 1, D, 11, dev)[0][:, :, 0], rows_of(B, H, 1, D, 11, dev)[1][:, :, 0] + 0.01

    def call(at):
        K.cache_write(cache, *new, table, at)
        return K.remax_attention_step(mq, Sq, cache, table, at + 1, scale=0.2)

    call(lengths)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(lengths)
        graphs.append((graph, out))
    for i in range(4):
        for t in new:
            t.mul_(1.05)
        for graph, out in graphs:
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, call(lengths)):
                assert torch.equal(a, b), i
        lengths += 1
