"""Attention and eviction over tens of millions of positions, whose pages a table names again and again, and prompts of many row tiles.

Tolerance of the attention: that of test_cache.py (u + 2^-12 of sum p |v|, u = eps / 2), and for 40 M positions 2^-10 more: a CTA adds up some 2200
tiles of 128 keys, 8 matrix instructions each whose fp32 sum is cut off (2^-23 each at most: 2^-9 where all values have one sign, far less for values of
both; l adds 1100 rounded numbers a thread, 2^-14)."""

import math

import pytest
import torch

from kohakufa_b200 import KVCache, _lib, attention_cached, cache_evict
from tests.test_cache import make_cache, rows


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,dim", [(1, 8), (9, 8), (20, 16), (40, 8)])  # 4, 36, 80, 160 rows
def test_attention_over_a_very_long_cache(tokens, dim):
    page, pages, repeats, heads = 4096, 4, 2500, 4
    gen = torch.Generator().manual_seed(tokens)
    k, v = (torch.randn(pages, page, 1, dim, generator=gen).half().cuda().transpose(1, 2) for _ in range(2))
    table = (torch.arange(repeats * pages, dtype=torch.int32) % pages).view(1, -1).cuda()
    cache = KVCache(k, v, torch.tensor([repeats * pages * page], dtype=torch.int32).cuda(), table)
    q = rows(1, heads, tokens, dim, torch.float16, tokens)
    out, stats = attention_cached(q, cache, return_stats=True, scale=0.25)
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    scores = q[0].double() @ k.double().reshape(-1, dim).T
    p = torch.softmax(scores * 0.25, -1)
    values = v.double().reshape(-1, dim)
    room = (2.0**-11 + 2.0**-12 + 2.0**-10) * (p @ values.abs()) + 2.0**-24
    off = (out[0].double() - p @ values).abs()
    assert bool((off <= room).all()), float((off / room).max())
    m = scores.amax(-1)
    assert torch.allclose(stats[0, :, 0].double(), m, rtol=2.0**-18, atol=2.0**-16)
    log2l = torch.exp((scores - m[..., None]) * 0.25).sum(-1).log2() + math.log2(repeats)
    assert torch.allclose(stats[0, :, 1].double(), log2l, rtol=0, atol=2.0**-12)


@pytest.mark.gpu
def test_eviction_of_a_very_long_cache():
    page, pages, length, keep, recent = 4096, 4, 40_000_001, 1000, 10
    gen = torch.Generator().manual_seed(0)
    k, v = (torch.randn(pages, page, 2, 8, generator=gen).half().cuda().transpose(1, 2) for _ in range(2))
    table = (torch.arange(-(-length // page), dtype=torch.int32) % pages).view(1, -1).cuda()
    cache = KVCache(k, v, torch.tensor([length], dtype=torch.int32).cuda(), table)
    weights = torch.randint(0, 70_000, (1, 2, cache.capacity), generator=gen).float().cuda()  # (ties at the border)
    got, w_out, kept = cache_evict(cache, weights, keep, recent=recent)
    best = weights[0, :, : length - recent].sort(dim=1, descending=True, stable=True).indices[:, : keep - recent].sort(dim=1).values
    want = torch.cat([best, torch.arange(length - recent, length, device="cuda").expand(2, -1)], 1)
    assert torch.equal(kept[0].long(), want) and torch.equal(w_out[0], weights[0].gather(1, want))
    for pages_, rows_ in ((k, got.k), (v, got.v)):
        for g in range(2):
            assert torch.equal(rows_[0, g], pages_[(want[g] // page) % pages, g, want[g] % page])
    assert got.lengths.tolist() == [keep] and _lib.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens,lengths,heads,kv_heads,dim", [(1500, [300, 0], 8, 2, 64), (1023, [0], 6, 2, 128), (700, [5, 2000, 64], 5, 1, 40)])
def test_prompts(tokens, lengths, heads, kv_heads, dim, dtype):
    """Many tiles of rows, each of which sees some of the call's own keys; tokens that counts leaves out, NaN in their rows."""
    batch = len(lengths)
    cache = make_cache(lengths, kv_heads, dim, dtype, 16, fill=math.nan, columns=-(-max(*lengths, 16) // 16) + 1)
    q, k, v = (rows(batch, h, tokens, dim, dtype, s) for h, s in ((heads, 1), (kv_heads, 2), (kv_heads, 3)))
    counts = [tokens - 130 * b for b in range(batch)]
    for b, n in enumerate(counts):
        for t in (q, k, v):
            t[b, :, n:] = math.nan
    out, stats = attention_cached(q, cache, k, v, counts=torch.tensor(counts, dtype=torch.int32).cuda(), return_stats=True)
    u = torch.finfo(dtype).eps / 2
    for b, (n, count) in enumerate(zip(lengths, counts)):
        at = torch.arange(n, device="cuda")
        page = cache.table[b].long()[at // 16]
        seen = torch.ones(count, n + count, dtype=torch.bool, device="cuda").tril(n)
        for h in range(heads):
            g = h // (heads // kv_heads)
            keys, values = (torch.cat([pages[page, g, at % 16], new[b, g, :count]]).double() for pages, new in ((cache.k, k), (cache.v, v)))
            s = (q[b, h, :count].double() @ keys.T).masked_fill(~seen, -math.inf)
            p = torch.softmax(s * dim**-0.5, -1)
            want = p @ values
            assert bool(((out[b, h, :count].double() - want).abs() <= (u + 2.0**-12) * (p @ values.abs()) + u * want.abs() + 2.0**-24).all())
            assert torch.allclose(stats[b, h, 0, :count].double(), s.amax(-1), rtol=2.0**-18, atol=2.0**-16)
        assert bool((out[b, :, count:] == 0).all()) and bool(torch.isinf(stats[b, :, 0, count:]).all())
    assert _lib.device_status() == 0
