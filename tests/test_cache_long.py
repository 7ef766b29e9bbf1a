"""Accumulated weights over caches of tens of millions of positions. The keys are a few pages that the table names again and again, so that what
every position gets is known from those pages. The exponent is off by 2^-24 of its terms (below 2^6 here), the exponential by 2^-22, the sum
over up to 300 rows by less than 2^-15: 2^-13 relative covers them (as in test_cache.py)."""

import pytest
import torch

from kohakufa_b200 import KVCache, _lib, cache_weights
from tests.test_cache import LOG2E





@pytest.mark.gpu
@pytest.mark.parametrize(
    "group,tokens,length",
    [(64, 1, 40_000_000), (32, 2, 70_000_000), (128, 1, 20_000_000), (64, 2, 40_000_000), (100, 3, 30_000_000)],
)
def test_weights_of_a_very_long_cache(group, tokens, length):
    """So many positions before the new tokens that their distance times the rows of a token passes 2^31. A log2 sum of 20 takes the
    form with two numbers a row where there is another."""
    dim, page, pages = 8, 4096, 4
    gen = torch.Generator().manual_seed(group)
    k = torch.randn(pages, page, 1, dim, generator=gen).half().cuda().transpose(1, 2)
    columns = -(-(length + tokens) // page)
    cache = KVCache(k, k, torch.tensor([length], dtype=torch.int32).cuda(), (torch.arange(columns, dtype=torch.int32) % pages).view(1, -1).cuda())
    q = torch.randn(1, tokens, group, dim, generator=gen).half().cuda().transpose(1, 2)
    stats = torch.zeros(1, group, 2, tokens, device="cuda")
    stats[:, :, 1] = 20.0
    got = cache_weights(cache, q, stats, scale=1.0)
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    scores = q[0].double().flatten(0, 1) @ k.double().reshape(-1, dim).T  # [group * tokens, positions of the pages]
    each = torch.exp2(scores * LOG2E - 20.0).view(group, tokens, -1)
    whole = length // (pages * page) * (pages * page)
    want = each.sum((0, 1))
    off = (got[0, 0, :whole].view(-1, pages * page) - want).abs().amax(0)
    assert bool((off <= want * 2.0**-13).all()), float((off / want).max())
    rest = torch.zeros(got.shape[2] - whole, dtype=torch.float64, device="cuda")
    for t in range(tokens):
        last = length + t + 1 - whole
        rest[:last] += each[:, t].sum(0).repeat(2)[:last]
    assert torch.allclose(got[0, 0, whole:].double(), rest, rtol=2.0**-13, atol=0)
