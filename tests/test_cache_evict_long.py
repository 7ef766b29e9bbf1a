"""Eviction of sequences longer than the selection holds in registers. Copies and selections are exact."""

import pytest
import torch

from kohakufa_b200 import _lib, cache_evict
from tests.test_cache import WEIGHTS, expect_evicted, logical, make_cache



@pytest.mark.gpu
@pytest.mark.parametrize("kind", WEIGHTS)
@pytest.mark.parametrize("lengths,keep,recent", [([20011, 8193, 8192, 12288], 5000, 100), ([131075], 2048, 256), ([40000, 9], 39999, 0)])
def test_eviction_of_long_sequences(kind, lengths, keep, recent):
    """More positions than the selection holds in registers (8 a thread), ties among them."""
    dim = 8
    cache = make_cache(lengths, 2, dim, torch.float16, 64)
    gen = torch.Generator().manual_seed(keep)
    weights = WEIGHTS[kind](torch.randn(len(lengths), 2, cache.capacity, generator=gen)).cuda()
    want = expect_evicted(weights, lengths, keep, recent)
    got, w_out, kept = cache_evict(cache, weights, keep, recent=recent)
    assert torch.equal(kept.cpu(), want) and got.lengths.tolist() == [min(n, keep) for n in lengths]
    picked = weights.cpu().gather(2, want.clamp(min=0).long()).masked_fill(want < 0, 0.0)
    assert torch.equal(torch.nan_to_num(w_out.cpu(), 7.0, 8.0, -8.0), torch.nan_to_num(picked, 7.0, 8.0, -8.0))
    for which in "kv":
        rows = logical(cache, which).gather(2, want.clamp(min=0).long()[..., None].expand(-1, -1, -1, dim))
        assert torch.equal(logical(got, which), rows.masked_fill((want < 0)[..., None], 0.0))
    assert _lib.device_status() == 0
