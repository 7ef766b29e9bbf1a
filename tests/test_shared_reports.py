"""Attention behind shared prefixes over caches that say what is not so, in every kernel: reported, and every output is NaN."""

import pytest
import torch

from kohakufa_b200 import KVCache, _lib, attention_shared
from tests.test_cache import make_cache, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,heads", [(1, 4), (6, 8), (40, 8)])  # 16 rows, 32, and as many as are matrix rows themselves
@pytest.mark.parametrize("which", ["prefix", "own"])
@pytest.mark.parametrize("fault", ["page", "negative page", "length", "negative length"])
def test_every_output_is_nan(which, fault, tokens, heads):
    dtype, dim = torch.bfloat16, 64
    prefix, cache = make_cache([100, 90], 2, dim, dtype, 16, seed=1), make_cache([30, 70, 400], 2, dim, dtype, 16)
    q, k, v = (rows(3, h, tokens, dim, dtype, s) for h, s in ((heads, 1), (2, 2), (2, 3)))
    starts = torch.tensor([0, 1, 3], dtype=torch.int32).cuda()
    clean = attention_shared(q, prefix, cache, k, v, starts=starts)
    good = prefix if which == "prefix" else cache
    table, lengths = good.table.clone(), good.lengths.clone()
    if "page" in fault:
        table[1, 2] = -1 if "negative" in fault else good.k.shape[0]
    else:
        lengths[1] = -5 if "negative" in fault else good.capacity + 1
    bad = KVCache(good.k, good.v, lengths, table)
    p, c = (bad, cache) if which == "prefix" else (prefix, bad)
    assert _lib.device_status() == 0
    try:
        out, stats = attention_shared(q, p, c, k, v, starts=starts, return_stats=True)
        assert _lib.device_status() == _lib.DEV_BAD_CACHE
        assert bool(torch.isnan(out).all()) and bool(torch.isnan(stats).all())
    finally:
        _lib.reset_device_status()
    assert torch.equal(attention_shared(q, prefix, cache, k, v, starts=starts), clean)
