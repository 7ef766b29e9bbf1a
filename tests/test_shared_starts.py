"""Attention behind shared prefixes with ``starts`` that say what is not so: reported, NaN, and nothing is shared out by them."""

import pytest
import torch

from kohakufa_b200 import KVCache, _lib, attention_shared
from tests.test_cache import make_cache, rows
from tests.test_shared import check_shared

gpu = pytest.mark.gpu


def pools(batch, prefixes, kv_heads, dim, columns, dtype=torch.bfloat16):
    """Caches of many prefixes and sequences whose positions all lie in a few pages, which are only read."""
    make = lambda s: rows(4, kv_heads, 64, dim, dtype, s)  # noqa: E731
    table = lambda n, m: (torch.arange(n * m) % 4).to(torch.int32).view(n, m).cuda()  # noqa: E731
    long = torch.full((prefixes,), 64 * columns - 7, dtype=torch.int32, device="cuda")
    prefix = KVCache(make(1), make(2), long, table(prefixes, columns))
    return prefix, KVCache(make(3), make(4), torch.full((batch,), 5, dtype=torch.int32, device="cuda"), table(batch, 1))


@gpu
@pytest.mark.parametrize("kind", ["in turn", "backwards", "outside"])
def test_prefixes_that_would_share_their_sequences(kind):
    """Every second prefix claims the whole batch: 2048 times 16384 items of 71 units pass 2^31, which 4096 prefixes that ascend (49144 items) do not."""
    batch, prefixes = 4096, 4096
    prefix, cache = pools(batch, prefixes, 8, 64, 32)
    q = rows(batch, 32, 1, 64, torch.bfloat16, 5)
    good = torch.arange(prefixes + 1, dtype=torch.int32)
    bad = {"in turn": good % 2 * batch, "backwards": good.flip(0), "outside": good + (good == prefixes)}[kind].to(torch.int32)
    assert _lib.device_status() == 0
    try:
        out, stats = attention_shared(q, prefix, cache, starts=bad.cuda(), return_stats=True)
        assert _lib.device_status() == _lib.DEV_BAD_CACHE
        assert bool(torch.isnan(out).all()) and bool(torch.isnan(stats).all())
    finally:
        _lib.reset_device_status()
    out = attention_shared(q, prefix, cache, starts=good.cuda())
    assert _lib.device_status() == 0 and bool(torch.isfinite(out).all())


@gpu
@pytest.mark.parametrize("at,value", [(0, -1), (0, 3), (600, 0), (600, 70), (1100, 71), (1100, 0)])
def test_one_entry_of_many(at, value):
    """An entry anywhere among more prefixes than a CTA has threads. (64 sequences: prefix 300 has 0 .. 9, prefix 700 the rest.)"""
    prefix, cache = pools(64, 1100, 2, 128, 3)
    starts = torch.zeros(1101, dtype=torch.int32)
    starts[301:], starts[701:] = 10, 64
    q = rows(64, 4, 2, 128, torch.bfloat16, 5)
    want = attention_shared(q, prefix, cache, starts=starts.cuda())
    assert _lib.device_status() == 0 and bool(torch.isfinite(want).all())
    bad = starts.clone()
    bad[at] = value
    try:
        out = attention_shared(q, prefix, cache, starts=bad.cuda())
        assert _lib.device_status() == _lib.DEV_BAD_CACHE and bool(torch.isnan(out).all())
    finally:
        _lib.reset_device_status()
    assert torch.equal(attention_shared(q, prefix, cache, starts=starts.cuda()), want)


@gpu
def test_nobody_goes_on_from_any():
    """starts inside the batch that leave no prefix anyone are right: every sequence has its own cache alone."""
    prefix, cache = make_cache([100, 90], 2, 64, torch.bfloat16, 16, seed=1), make_cache([30, 20, 400], 2, 64, torch.bfloat16, 16)
    got = [check_shared(prefix, cache, [n] * 3, 4, 1, torch.bfloat16) for n in (0, 2, 3)]
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
