"""What must not and what must reach a row, in each of the kernels of attention over a cache: up to 64 rows a K / V head (2 and 5 tokens of 4
heads), up to 128 (20) and up to 256 (40), over caches short enough for whole items and long enough for cut ones. Tolerances as in test_cache.py."""

import math

import pytest
import torch

from kohakufa_b200 import KVCache, _lib, attention_cached
from tests.test_cache import check_attention, make_cache, random_tree, rows

TOKENS = [2, 5, 20, 40]  # 8, 20, 80 and 160 rows


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", TOKENS)
@pytest.mark.parametrize("fill", [math.nan, math.inf])
@pytest.mark.parametrize("lengths", [[60, 0, 33, 64], [2500, 0, 31, 700]], ids=["short", "long"])
@pytest.mark.parametrize("page", [None, 16])
def test_what_lies_behind(tokens, fill, lengths, page):
    """Stale positions, and all that counts leaves out."""
    dtype, counts = torch.bfloat16, [tokens - 1, tokens // 2, 0, tokens]
    cache = make_cache(lengths, 2, 64, dtype, page, fill=fill, columns=None if page is None else -(-max(lengths) // page) + 1)
    q, k, v = (rows(4, h, tokens, 64, dtype, s) for h, s in ((8, 1), (2, 2), (2, 3)))
    for b, n in enumerate(counts):
        for t in (q, k, v):
            t[b, :, n:] = fill
    got = check_attention(cache, 8, tokens, dtype, "tree", counts, q=q, k=k, v=v)
    assert bool(torch.isfinite(got).all())
    for b, n in enumerate(counts):
        assert bool((got[b, :, n:] == 0).all())
    got = check_attention(cache, 8, tokens, dtype, "none", counts, q=q)
    assert bool(torch.isfinite(got).all()) and bool((got[1] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", TOKENS[1:])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lengths", [[50, 0], [3001, 77]], ids=["short", "long"])
def test_hidden_new_tokens(tokens, dim, lengths):
    """A new token whose key or value is NaN or infinite reaches exactly the rows that see it."""
    dtype = torch.float16
    cache = make_cache(lengths, 2, dim, dtype, 16)
    q, k, v = (rows(2, h, tokens, dim, dtype, s) for h, s in ((8, 1), (2, 2), (2, 3)))
    tree = random_tree(2, tokens, 5)
    clean = attention_cached(q, cache, k, v, tree=tree.cuda())
    for token in (0, tokens - 2):
        for what, place in ((math.nan, "k"), (math.nan, "v"), (math.inf, "v"), (-math.inf, "v")):
            k2, v2 = k.clone(), v.clone()
            (k2 if place == "k" else v2)[0, 1, token, 3] = what
            got = attention_cached(q, cache, k2, v2, tree=tree.cuda())
            touched = torch.zeros_like(clean, dtype=torch.bool)
            seen = tree[0, :, token]
            if place == "k":
                touched[0, 4:, seen] = True
            else:
                touched[0, 4:, seen, 3] = True
            assert torch.equal(got[~touched], clean[~touched])
            if place == "k" or what != what:
                assert bool(torch.isnan(got[touched]).all())
            else:
                assert bool((got[touched] == what).all())
    assert _lib.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", TOKENS)
@pytest.mark.parametrize("columns", [3, 200])
def test_rows_that_see_nothing(tokens, columns):
    dtype = torch.bfloat16
    tree = torch.zeros(tokens, tokens, dtype=torch.bool)
    tree[tokens - 1, 1] = True
    got = check_attention(make_cache([0, 0], 2, 64, dtype, 16, columns=columns), 8, tokens, dtype, tree)
    assert bool((got[:, :, :-1] == 0).all()) and bool((got[:, :, -1] != 0).any())
    got = check_attention(make_cache([0, 40], 2, 64, dtype, 16, columns=columns), 8, tokens, dtype, tree)
    assert bool((got[0, :, :-1] == 0).all()) and bool((got[1] != 0).any(-1).all())
    got = check_attention(make_cache([0, 10], 2, 128, dtype, 16, columns=columns), 8, tokens, dtype, "none")
    assert bool((got[0] == 0).all()) and bool((got[1] != 0).any(-1).all())


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", TOKENS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("length,places", [(240, [50, 130, 239]), (6000, [0, 200, 3000, 5990])], ids=["short", "long"])
def test_a_value_that_is_seen_is_passed_on_whatever_its_weight(tokens, dtype, length, places):
    """0 * NaN is NaN: a visible value that is not finite shows in its column also where its weight is 0 in fp32, whichever tile, stream or part
    it lies in. The first 128 positions' scores are 1024, the others' -1024."""
    dim = 64
    cache = make_cache([length], 2, dim, dtype, 16, spare=0)
    at = torch.arange(length, device="cuda")
    page, slot = cache.table[0].long()[at // 16], at % 16
    cache.k.transpose(1, 2)[page, slot] = torch.where(at < 128, 4.0, -4.0).to(dtype)[:, None, None].expand(length, 2, dim)
    q = torch.full((1, tokens, 8, dim), 4.0, dtype=dtype, device="cuda").transpose(1, 2)
    clean = attention_cached(q, cache, scale=1.0)
    assert bool(torch.isfinite(clean).all())
    for place in places:
        for what in (math.nan, math.inf):
            v = cache.v.clone()
            v[int(page[place]), 1, int(slot[place]), 5] = what
            got = attention_cached(q, KVCache(cache.k, v, cache.lengths, cache.table), scale=1.0)
            touched = torch.zeros_like(clean, dtype=torch.bool)
            touched[:, 4:, :, 5] = True
            assert not bool(torch.isfinite(got[touched]).any()), place
            assert torch.equal(got[~touched], clean[~touched])
    assert _lib.device_status() == 0
