"""Attention behind shared prefixes where scores are a million and differ by a few units.

Queries and keys are small integers beside one large column, so that every score is a whole number below 2^22, exact in the tensor core's fp32. What is left of an
exponent's error is that of one multiply-add, score * c - m: c is off by 2^-24 of itself, which counts for the difference of two scores (below 2^8 units of
log2 that matter, so 2^-16), and the rounding of m is in P, l and O alike. That is inside the 2^-12 of test_shared.py's tolerances, which hold here as they are: with
an exponent taken of the rounded product the error would be half of 2^21's last place, 2^-3, and P off by a tenth."""

import pytest
import torch

from tests.test_cache import make_cache
from tests.test_shared import check_shared

pytestmark = pytest.mark.gpu
SCALE = 0.5


def whole(shape, dtype, seed, first):
    """[n, rows, heads, D] -> [n, heads, rows, D]: column 0 is `first`, column 1 zero, the others -1, 0 or 1."""
    x = torch.randint(-1, 2, shape, generator=torch.Generator().manual_seed(seed)).float()
    x[..., 0], x[..., 1] = first, 0.0
    return x.to(dtype).cuda().transpose(1, 2)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("lead", [-60.0, -6.0, 0.0, 6.0, 60.0])  # of the prefix' scores
@pytest.mark.parametrize("batch,tokens,dim", [(2, 1, 64), (9, 1, 128), (3, 6, 64), (40, 4, 128), (2, 40, 128), (80, 1, 64)])
def test_scores_of_a_million(batch, tokens, dim, lead, sign, dtype):
    kv_heads, heads = 2, 8
    prefix, cache = make_cache([700], kv_heads, dim, dtype, 16, seed=1), make_cache([[300, 40, 0, 150][b % 4] for b in range(batch)], kv_heads, dim, dtype, 16)
    for c, s in ((prefix, 2), (cache, 3)):
        n, h, size, d = c.k.shape
        c.k.copy_(whole((n, size, h, d), dtype, s, sign * 1024.0))
    prefix.k[..., 1] = lead
    q = whole((batch, tokens, heads, dim), dtype, 4, 2048.0)
    q[..., 1] = 1.0
    k, v = whole((batch, tokens, kv_heads, dim), dtype, 5, sign * 1024.0), make_cache([tokens] * batch, kv_heads, dim, dtype).v
    check_shared(prefix, cache, None, heads, tokens, dtype, "causal", q=q, k=k, v=v, scale=SCALE)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("down", [False, True])
@pytest.mark.parametrize("batch,tokens", [(2, 1), (3, 6), (40, 4), (2, 40), (80, 1)])
def test_maxima_that_grow_along_the_keys(batch, tokens, down, dtype):
    """A unit of a score every fourth position: sums and outputs are rescaled many times, between references of a million, or never."""
    kv_heads, heads, dim = 2, 8, 64
    prefix = make_cache([900], kv_heads, dim, dtype, seed=1)
    cache = make_cache([[700, 33, 900, 0][b % 4] for b in range(batch)], kv_heads, dim, dtype)
    for c, s in ((prefix, 2), (cache, 3)):
        n, h, size, d = c.k.shape
        c.k.copy_(whole((n, size, h, d), dtype, s, 1024.0))
        steps = (torch.arange(size, device="cuda") // 4).to(dtype)
        c.k[..., 1] = -steps if down else steps
    q = whole((batch, tokens, heads, dim), dtype, 4, 2048.0)
    q[..., 1] = 1.0
    check_shared(prefix, cache, None, heads, tokens, dtype, "none", q=q, scale=SCALE)
