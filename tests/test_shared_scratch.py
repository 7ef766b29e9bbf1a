"""How much scratch attention behind shared prefixes asks for: what the header says (no GPU)."""

import pytest

from kohakufa_b200 import _lib
from tests.test_rotary_abi import cache, ref, tensor4


@pytest.mark.parametrize("batch,heads,kv_heads,tokens", [(1, 8, 8, 1), (64, 32, 8, 1), (32, 32, 8, 8), (2, 300, 1, 2), (16, 32, 8, 512), (5, 7, 7, 4000), (4096, 32, 8, 1), (3, 16, 1, 129)])
@pytest.mark.parametrize("prefixes", [1, 5])
@pytest.mark.parametrize("dim", [64, 128])
def test_scratch(batch, heads, kv_heads, tokens, prefixes, dim):
    q, k = tensor4((batch, heads, tokens, dim)), tensor4((batch, kv_heads, tokens, dim))
    prefix, own = cache(batch=prefixes, heads=kv_heads, dim=dim), cache(batch=batch, heads=kv_heads, dim=dim)
    room = _lib.load().kfa_cache_attend_shared_bytes(ref(q), ref(prefix), ref(own), ref(k))
    rows, group = batch * heads * tokens, heads // kv_heads
    tiles = -(-group // 128) * -(-tokens // (128 // min(group, 128)))
    known = 1048 * rows + 16 * kv_heads * tiles * batch
    assert known < room <= known + 40 * 10**6, (room, known)
