"""Written tensors whose entries share memory: refused before anything is launched (on the CPU as well), wherever two rows can meet; rows that lie
between one another without meeting are taken."""

import itertools

import pytest
import torch

from kohakufa_b200 import KVCache, cache_evict, cache_weights
from tests.test_cache import cpu_cache


@pytest.mark.parametrize("batch,heads", [(1, 3), (2, 2), (3, 2), (2, 3), (4, 1)])
def test_weights_that_overlap_themselves(batch, heads):
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    c = cpu_cache(k=bf(4, heads, 16, 64), v=bf(4, heads, 16, 64), lengths=torch.zeros(batch, dtype=torch.int32),
                  table=torch.zeros(batch, 2, dtype=torch.int32))  # fmt: skip
    q, stats, memory = bf(batch, heads, 3, 64), torch.zeros(batch, heads, 2, 3), torch.zeros(4000)
    for s, t in itertools.product([0, 1, 31, 32, 33, 63, 64, 65, 96, 100, 128, 160], repeat=2):
        w = memory.as_strided((batch, heads, 32), (s, t, 1))
        starts = sorted(b * s + g * t for b in range(batch) for g in range(heads))
        meet = any(y - x < 32 for x, y in zip(starts, starts[1:]))
        with pytest.raises(ValueError, match="overlap" if meet else "CUDA tensors only"):
            cache_weights(c, q, stats, weights=w)


def test_eviction_into_the_pages_that_it_reads():
    c, other, w, ints = cpu_cache(), cpu_cache(), torch.zeros(2, 2, 32), torch.zeros(2, dtype=torch.int32)
    for k, v in ((c.k, other.v), (other.k, c.v), (c.v, other.v), (other.k, c.k), (c.v, c.k)):
        with pytest.raises(ValueError, match="pages of its own"):
            cache_evict(c, w, 4, out=KVCache(k, v, ints, c.table))
        with pytest.raises(ValueError, match="pages of its own"):
            cache_evict(c, w, 4, out=KVCache(k[:2], v[:2], ints))
        with pytest.raises(ValueError, match="CUDA tensors only"):  # (two tables over one pool may name different pages)
            cache_evict(c, w, 4, out=KVCache(k, v, ints, c.table.clone()))
