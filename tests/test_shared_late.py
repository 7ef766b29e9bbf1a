"""Attention behind shared prefixes with warps that come late: a library in which the producers of values begin 200,000 clk behind everything else (see
``kohakufa_b200/build.py``), as they would on an SM that another kernel keeps busy. Nothing may depend on their coming together with the others:
outputs and statistics are those of the shipped library, bit for bit, and no wait runs out."""

import ctypes

import pytest
import torch

from kohakufa_b200 import _lib, attention_shared, build
from tests.test_cache import make_cache, rows
from tests.test_shared import describe, ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def late():
    if not build.LIB_LATE.exists():
        pytest.fail(f"{build.LIB_LATE} is missing: run `python -m kohakufa_b200.build`")
    lib, shipped = ctypes.CDLL(str(build.LIB_LATE)), _lib.load()
    for name in ("kfa_cache_attend_shared", "kfa_cache_attend_shared_bytes"):
        getattr(lib, name).argtypes, getattr(lib, name).restype = getattr(shipped, name).argtypes, getattr(shipped, name).restype
    return lib


# prefix, own lengths, heads, K / V heads, tokens: stretches of one tile, of two, of as many as there are stages, of many; 16, 32, 128 rows and pairs of 128
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize(
    "before,lengths,heads,kv_heads,tokens",
    [
        (20, [10, 0], 4, 1, 1),
        (250, [200, 256, 130], 4, 1, 1),
        (250, [200, 256, 130], 8, 1, 3),
        (600, [500, 380] * 6, 8, 2, 1),
        (40000, [5000, 20], 4, 1, 1),
        (3000, [700, 90, 0, 260] * 4, 8, 2, 3),
        (3000, [700, 90, 0, 260] * 12, 8, 2, 2),
        (130, [100, 64], 8, 2, 40),
        (20000, [1500, 300] * 40, 8, 2, 1),
    ],
)
def test_values_that_come_late(late, before, lengths, heads, kv_heads, tokens, dim):
    dtype, batch = torch.bfloat16, len(lengths)
    prefix, cache = make_cache([before], kv_heads, dim, dtype, 32, seed=1), make_cache(lengths, kv_heads, dim, dtype, 16)
    q, k, v = (rows(batch, h, tokens, dim, dtype, s) for h, s in ((heads, 1), (kv_heads, 2), (kv_heads, 3)))
    want, want_stats = attention_shared(q, prefix, cache, k, v, return_stats=True)
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, stats = torch.zeros_like(want), torch.zeros_like(want_stats)
    room = late.kfa_cache_attend_shared_bytes(ref(q), describe(prefix), describe(cache), ref(k))
    scratch = torch.zeros(room // 4 + 8, device="cuda")
    rc = late.kfa_cache_attend_shared(ref(q), describe(prefix), None, describe(cache), ref(k), ref(v), None, None, None, ref(out), stats.data_ptr(),
                                      scratch.data_ptr(), dim**-0.5, 1, word.data_ptr(), _lib.stream_ptr(torch.device("cuda", 0)))  # fmt: skip
    assert rc == 0
    torch.cuda.synchronize()
    assert int(word.item()) == 0 and _lib.device_status() == 0
    assert torch.equal(out, want) and torch.equal(stats, want_stats)
