"""The give-up path of the kernels on a cache, run on a device as in test_abort.py: the library built with waits of a few hundred cycles, whose
first wait for a copy from global memory runs out by itself. Every call ends, reports ``100 + wait id``, leaves NaN where its results
would be, and the shipped library goes on working beside it."""

import ctypes

import pytest
import torch

from kohakufa_b200 import KVCache, _lib, attention_cached, build

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def short():
    if not build.LIB_SHORT_WAIT.exists():
        pytest.fail(f"{build.LIB_SHORT_WAIT} is missing: run `python -m kohakufa_b200.build`")
    lib = ctypes.CDLL(str(build.LIB_SHORT_WAIT))
    shipped = _lib.load()
    for name in ("kfa_cache_attend", "kfa_cache_attend_bytes", "kfa_cache_weigh", "kfa_cache_weigh_bytes"):
        getattr(lib, name).argtypes = getattr(shipped, name).argtypes
        getattr(lib, name).restype = getattr(shipped, name).restype
    return lib


def describe(cache):
    c = _lib.KfaCache()
    c.k, c.v = _lib.tensor4(cache.k), _lib.tensor4(cache.v)
    c.table, c.table_stride, c.table_cols = cache.table.data_ptr(), cache.table.stride(0), cache.table.shape[1]
    c.lengths, c.batch = cache.lengths.data_ptr(), cache.lengths.numel()
    return ctypes.byref(c)


def ref(t):
    return ctypes.byref(_lib.tensor4(t))


@pytest.mark.parametrize("tokens,columns", [(1, 4), (1, 80), (20, 80), (40, 80)])
@pytest.mark.parametrize("dim", [64, 128])
def test_a_wait_that_runs_out_is_reported_and_the_context_survives(short, tokens, columns, dim):
    dtype, heads, stream = torch.bfloat16, 8, _lib.stream_ptr(torch.device("cuda", 0))
    gen = torch.Generator().manual_seed(dim)
    make = lambda *s: torch.randn(*s, generator=gen).to(dtype).cuda().transpose(1, 2)  # noqa: E731
    cache = KVCache(make(2 * columns, 16, 2, dim), make(2 * columns, 16, 2, dim),
                    torch.tensor([16 * columns - 40, 20], dtype=torch.int32).cuda(),
                    torch.arange(2 * columns, dtype=torch.int32).cuda().view(2, columns))  # fmt: skip
    q, k, v = make(2, tokens, heads, dim), make(2, tokens, 2, dim), make(2, tokens, 2, dim)
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, stats = torch.zeros_like(q), torch.zeros(2, heads, 2, tokens, device="cuda")
    room = short.kfa_cache_attend_bytes(ref(q), describe(cache), ref(k))
    assert (room > 0) == (columns > 4)
    scratch = torch.zeros(room // 4 + 4, device="cuda")
    rc = short.kfa_cache_attend(ref(q), describe(cache), ref(k), ref(v), None, None, None, ref(out), stats.data_ptr(), scratch.data_ptr(),
                                dim**-0.5, 1, word.data_ptr(), stream)  # fmt: skip
    assert rc == 0
    torch.cuda.synchronize()  # returns: nothing hangs
    assert 170 <= int(word.item()) <= 190, int(word.item())
    assert bool(torch.isnan(out).all()) and bool(torch.isnan(stats).all())

    word.zero_()
    rows = _lib.KfaRows(None, 0, None, tokens)
    weights = torch.zeros(2, 2, 16 * columns, device="cuda")
    stride = (ctypes.c_int64 * 2)(weights.stride(0), weights.stride(1))
    room = short.kfa_cache_weigh_bytes(ref(q), describe(cache), ctypes.byref(rows))
    scratch = torch.zeros(room // 4 + 4, device="cuda")
    stats.fill_(1.0)
    rc = short.kfa_cache_weigh(ref(q), stats.data_ptr(), describe(cache), ctypes.byref(rows), weights.data_ptr(), stride, 16 * columns, 0,
                               scratch.data_ptr(), dim**-0.5, 1, word.data_ptr(), stream)  # fmt: skip
    assert rc == 0
    torch.cuda.synchronize()
    assert 170 <= int(word.item()) <= 190, int(word.item())
    for b, n in enumerate(cache.lengths.tolist()):
        assert bool(torch.isnan(weights[b, :, : n + tokens]).all())

    # the shipped library, with its own status word, in the same process
    assert bool(torch.isfinite(attention_cached(q, cache, k, v)).all()) and _lib.device_status() == 0
