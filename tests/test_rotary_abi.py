"""The C entries of rotary positions refuse what they cannot take before they touch the device: descriptors with made-up addresses, no GPU."""

import ctypes
import math

import pytest

from kohakufa_b200 import _lib

BASE = 1 << 20


def tensor4(shape, stride=None, ptr=BASE):
    d = _lib.KfaTensor4()
    d.ptr = ptr
    if stride is None:  # [B, H, S, D] views of [B, S, H, D] storage
        b, h, s, n = shape
        stride = (s * h * n, n, h * n, 1)
    for i in range(4):
        d.shape[i], d.stride[i] = shape[i], stride[i]
    return d


def rotary(pairs=32, amplitude=1.0, turns=BASE):
    r = _lib.KfaRotary()
    r.turns, r.pairs, r.amplitude = turns, pairs, amplitude
    return r


def cache(batch=2, heads=2, dim=64, **more):
    c = _lib.KfaCache()
    c.k = c.v = tensor4((8, heads, 16, dim))
    c.v.ptr = 2 * BASE
    c.table, c.table_stride, c.table_cols, c.lengths, c.batch = BASE, 4, 4, BASE, batch
    for name, value in more.items():
        setattr(c, name, value)
    return c


def ref(x):
    return None if x is None else ctypes.byref(x)


Q, K = (2, 4, 3, 64), (2, 2, 3, 64)
OVERLAP = (3 * 4 * 64, 32, 4 * 64, 1)

ROTARY = [
    {"q": None},
    {"q_out": None},
    {"q": tensor4(Q, ptr=BASE + 1)},
    {"q": tensor4(Q, (768, 64, 256, 2))},
    {"q": tensor4(Q, (-768, 64, 256, 1))},
    {"q": tensor4((2, 4, 0, 64))},
    {"q_out": tensor4(Q, OVERLAP)},
    {"q_out": tensor4((2, 4, 4, 64))},
    {"k_out": None},
    {"k": None},
    {"k": tensor4((2, 2, 4, 64))},
    {"k_out": tensor4((2, 3, 3, 64))},
    {"r": None},
    {"r": rotary(0)},
    {"r": rotary(33)},
    {"r": rotary(turns=None)},
    {"r": rotary(amplitude=math.nan)},
    {"dtype": 3},
    {"q": tensor4((1, 1, 1, 1032)), "q_out": tensor4((1, 1, 1, 1032)), "k": None, "k_out": None},
]


@pytest.mark.parametrize("change", range(len(ROTARY)))
def test_rotary_refuses(change):
    a = {"q": tensor4(Q), "k": tensor4(K), "q_out": tensor4(Q), "k_out": tensor4(K), "r": rotary(), "dtype": _lib.KFA_BF16, **ROTARY[change]}
    lib = _lib.load()
    assert lib.kfa_rotary(*(ref(a[n]) for n in ("q", "k", "q_out", "k_out", "r")), 0, a["dtype"], None) == -1
    assert lib.kfa_last_error()


def steps(n=3, index=None):
    return _lib.KfaRows(index, 3, None, n)


APPEND = [
    {"cache": None},
    {"cache": cache(lengths=None)},
    {"cache": cache(heads=4)},
    {"cache": cache(dim=72)},
    {"cache": cache(batch=3)},
    {"k": None},
    {"v": None},
    {"v": tensor4((2, 2, 4, 64))},
    {"k": tensor4(K, ptr=BASE + 8)},
    {"rows": steps(0)},
    {"rows": steps(4)},
    {"rows": steps(2)},  # with queries all tokens are taken
    {"rows": steps(3, BASE)},
    {"rows": steps(3, BASE), "q": None, "q_out": None},  # turned keys with an index
    {"q": None},
    {"q_out": None},
    {"q": tensor4((2, 3, 3, 64))},
    {"q": tensor4((2, 4, 2, 64)), "q_out": tensor4((2, 4, 2, 64))},
    {"q_out": tensor4(Q, OVERLAP)},
    {"k_out": tensor4((2, 2, 3, 64), (384, 32, 128, 1))},
    {"r": rotary(33)},
    {"r": None},
    {"dtype": _lib.KFA_F32},
    {"status": None},
]


@pytest.mark.parametrize("change", range(len(APPEND)))
def test_append_refuses(change):
    a = {"cache": cache(), "q": tensor4(Q), "k": tensor4(K), "v": tensor4(K), "rows": steps(), "r": rotary(), "q_out": tensor4(Q), "k_out": tensor4(K),
         "dtype": _lib.KFA_BF16, "status": BASE, **APPEND[change]}  # fmt: skip
    lib = _lib.load()
    args = [ref(a[n]) for n in ("cache", "q", "k", "v", "rows", "r", "q_out", "k_out")]
    assert lib.kfa_cache_append_rotary(*args, a["dtype"], a["status"], None) == -1
    assert lib.kfa_last_error()


def test_shared_scratch_of_nothing():
    lib = _lib.load()
    q, c = tensor4(Q), cache()
    assert lib.kfa_cache_attend_shared_bytes(None, ref(c), ref(c), None) == 0
    assert lib.kfa_cache_attend_shared_bytes(ref(tensor4((0, 4, 3, 64))), ref(c), ref(c), None) == 0
    assert lib.kfa_cache_attend_shared_bytes(ref(q), ref(c), ref(c), None) > 0
