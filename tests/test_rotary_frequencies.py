"""Frequencies of rotary positions for longer contexts, against their formulas (no GPU)."""

import math

import pytest
import torch

from kohakufa_b200 import Rotary, rotary_frequencies


@pytest.mark.parametrize("factor", [0.5, 1e-3, 1e-6])
def test_a_context_that_shrinks_has_no_amplitude(factor):
    """0.1 ln(factor) + 1 is for contexts that grow: below a factor of 4.5e-5 it would be negative."""
    f, amplitude = rotary_frequencies(64, 1e4, method="yarn", factor=factor, length=4096)
    assert amplitude == 1.0 and bool((f > 0).all())
    assert rotary_frequencies(64, 1e4, method="yarn", factor=1.0, length=4096)[1] == 1.0
    assert Rotary.of(64, method="yarn", factor=factor, length=4096, device="cpu").amplitude == 1.0


# dim, base, length, high, low: and the pairs between which the ramp lies, dim ln(length / (2 pi turns)) / (2 ln base) down for `high` and up for `low`
RAMPS = [
    ((128, 1e4, 4096, 32.0, 1.0), (20, 46)),  # 20.94, 45.03
    ((64, 1e4, 4096, 32.0, 1.0), (10, 23)),  # 10.47, 22.51
    ((128, 5e5, 8192, 32.0, 1.0), (18, 35)),  # 18.08, 34.98
    ((96, 1e6, 2048, 4.0, 0.5), (15, 23)),  # 15.28, 22.51
]


@pytest.mark.parametrize("args,between", RAMPS, ids=str)
@pytest.mark.parametrize("factor", [4.0, 16.0])
def test_yarn_by_pairs(args, between, factor):
    dim, base, length, high, low = args
    first, last = between
    f, amplitude = rotary_frequencies(dim, base, method="yarn_pairs", factor=factor, length=length, high=high, low=low)
    assert math.isclose(amplitude, 0.1 * math.log(factor) + 1)
    for i in range(dim // 2):
        plain = base ** (-2 * i / dim)
        left = min(max((last - i) / (last - first), 0.0), 1.0)  # of the frequency as it is
        assert math.isclose(float(f[i]), plain * left + plain / factor * (1 - left), rel_tol=1e-13), i
    assert Rotary.of(dim, base, method="yarn_pairs", factor=factor, length=length, high=high, low=low, device="cpu").amplitude == amplitude


def test_the_two_ramps_differ_between_their_ends():
    by_turns, by_pairs = (rotary_frequencies(128, method=m, factor=16.0, length=4096)[0] for m in ("yarn", "yarn_pairs"))
    assert torch.allclose(by_turns[:21], by_pairs[:21], rtol=1e-14) and torch.allclose(by_turns[46:], by_pairs[46:], rtol=1e-14)
    ratio = by_pairs / by_turns
    assert int(((ratio - 1).abs() > 0.05).sum()) == 24 and int(ratio.argmax()) == 38 and 3.0 < float(ratio.max()) < 3.1


@pytest.mark.parametrize("dim", [2, 4, 32])
@pytest.mark.parametrize("length", [1, 6, 40, 10**6])
@pytest.mark.parametrize("low", [0.0, 1.0])
def test_yarn_by_pairs_at_its_bounds(dim, length, low):
    """Lengths over which no pair turns often, or all do, and a `low` that nothing gets below: between the frequency and its `factor`th, and falling."""
    f, _ = rotary_frequencies(dim, method="yarn_pairs", factor=8.0, length=length, low=low)
    plain, _ = rotary_frequencies(dim)
    assert bool(torch.isfinite(f).all()) and bool((f <= plain * (1 + 1e-15)).all()) and bool((f >= plain / 8 * (1 - 1e-15)).all())
    assert bool((f[1:] < f[:-1]).all())


@pytest.mark.parametrize("more", [{"base": 1.0}, {"base": 0.5}, {"length": None}, {"low": 4.0, "high": 4.0}])
def test_yarn_by_pairs_refuses(more):
    with pytest.raises(ValueError):
        rotary_frequencies(16, method="yarn_pairs", factor=2.0, **{"length": 4096, **more})


def inverse_of_two_pi(bits):
    """floor(2^bits / (2 pi)) in whole numbers, by Machin's formula: pi / 4 = 4 arctan(1 / 5) - arctan(1 / 239)."""
    room = 1 << (bits + 64)

    def arctan(n):
        power, total, k = room // n, 0, 0
        while power:
            total += (power // (2 * k + 1)) * (-1) ** k
            power //= n * n
            k += 1
        return total

    return (room << bits) // (8 * (4 * arctan(5) - arctan(239)))


@pytest.mark.parametrize("dim,base,more", [(128, 1e4, {}), (64, 5e5, {"method": "yarn", "factor": 16.0, "length": 4096}), (1024, 1e6, {"method": "linear", "factor": 3.0})])
def test_turns_within_their_bound(dim, base, more):
    """2^-52 of the frequency and half a unit: 2 pi in 64 bits is off by 2^-54.5 of itself, the quotient by 2^-53."""
    f, _ = rotary_frequencies(dim, base, **more)
    turns = Rotary(f, device="cpu").turns.tolist()
    assert inverse_of_two_pi(64) == 2935890503282001226  # 0.15915494309189533577 * 2^64
    one = inverse_of_two_pi(256)
    for x, got in zip(f.tolist(), turns):
        num, den = x.as_integer_ratio()
        off = got * 2**192 - num * one // den  # in units of 2^-256 turns
        off = (off + 2**255) % 2**256 - 2**255
        assert abs(off) <= num * one // den // 2**52 + 2**191, (x, off / 2**192)
