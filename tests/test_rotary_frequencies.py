"""Frequencies of rotary positions for longer contexts, against their formulas (no GPU)."""

import pytest

from kohakufa_b200 import Rotary, rotary_frequencies


@pytest.mark.parametrize("factor", [0.5, 1e-3, 1e-6])
def test_a_context_that_shrinks_has_no_amplitude(factor):
    """0.1 ln(factor) + 1 is for contexts that grow: below a factor of 4.5e-5 it would be negative."""
    f, amplitude = rotary_frequencies(64, 1e4, method="yarn", factor=factor, length=4096)
    assert amplitude == 1.0 and bool((f > 0).all())
    assert rotary_frequencies(64, 1e4, method="yarn", factor=1.0, length=4096)[1] == 1.0
    assert Rotary.of(64, method="yarn", factor=factor, length=4096, device="cpu").amplitude == 1.0
