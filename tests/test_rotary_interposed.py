"""``apply_rotary`` where something stands between it and the kernels (a compiler, a mode): it takes and refuses what a plain call does."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from kohakufa_b200 import Rotary, apply_rotary


def test_a_last_dim_that_is_not_contiguous_is_refused():
    with FakeTensorMode():
        r = Rotary.__new__(Rotary)
        r.turns, r.interleaved, r.amplitude = torch.empty(4, dtype=torch.int64, device="cuda"), False, 1.0
        right, odd = torch.empty(2, 4, 3, 8, device="cuda"), torch.empty(2, 4, 8, 3, device="cuda").transpose(2, 3)
        assert apply_rotary(right, None, r).shape == right.shape
        assert [x.shape for x in apply_rotary(right, right[:, :2], r)] == [right.shape, right[:, :2].shape]
        for q, k in ((odd, None), (odd, right), (right, odd)):
            with pytest.raises(ValueError, match="contiguous last dim"):
                apply_rotary(q, k, r)


@pytest.mark.gpu
def test_compiled_and_plain_refuse_the_same():
    r = Rotary.of(8)
    odd = torch.randn(2, 4, 8, 3, device="cuda").transpose(2, 3)
    for call in (apply_rotary, torch.compile(apply_rotary, backend="aot_eager")):
        with pytest.raises(ValueError, match="contiguous last dim"):
            call(odd, None, r)
    one = torch.randn(2, 3, 5, device="cuda")[..., None].transpose(1, 2).expand(2, 5, 3, 1)  # a last dim of one column has no order
    with pytest.raises(ValueError, match="does not fit"):
        apply_rotary(one, None, r)
