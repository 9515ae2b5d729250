"""CPU tests of the row stride that the norm's backward pass takes h at: x's, or the sum's."""
from __future__ import annotations

import pytest
import torch

from einsum_ir_b200 import cabi, operators as op

ROWS, COLS, LD = 6, 40, 48


class Calls(op.NormPlan):
    """records the row stride of h that a backward call passes on"""

    def stride_of(self, h):
        seen = []
        self._backward = lambda handle, dy, at, stride_h, *rest: seen.append(stride_h) or 0
        self.backward(1 << 20, h, 1 << 20, 1 << 20)
        return seen[0]


def padded(lead=(ROWS,), ld=LD):
    return torch.zeros(*lead, ld, dtype=torch.bfloat16)[..., :COLS]


def test_tensors_say_how_their_rows_lie():
    plan = Calls(ROWS, COLS, cabi.BF16, stride_x=LD, stride_residual=LD)
    packed = torch.zeros(ROWS, COLS, dtype=torch.bfloat16)
    assert plan.stride_of(padded()) == LD  # x, where the forward call had no residual
    assert plan.stride_of(packed) == COLS  # the sum, packed by default
    assert plan.stride_of(packed.view(2, 3, COLS)) == COLS and plan.stride_of(padded((2, 3))) == LD
    other = Calls(ROWS, COLS, cabi.BF16, stride_sum=LD)
    assert other.stride_of(packed) == COLS and other.stride_of(padded()) == LD


def test_flat_buffers_and_addresses_stand_for_x_where_they_can():
    plan = Calls(ROWS, COLS, cabi.BF16, stride_x=LD)
    assert plan.stride_of(torch.zeros(ROWS * COLS, dtype=torch.bfloat16)) == COLS  # ends before x's rows would
    assert plan.stride_of(torch.zeros(ROWS * LD, dtype=torch.bfloat16)) == LD
    assert plan.stride_of(torch.zeros(ROWS * LD * 2, dtype=torch.uint8)) == LD
    assert plan.stride_of(1 << 20) == LD


def test_given_strides_hold():
    assert Calls(ROWS, COLS, cabi.BF16, stride_x=LD, stride_h=56).stride_of(torch.zeros(ROWS, COLS)) == 56
    assert Calls(ROWS, COLS, cabi.BF16, stride_x=LD, stride_sum=LD).stride_of(torch.zeros(ROWS, COLS)) == LD
    assert Calls(1, COLS, cabi.BF16, stride_x=LD).stride_of(torch.zeros(1, COLS)) == LD


def test_rows_that_lie_like_neither_are_refused():
    plan = Calls(ROWS, COLS, cabi.BF16, stride_x=LD)
    for h in (padded(ld=56), torch.zeros(1, COLS, dtype=torch.bfloat16).expand(ROWS, COLS), padded((2, 4))[:, :3]):
        with pytest.raises(cabi.EirError) as e:
            plan.stride_of(h)
        assert e.value.code == 52


def test_stride_of_a_call_is_checked():
    plan, a = op.NormPlan(ROWS, COLS, cabi.BF16), 1 << 20
    assert cabi.lib().eir_norm_backward_strided(plan.handle, a, a, -1, a, a, a, a, a, 0) == 52
    assert cabi.lib().eir_norm_backward_strided(None, a, a, COLS, a, a, a, a, a, 0) == 52
