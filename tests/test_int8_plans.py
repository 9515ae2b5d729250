"""CPU tests of what 8-bit contraction plans say of themselves: kernel, family and workspace."""
from __future__ import annotations

import pytest

from einsum_ir_b200 import cabi, operators as op


@pytest.mark.parametrize("n,k", [(2, 1), (4096, 4096), (16382, 4096), (64, 131071)])
def test_one_token_is_the_row_kernels(n, k):
    plan = op.Int8ContractPlan(1, n, k)
    assert plan.describe().startswith("int8 row ") and "split" not in plan.describe()
    assert plan.family == cabi.FAMILY_SIMT
    assert plan.workspace_bytes == 0  # operands of any alignment are read in place


@pytest.mark.parametrize("act", [op.ACT_NONE, op.ACT_GATED_SILU])
def test_one_token_of_a_large_layer(act):
    """the tensor cores where they can stream the rows in place, the row kernel elsewhere; no copies either way"""
    plan = op.Int8ContractPlan(1, 16384, 4096, activation=act)
    assert plan.family == cabi.FAMILY_TC and plan.describe().startswith("int8 split ")
    assert plan.describe().endswith("(row where operands are off the 16-byte grid)")
    assert plan.workspace_bytes == 0


@pytest.mark.parametrize("m,n,k,kernel", [(2, 64, 64, "split"), (77, 10922, 4096, "split"), (8192, 4096, 4096, "pair")])
def test_more_tokens_are_the_tensor_cores(m, n, k, kernel):
    plan = op.Int8ContractPlan(m, n, k)
    assert plan.family == cabi.FAMILY_TC and plan.describe().startswith(f"int8 {kernel} ")
    assert plan.workspace_bytes > 0


def test_nothing_to_sum_is_the_epilogue_alone():
    for m in (1, 40):
        plan = op.Int8ContractPlan(m, 64, 0)
        assert plan.family == cabi.FAMILY_SIMT and plan.describe().startswith("int8 simt ")
        assert plan.workspace_bytes == 0
