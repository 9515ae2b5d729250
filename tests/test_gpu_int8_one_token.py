"""One token through layers on both sides of the size from which the tensor cores take them."""
from __future__ import annotations

import pytest

from einsum_ir_b200 import operators as op
from tests.test_gpu_operators import ACTS, BF16, F32, contract_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("ld,offset", [(4096, 0), (4112, 16), (4099, 0), (4096, 3)])
@pytest.mark.parametrize("n", [16382, 16384, 16386])
def test_contract_one_token(cuda, n, ld, offset, act, out):
    plan = contract_case(1, n, 4096, act, out, ld=ld, offset=offset)
    assert plan.describe().startswith("int8 row" if n < 16384 else "int8 split")


@pytest.mark.parametrize("act", [op.ACT_NONE, op.ACT_GATED_SILU])
def test_contract_one_token_of_a_wide_layer(cuda, act):
    """a vocabulary's channels, K not a whole block"""
    contract_case(1, 65538, 1040, act, BF16)
    contract_case(1, 65538, 1040, act, F32, bias=False, scales=False)
