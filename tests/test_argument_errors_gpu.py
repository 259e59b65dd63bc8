"""Argument errors whose message carries a number are raised, in the process that made the call."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_mx_quant_of_an_odd_width():
    from nano_gpic_b200._ext import ext
    with pytest.raises(RuntimeError, match="multiple of 128, got 104"):
        ext().mx_quant(torch.zeros(4, 104, dtype=torch.bfloat16, device="cuda"))


def test_gemm_operand_of_an_odd_row_stride():
    from nano_gpic_b200.ops import gemm as G
    x, w = (torch.zeros(n, 101, dtype=torch.bfloat16, device="cuda")[:, :64] for n in (8, 16))
    with pytest.raises(RuntimeError, match="got ld=101"):
        G.linear(x, w)
