"""The norm's results over its weight are refused, whatever their type: a lane stores a row's sum in front of its weight's load.  Every check comes before any device work, so no GPU is needed."""
import pytest

from onenew_amd import abi
from test_f8_refusals_cpu import A, B, D, S, _norm, _refused


@pytest.mark.parametrize("f8", [0, 1])
def test_a_sum_over_the_weight(f8):
    """one fp32 row: sum and weight have the same place, bytes and (no) stride"""
    _refused(_norm(rows=1, compute=abi.COMPUTE_F32, f8=f8, residual=D, weight=D + (1 << 20), total=D + (1 << 20)), "operand")
    _refused(_norm(rows=1, compute=abi.COMPUTE_F32, f8=f8, residual=D, weight=D + (1 << 20), total=D + (1 << 20) + 4), "operand")


def test_a_result_over_the_weight():
    _refused(_norm(rows=1, compute=abi.COMPUTE_F32, f8=0, weight=B, out=B), "operand")
    _refused(_norm(rows=1, compute=abi.COMPUTE_F32, f8=0, residual=A + (1 << 20), weight=B, out=B, total=D), "operand")
    _refused(_norm(rows=1, compute=abi.COMPUTE_F32, f8=1, weight=S, scale=S), "operand")
