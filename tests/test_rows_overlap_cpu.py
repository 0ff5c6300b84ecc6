"""Rows of two operands in one buffer, on a machine without a GPU: beside each other they are taken, over each other refused.
Accepted calls end at the missing stream."""
import pytest

from n550_qwen3_bringup_handover_amd import runtime
from tests.test_int8_cpu import A, C, EINVAL, ESTATE, rules

pytestmark = pytest.mark.skipif(runtime.gpu_visible(), reason="accepted calls would launch")


def test_logits_beside_their_results():
    """columns of one matrix: 1,000 logits and 1,000 results a row, in either order, with room between and without"""
    for ld in (2000, 2500):
        for at in (1000, ld - 1000):
            assert rules(out=C + 4 * at, x=C, ld=ld, ldo=ld) == ESTATE, (ld, at)
            assert rules(out=C, x=C + 4 * at, ld=ld, ldo=ld) == ESTATE, (ld, at)
            # a row further on, so that the first logits lie before the first results or the last behind the last
            assert rules(out=C + 4 * (at + ld), x=C, ld=ld, ldo=ld) == ESTATE and rules(out=C, x=C + 4 * (at + ld), ld=ld, ldo=ld) == ESTATE
        for at in (999, ld - 999):
            assert rules(out=C + 4 * at, x=C, ld=ld, ldo=ld) == EINVAL and rules(out=C, x=C + 4 * at, ld=ld, ldo=ld) == EINVAL
    # strides that differ: the memory that they span has to be apart
    assert rules(out=C + 4 * 1000, x=C, ld=2000, ldo=2001) == EINVAL
    assert rules(out=C + 4 * 7000, x=C, ld=2000, ldo=2001) == ESTATE and rules(out=C + 4 * 6999, x=C, ld=2000, ldo=2001) == EINVAL
    # one row: whatever its stride
    assert rules(out=C + 4 * 1000, x=C, ld=2000, ldo=5000, n=1) == ESTATE and rules(out=C + 4 * 999, x=C, ld=2000, ldo=5000, n=1) == EINVAL
