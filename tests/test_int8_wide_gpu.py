"""8-bit products into rows of C that lie further apart than 2^20 values, and the tiles that such rows go to, against their
definition (tests/int8_oracle.py)."""
import pytest

from n550_qwen3_bringup_handover_amd import abi, runtime
from tests.test_int8_gpu import At, Product

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def lib():
    return runtime.init()


# the widest rows that tiles of 64 rows take; a little further apart: the narrow kernel; tiles' rows behind 2^20
@pytest.mark.parametrize("m,n,ldc,gated,bf16", [(5, 9000, 1 << 23, False, False), (5, 9000, (1 << 23) + 1, False, False),
                                                (5, 4600, 1 << 23, True, True), (6, 9000, (1 << 23) + 5, True, True),
                                                (70, 5000, (1 << 20) + 16, False, False), (130, 2801, (1 << 20) + 3, True, False),
                                                (300, 3100, (1 << 20) + 24, False, True)])
def test_far_rows(m, n, ldc, gated, bf16):
    p = Product(m, 300, n, gated=gated, bf16=bf16, ldc=ldc, seed=6)
    p.run()


@pytest.mark.parametrize("gated", [False, True])
def test_columns_behind_2_20(gated):
    """sizes on both sides of the border that used to end the tiles"""
    for n in (1 << 20, (1 << 20) + 16):
        assert abi.int8_plan(40, 64, n, gated).startswith("tile")
        Product(40, 64, n, gated=gated, seed=7).run()


# a size of every kernel
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,n", [(3, 1001), (60, 1400), (60, 4010), (130, 5603), (700, 3301), (1001, 4301), (1905, 7001)])
def test_results_at_any_address_of_their_own_size(m, n, gated, bf16):
    p = Product(m, 200, n // (1 + gated), gated=gated, bf16=bf16, ldc=-(-n // 32) * 32, seed=8)
    for shift in (2, 6) if bf16 else (4, 12):
        p.cd = At(p.mark, shift)
        p.run()
