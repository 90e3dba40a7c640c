"""Block-scaled FP8 operators at their edges: few rows with K over a cluster,
gates far below zero, operands and outputs that are refused.

Tolerances of the products: tests/test_gpu_fp8_block.py."""
import pytest
import torch

from tests.test_gpu_fp8_block import assert_rounded_from, check_mm, check_swiglu, operands, sum_slack
from tests.util import assert_no_device_error

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- few rows, K over a cluster
@pytest.mark.parametrize("m", [1, 7, 16, 17, 32])
@pytest.mark.parametrize("n,k", [(128, 128), (512, 256), (512, 512), (1000, 1024), (3072, 1024), (128, 4096)])
def test_mm_few_rows_short_ranges(m, n, k):
    """One to a few k-tiles for each CTA of a cluster of 1 to 8: a CTA sends its
    partials to the others as early as it can."""
    check_mm(m, n, k)
    assert_no_device_error()


@pytest.mark.parametrize("m", [1, 16, 17, 32])
@pytest.mark.parametrize("h,k", [(128, 256), (2048, 512), (1040, 1024)])
def test_swiglu_few_rows_short_ranges(m, h, k):
    check_swiglu(m, h, k)
    assert_no_device_error()


@pytest.mark.parametrize("n,k", [(512, 512), (3072, 1024), (14336, 256)])
def test_few_rows_back_to_back(n, k):
    """Launches queued back to back: clusters start while earlier ones end, and every result is the same."""
    from recavsr_b200.runtime import fp8_block
    (ac, asc), (bc, bsc), av, bv = operands(3, n, k, 31)
    outs = [fp8_block.mm(ac, bc, asc, bsc) for _ in range(200)]
    assert_rounded_from(outs[0], av @ bv.t(), sum_slack(av, bv, k))
    for out in outs[1:]:
        assert torch.equal(out, outs[0])
    assert_no_device_error()
