"""8-bit products of few tokens whose k is cut into slices, in every number of them.  Tolerances as in ``test_fp8_gpu.py``."""
import pytest
import torch
from test_fp8_gpu import check_product, ops, product_case  # noqa: F401  (ops: a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scales", ["", "w", "xw"])       # which of the two are float32 numbers, not powers of two
@pytest.mark.parametrize("M,N,K", [(3, 256, 4200), (20, 130, 5300), (60, 128, 6200), (64, 300, 4480), (1, 1000, 5121), (17, 120, 1300), (9, 640, 2200),
                                   (33, 130, 14336), (2, 128, 1024), (50, 257, 8321)])
def test_slices_that_are_no_power_of_two(ops, M, N, K, scales, out_dtype):  # noqa: F811
    """K of 33 to 35, 41, 42 and 49 blocks is cut into seven slices, other lengths into two, four or eight, the last one shorter."""
    x, xs, w, ws = product_case(ops, M, N, K, scales, M + N + K)
    check_product(ops.linear_fp8(x, xs, w, ws, out_dtype=out_dtype), x, xs, w, ws)
    ops.check_status()
