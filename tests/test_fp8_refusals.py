"""What the 8-bit operators and the routed layer refuse before they need a device or the kernel library."""
import pytest
import torch

from batchspec_b200.kernels import ops


def test_tensors_on_the_host_are_refused():
    bf = torch.zeros(4, 64, dtype=torch.bfloat16)
    q, s = torch.zeros(4, 64).to(torch.float8_e4m3fn), torch.ones(4, 1)
    w = torch.zeros(2, 64, 64, dtype=torch.bfloat16)
    with pytest.raises(ops.KernelError, match="CUDA device"):
        ops.quantize_fp8(bf)
    with pytest.raises(ops.KernelError, match="CUDA device"):
        ops.linear_fp8(q, s, q, torch.ones(1, 1))
    with pytest.raises(ops.KernelError, match="CUDA device"):
        ops.moe_layer(bf, torch.zeros(2, 64, dtype=torch.bfloat16), None, 1, 1, 1, 1.0, w, w)


def test_rows_and_scales_that_the_products_cannot_read_are_refused():
    q = torch.zeros(4, 72).to(torch.float8_e4m3fn)
    for bad in (q, q[:, 1:65], torch.zeros(4, 64), q[:, :64].t()):
        with pytest.raises(ops.KernelError):
            ops._fp8_rows(bad, "x")
    assert ops._fp8_rows(torch.zeros(4, 64).to(torch.float8_e4m3fn), "x") == 64
    assert ops._fp8_rows(q[:1], "x") == 80                          # a single row: padded as quantize_fp8 would
    for bad in (torch.ones(4, 2).double(), torch.ones(3, 2), torch.ones(2, 4).t(), torch.ones(8)):
        with pytest.raises(ops.KernelError):
            ops._fp8_scales(bad, 4, 2, "scale")
    assert ops._fp8_scales(torch.ones(4, 2), 4, 2, "scale") == (2, 0)
    assert ops._fp8_scales(torch.ones(4, 2).to(torch.float8_e8m0fnu), 4, 2, "scale") == (2, 1)
