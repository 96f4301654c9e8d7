"""8-bit products that follow the kernel which makes their operands.  Tolerances as in ``test_fp8_gpu.py``."""
import pytest
import torch
from test_fp8_gpu import SIZES, check_product, generator, ops, product_case  # noqa: F401  (ops: a fixture)

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.mark.parametrize("M,N,K", [(1, 8192, 4096), (8, 8192, 4096), (30, 8192, 2048), (61, 4096, 4096), (130, 4096, 4096), (2048, 8192, 1024)])
def test_products_that_follow_the_kernel_which_makes_the_weights(ops, M, N, K):  # noqa: F811
    """The quantiser, which lets its successor start at once, writes the weights that the product right behind it reads; each time other weights in the
    memory of the last ones, in a graph, so that nothing comes between the two kernels."""
    g = generator(M)
    wf = [torch.randn(N, K, device=DEV, generator=g) * 2.0 ** (3 * i) for i in range(3)]
    x, xs = ops.quantize_fp8(torch.randn(M, K, device=DEV, generator=g))
    parts = [ops.quantize_fp8(f, 128) for f in wf]
    want = [ops.linear_fp8(x, xs, *p, out_dtype=torch.float32) for p in parts]
    for out, p in zip(want, parts):
        check_product(out, x, xs, *p)
    torch.cuda.synchronize()
    graph, got = torch.cuda.CUDAGraph(), []
    with torch.cuda.graph(graph):
        places = set()
        for i in range(9):
            q, s = ops.quantize_fp8(wf[i % 3], 128)
            places.add(q.data_ptr())
            got.append(ops.linear_fp8(x, xs, q, s, out_dtype=torch.float32))
            del q, s
    assert len(places) < 9, "memory is used again"
    for _ in range(10):
        for o in got:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for i, o in enumerate(got):
            assert torch.equal(o, want[i % 3])
    ops.check_status()


@pytest.mark.parametrize("M,N,K", [c for c in SIZES if c[0] <= 128] + [(3, 256, 4200), (61, 8192, 2048)])
def test_parameters_read_ahead_of_the_tokens(ops, M, N, K):  # noqa: F811
    """``w_is_parameter``: weights are fetched while the kernel that makes the tokens runs."""
    x, xs, w, ws = product_case(ops, M, N, K, "", M + N + K)
    g = generator(7)
    tokens = [torch.randn(M, K, device=DEV, generator=g) * 2.0 ** (3 * i) for i in range(3)]
    want = [ops.linear_fp8(*ops.quantize_fp8(t), w, ws) for t in tokens]
    for t, o in zip(tokens, want):
        check_product(o, *ops.quantize_fp8(t), w, ws)
    torch.cuda.synchronize()
    graph, got = torch.cuda.CUDAGraph(), []
    with torch.cuda.graph(graph):
        for i in range(9):
            q, s = ops.quantize_fp8(tokens[i % 3])
            got.append(ops.linear_fp8(q, s, w, ws, w_is_parameter=True))
            del q, s
    for _ in range(5):
        for o in got:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for i, o in enumerate(got):
            assert torch.equal(o, want[i % 3])
    ops.check_status()
