"""8-bit products at the ends of float32's range, against 64-bit arithmetic.

Tolerance of a float32 result over K numbers: (2 K + 8) 2^-24 of the sum of the products' magnitudes (fewer than K additions of half a step
each, doubled where the tensor core cuts off instead of rounding, and three roundings per block's scales), and for every block of 128 the
half step of a number below the normal range, 2^-150, twice (the block's number and the sum it joins)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
# few tokens (16, 32 and 64 columns), many tokens, and with powers of two as scales pairs of CTAs
SIZES = [(5, 300, 512), (30, 130, 640), (64, 257, 1152), (2048, 8192, 1024)]


@pytest.fixture(scope="module")
def ops():
    from batchspec_b200.kernels import ops
    ops.load_library()
    return ops


def spread(s, block_rows, rows, cols):
    return s.double().repeat_interleave(block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :cols]


def product_case(ops, M, N, K, powers, x_exp, w_exp):
    """Two quantised matrices whose scales are then moved by powers of two."""
    g = torch.Generator(device=DEV).manual_seed(M + N + K)
    x, xs = ops.quantize_fp8(torch.randn(M, K, device=DEV, generator=g))
    w, ws = ops.quantize_fp8(torch.randn(N, K, device=DEV, generator=g), 128)
    xs, ws = xs.float() * 2.0 ** x_exp, ws.float() * 2.0 ** w_exp
    if powers:
        return x, xs.to(torch.float8_e8m0fnu), w, ws.to(torch.float8_e8m0fnu)
    return x, xs * (1 + torch.rand(xs.shape, device=DEV, generator=g)), w, ws * (1 + torch.rand(ws.shape, device=DEV, generator=g))


def check_product(out, x, xs, w, ws):
    K = x.shape[1]
    a, b = x.double() * spread(xs, 1, *x.shape), w.double() * spread(ws, 128, *w.shape)
    want, room = a @ b.t(), (a.abs() @ b.abs().t()) * (2 * K + 8) * 2.0 ** -24 + 2 * math.ceil(K / 128) * 2.0 ** -150
    off = (out.double() - want).abs()
    assert bool((off <= room).all()), float((off / room).max())
    return float(((off ** 2).mean() / (want ** 2).mean()).sqrt())


@pytest.mark.parametrize("powers", [False, True])
@pytest.mark.parametrize("x_exp,w_exp", [(-62, -62), (-10, -110), (-110, -10), (100, -110), (-110, 100), (50, 50)])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_scales_whose_product_is_small_or_large(ops, M, N, K, x_exp, w_exp, powers):
    """A product of two scales below 2^-126 keeps its bits: results are normal numbers, as sums of products of e4m3 numbers are large.  The error
    over all results is a few half steps, 2^-24: each of K / 128 blocks' sums has at most 10 of them (four cuts of two half steps in the tensor core,
    one of the scales, one of the addition) and the magnitudes of sums of random signs stay within sqrt(K / 128) of the result's."""
    x, xs, w, ws = product_case(ops, M, N, K, powers, x_exp, w_exp)
    off = check_product(ops.linear_fp8(x, xs, w, ws, out_dtype=torch.float32), x, xs, w, ws)
    assert off <= 10 * math.sqrt(K / 128) * 2.0 ** -24
    ops.check_status()


@pytest.mark.parametrize("powers", [False, True])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_zeros_stay_zeros_where_the_scales_overflow(ops, M, N, K, powers):
    x, xs, w, ws = product_case(ops, M, N, K, powers, 100, 100)
    codes = w.view(torch.uint8)
    codes[::3] = 0                                     # rows of zeros, and zeros behind the first block in the others
    codes[:, 128:] = 0
    out = ops.linear_fp8(x, xs, w, ws, out_dtype=torch.float32)
    exact = x[:, :128].double() @ w[:, :128].double().t()      # without scales
    assert bool((out[:, ::3] == 0).all())
    assert not bool(torch.isfinite(out[exact != 0]).any()), "beyond the largest float32 number"
    x.view(torch.uint8)[0] = 0
    assert bool((ops.linear_fp8(x, xs, w, ws, out_dtype=torch.float32)[0] == 0).all())
    ops.check_status()


@pytest.mark.parametrize("M,N,K", SIZES)
def test_rows_with_ordinary_scales_beside_extreme_ones(ops, M, N, K):
    """Scales far apart from token to token and from block to block, zeros among them."""
    x, xs, w, ws = product_case(ops, M, N, K, False, 0, 0)
    xs[::2] *= 2.0 ** -75
    xs[1::4, 1] = 0
    ws[:, 2:] *= 2.0 ** -70
    check_product(ops.linear_fp8(x, xs, w, ws, out_dtype=torch.float32), x, xs, w, ws)
    ops.check_status()


@pytest.mark.parametrize("M,N,K", [(2048, 8192, 4096), (1500, 7000, 2304), (2048, 8192, 512), (3000, 4480, 4200)])
def test_float32_results_of_products_of_one_sign(ops, M, N, K):
    """Cuts towards 0 add up where every product has one sign.  Sums of 128 products are cut by the tensor core four times at most, by up to two half
    steps (2^-24 of the sum each), their scales are exact here, and K / 128 additions in float32 round evenly to either side: together, as a root
    mean square over many results, below (8 + sqrt(K / 128)) half steps."""
    x, xs, w, ws = product_case(ops, M, N, K, True, 0, 0)
    for t in (x, w):
        t.view(torch.uint8).bitwise_and_(0x7F)
    out = ops.linear_fp8(x, xs, w, ws, out_dtype=torch.float32)
    off = check_product(out, x, xs, w, ws)
    assert off <= (8 + math.sqrt(K / 128)) * 2.0 ** -24
    ops.check_status()


@pytest.mark.parametrize("kind", ["e8m0", "float32"])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_blocks_of_nan_show_in_their_rows_and_columns_alone(ops, M, N, K, kind):
    """A token with an infinity, a block of weights with a NaN (as the quantiser marks them), and scales of zero."""
    g = torch.Generator(device=DEV).manual_seed(3)
    xf, wf = torch.randn(M, K, device=DEV, generator=g), torch.randn(N, K, device=DEV, generator=g)
    xf[2, 300], wf[130 if N > 130 else 5, 200] = math.inf, math.nan
    (x, xs), (w, ws) = ops.quantize_fp8(xf), ops.quantize_fp8(wf, 128)
    if kind == "float32":
        xs, ws = xs.float(), ws.float()
        xs[0] = 0
    out = ops.linear_fp8(x, xs, w, ws, out_dtype=torch.float32)
    nan = torch.zeros(M, N, dtype=torch.bool, device=DEV)
    nan[2] = True
    first = 128 if N > 130 else 0
    nan[:, first:first + 128] = True
    assert torch.equal(torch.isnan(out), nan)
    if kind == "float32":
        assert bool((out[0, ~nan[0]] == 0).all())
    keep = [i for i in range(M) if i != 2][:200]
    cols = torch.nonzero(~nan[0])[:, 0]
    if len(cols):
        a = x[keep].double() * spread(xs[keep], 1, len(keep), K)
        b = (w.double() * spread(ws, 128, N, K))[cols]
        room = (a.abs() @ b.abs().t()) * (2 * K + 8) * 2.0 ** -24
        assert bool(((out[keep][:, cols].double() - a @ b.t()).abs() <= room).all())
    ops.check_status()


@pytest.mark.parametrize("M,N,K", SIZES)
def test_the_smallest_and_largest_powers(ops, M, N, K):
    """Scales of 2^-127, which is below float32's normal numbers, meet scales that bring the products back."""
    for xe, we in ((0, 200), (190, 40)):
        x, xs, w, ws = product_case(ops, M, N, K, True, 0, 0)
        xs, ws = torch.full(xs.shape, xe, dtype=torch.uint8, device=DEV), torch.full(ws.shape, we, dtype=torch.uint8, device=DEV)
        xs, ws = xs.view(torch.float8_e8m0fnu), ws.view(torch.float8_e8m0fnu)
        check_product(ops.linear_fp8(x, xs, w, ws, out_dtype=torch.float32), x, xs, w, ws)


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("batch,R,K", [(70001, 5, 8), (33000, 130, 8), (3, 1, 70000)])
def test_quantising_more_matrices_than_a_grid_is_high(ops, batch, R, K, block_rows):
    g = torch.Generator(device=DEV).manual_seed(batch)
    x = torch.randn(batch, R, K, device=DEV, generator=g)
    q, s = ops.quantize_fp8(x, block_rows)
    for i in (0, 1, batch // 2, 65534 // -(-R // block_rows) if batch > 3 else 1, batch - 1):
        i = min(i, batch - 1)
        want_q, want_s = ops.quantize_fp8(x[i], block_rows)
        assert torch.equal(q[i].float(), want_q.float()) and torch.equal(s[i].float(), want_s.float())
    room = q.float() * s.float().repeat_interleave(block_rows, 1)[:, :R].repeat_interleave(128, 2)[:, :, :K] - x
    assert bool((room.abs() <= x.abs() * 2.0 ** -4 + s.float().amax() * 2.0 ** -10).all())
