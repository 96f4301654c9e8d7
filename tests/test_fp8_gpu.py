"""Matrices in 8-bit floating point with a scale per block of 128, and their products, against 64-bit arithmetic.

Tolerances.  Quantising: every result is one exactly defined number, so results are equal.  Products: the products of two e4m3
numbers are exact in float32, and the sum over K numbers in any order is off by at most K 2^-24 of the sum of their magnitudes
(each of fewer than K additions rounds by half a step, 2^-24, of a partial sum that the magnitudes bound); the tensor core may cut off
instead of rounding, which doubles that, and each block's sum meets its scales in three more roundings.  So a float32 result is within
(2 K + 8) 2^-24 * sum |x w|, a bfloat16 one within half a step, 2^-8 of its value, more."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from batchspec_b200.kernels import ops
    ops.load_library()
    return ops


def blocks(n, b=128):
    return -(-n // b)


def generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def spread(s, block_rows, rows, cols):
    return s.double().repeat_interleave(block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :cols]


def quantized(x, block_rows):
    """(q, s) in 64 bits from the definition, number by block."""
    x = x.double()
    rows, cols = x.shape
    q, s = torch.empty_like(x), torch.empty((blocks(rows, block_rows), blocks(cols)), dtype=torch.float64, device=x.device)
    for i in range(s.shape[0]):
        for j in range(s.shape[1]):
            at = (slice(i * block_rows, (i + 1) * block_rows), slice(128 * j, 128 * j + 128))
            top = float(x[at].abs().max())
            if not math.isfinite(top):
                s[i, j], q[at] = math.nan, math.nan
                continue
            e = 0
            if top:
                e = max(-127, math.frexp(top)[1] - 10)
                while top > 448 * 2.0 ** e:
                    e += 1
            s[i, j] = 2.0 ** e
            v = x[at] / 2.0 ** e
            step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
            q[at] = torch.round(v / step) * step
    return q, s


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 129), (7, 300), (130, 264), (129, 1000), (300, 520)])
def test_quantize(ops, dtype, block_rows, rows, cols):
    x = torch.randn(rows, cols, device=DEV, generator=generator(rows * 1000 + cols))
    x *= torch.exp2(torch.randint(-30, 30, (rows, 1), device=DEV, generator=generator(3)).float())
    x = x.to(dtype)
    q, s = ops.quantize_fp8(x, block_rows)
    want_q, want_s = quantized(x, block_rows)
    assert q.dtype == torch.float8_e4m3fn and s.dtype == torch.float8_e8m0fnu and q.shape == x.shape
    assert q.stride(0) % 16 == 0 and q.data_ptr() % 16 == 0
    assert torch.equal(s.double(), want_s)
    assert torch.equal(q.double(), want_q)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_of_borders(ops, dtype, block_rows):
    """Largest numbers on and just above 448 times a power of two, zeros, the smallest and largest numbers of the type, ties."""
    top = torch.finfo(dtype).max
    tiny = torch.finfo(dtype).smallest_normal
    firsts = [448.0, 449.0 if dtype == torch.float32 else 450.0, 0.0, tiny, tiny / 4, top, -top, -448 * 2.0 ** -100, 1.75 * 2.0 ** -119, 2.0 ** -130]
    x = torch.zeros(len(firsts), 256, device=DEV, dtype=torch.float32)
    for i, f in enumerate(firsts):
        x[i, 128 + 17] = f
        x[i, 128 + 20:128 + 28] = torch.tensor([17, 19, 21, -23, 1.0625, 0.0009765625, 0.0029296875, -0.01], device=DEV) * (abs(f) / 448 if f else 0)
    x = x.to(dtype)
    if block_rows == 128:
        x = torch.cat([r[None] * torch.ones(128, 1, device=DEV, dtype=dtype) for r in x])
    q, s = ops.quantize_fp8(x, block_rows)
    want_q, want_s = quantized(x, block_rows)
    assert torch.equal(s.double(), want_s)
    assert torch.equal(q.double(), want_q)


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_a_block_with_an_infinity_or_nan_is_nan_and_its_neighbours_are_not(ops, block_rows, bad):
    x = torch.randn(200, 300, device=DEV, generator=generator(5))
    x[3, 140] = bad
    q, s = ops.quantize_fp8(x, block_rows)
    want_q, want_s = quantized(x, block_rows)
    torch.testing.assert_close(s.double(), want_s, rtol=0, atol=0, equal_nan=True)
    torch.testing.assert_close(q.double(), want_q, rtol=0, atol=0, equal_nan=True)
    assert int(torch.isnan(s.float()).sum()) == 1


def test_quantize_of_views_and_stacks(ops):
    wide = torch.randn(40, 1003, device=DEV, generator=generator(6)).to(torch.bfloat16)
    for view in (wide[:, :300], wide[:, 3:260], wide[::2, 8:264], wide[:, 1:2], wide[5:6, 7:]):
        q, s = ops.quantize_fp8(view)
        want_q, want_s = quantized(view, 1)
        assert torch.equal(q.double(), want_q) and torch.equal(s.double(), want_s)
    stack = torch.randn(3, 2, 130, 150, device=DEV, generator=generator(7))
    for block_rows in (1, 128):
        q, s = ops.quantize_fp8(stack, block_rows)
        assert q.shape == stack.shape and s.shape == (3, 2, blocks(130, block_rows), 2)
        for i in range(3):
            for j in range(2):
                want_q, want_s = quantized(stack[i, j], block_rows)
                assert torch.equal(q[i, j].double(), want_q) and torch.equal(s[i, j].double(), want_s)
    for shape in ((0, 5), (2, 0, 7)):
        q, s = ops.quantize_fp8(torch.empty(shape, device=DEV))
        assert q.shape == shape and s.numel() == 0


def product_case(ops, M, N, K, scales, seed):
    g = generator(seed)
    x = torch.randn(M, K, device=DEV, generator=g) * torch.exp(torch.randn(M, 1, device=DEV, generator=g))
    w = torch.randn(N, K, device=DEV, generator=g) * torch.exp(torch.randn(1, K, device=DEV, generator=g))
    x, xs = ops.quantize_fp8(x)
    w, ws = ops.quantize_fp8(w, 128)
    if "x" in scales:
        xs = xs.float() * (1 + torch.rand(xs.shape, device=DEV, generator=g))
    if "w" in scales:
        ws = ws.float() * (1 + torch.rand(ws.shape, device=DEV, generator=g))
    return x, xs, w, ws


def check_product(out, x, xs, w, ws):
    K = x.shape[1]
    a, b = x.double() * spread(xs, 1, *x.shape), w.double() * spread(ws, 128, *w.shape)
    want, room = a @ b.t(), (a.abs() @ b.abs().t()) * (2 * K + 8) * 2.0 ** -24
    if out.dtype == torch.bfloat16:
        room += want.abs() * 2.0 ** -8
    off = (out.double() - want).abs()
    assert bool((off <= room).all()), float((off / room.clamp(min=1e-300)).max())


SIZES = [(1, 1, 1), (1, 128, 128), (1, 130, 1000), (5, 257, 300), (16, 4096, 512), (17, 1000, 1111), (33, 384, 2048), (64, 129, 4096),
         (65, 200, 640), (100, 2048, 1536), (128, 128, 129), (129, 520, 260), (300, 1000, 2000), (700, 4100, 384), (1300, 2570, 130)]


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scales", ["", "x", "w", "xw"])       # which of the two are float32 numbers, not powers of two
@pytest.mark.parametrize("M,N,K", SIZES)
def test_product(ops, M, N, K, scales, out_dtype):
    x, xs, w, ws = product_case(ops, M, N, K, scales, M + N + K)
    out = ops.linear_fp8(x, xs, w, ws, out_dtype=out_dtype)
    assert out.shape == (M, N) and out.dtype == out_dtype and out.is_contiguous()
    check_product(out, x, xs, w, ws)
    ops.check_status()


@pytest.mark.parametrize("scales", ["", "w"])       # powers of two alone go to the pairs of CTAs, the others not
@pytest.mark.parametrize("M,N,K", [(2048, 8192, 1024), (1500, 10001, 650), (513, 16800, 2000), (3000, 4480, 4200), (257, 20011, 129), (1025, 7168, 384),
                                   (300, 33000, 640)])
def test_product_of_many_tiles(ops, M, N, K, scales):
    """Several tiles per CTA, ends inside tiles and inside groups of four blocks of k, rows of the result on odd places."""
    x, xs, w, ws = product_case(ops, M, N, K, scales, M + N + K)
    for out_dtype in (torch.bfloat16, torch.float32):
        check_product(ops.linear_fp8(x, xs, w, ws, out_dtype=out_dtype), x, xs, w, ws)
    ops.check_status()


def test_millions_of_rows_by_a_narrow_matrix(ops):
    """More tiles of tokens than a grid's second dimension takes."""
    M = 65536 * 64 + 70
    x = torch.zeros(M, 32, device=DEV, dtype=torch.bfloat16)
    x[-5:] = torch.randn(5, 32, device=DEV, generator=generator(5)).to(torch.bfloat16)
    w, ws = ops.quantize_fp8(torch.randn(16, 32, device=DEV, generator=generator(6)), 128)
    q, s = ops.quantize_fp8(x)
    for scales in (s, s.float()):
        out = ops.linear_fp8(q, scales, w, ws)
        check_product(out[-70:], q[-70:], scales[-70:], w, ws)
        assert not bool(out[:-70].any())
    ops.check_status()


def test_offsets_beyond_32_bits(ops):
    """Matrices of more than 2^31 numbers: the last rows of a quantised one, of the weights and of a result."""
    g = generator(41)
    x = torch.zeros(70000, 40000, device=DEV, dtype=torch.bfloat16)
    x[-200:] = torch.randn(200, 40000, device=DEV, generator=g).to(torch.bfloat16)
    tail = x[-200:].clone()
    for block_rows in (1, 128):
        q, s = ops.quantize_fp8(x, block_rows)
        top = 70000 // 128 * 128                                   # the last whole block row begins here
        want_q, want_s = ops.quantize_fp8(x[top:] if block_rows == 128 else x[-3:], block_rows)
        assert torch.equal(q[-3:].float(), want_q[-3:].float()) and torch.equal(s[-1:].float(), want_s[-1:].float())
        assert int((q[:1000].float() != 0).sum()) == 0
    del x
    a, sa = ops.quantize_fp8(tail[:3])
    out = ops.linear_fp8(a, sa, q, s, out_dtype=torch.float32)     # weights of 2.8 GB
    check_product(out[:, top:], a, sa, q[top:], s[top // 128:])
    del q, s, out
    w, sw = ops.quantize_fp8(torch.randn(40000, 128, device=DEV, generator=g), 128)
    y, sy = ops.quantize_fp8(torch.randn(70000, 128, device=DEV, generator=g))
    for scales in (sy, sy.float()):                                # results of 5.6 GB
        out = ops.linear_fp8(y, scales, w, sw)
        check_product(out[-300:], y[-300:], scales[-300:], w, sw)
        check_product(out[:3], y[:3], scales[:3], w, sw)
        del out


@pytest.mark.parametrize("M", [3, 40, 96, 2000])
def test_product_of_views(ops, M):
    """Rows of wider matrices, scales of wider matrices, and neighbours of the result left alone."""
    x, xs, w, ws = product_case(ops, M + 5, 700, 800, "", 11)
    x, xs, w, ws = x[5:, 32:700], xs[5:], w[128:600, 32:700], ws[1:5]
    xs, ws = xs[:, :6], ws[:, :6]                      # (block borders move with the view: only shapes matter here)
    out = ops.linear_fp8(x, xs, w, ws, out_dtype=torch.float32)
    check_product(out, x, xs, w, ws)


def test_product_of_large_and_small_scales(ops):
    """Scales far apart from block to block; zeros; a NaN stays in its row."""
    g = generator(12)
    for M in (4, 200, 2000):
        x = torch.randn(M, 512, device=DEV, generator=g)
        x[:, :128] *= 2.0 ** 30
        x[:, 128:256] *= 2.0 ** -30
        x[:, 256:384] = 0
        w = torch.randn(2048, 512, device=DEV, generator=g)
        w[:, :128] *= 2.0 ** -40
        x, xs = ops.quantize_fp8(x)
        w, ws = ops.quantize_fp8(w, 128)
        check_product(ops.linear_fp8(x, xs, w, ws, out_dtype=torch.float32), x, xs, w, ws)
        bad = x.float()
        bad[1, 400] = math.nan
        out = ops.linear_fp8(bad.to(torch.float8_e4m3fn), xs, w, ws, out_dtype=torch.float32)
        assert bool(torch.isnan(out[1]).all()) and int(torch.isnan(out).sum()) == out.shape[1]


def test_product_that_follows_its_weights(ops):
    """Without ``w_is_parameter`` the weights may come from the kernel before."""
    g = generator(13)
    wf = [torch.randn(4096, 2048, device=DEV, generator=g) for _ in range(2)]
    x, xs = ops.quantize_fp8(torch.randn(8, 2048, device=DEV, generator=g))
    w, ws = ops.quantize_fp8(wf[0], 128)
    for _ in range(20):
        for f in wf:
            q, s = ops.quantize_fp8(f, 128)
            w.copy_(q)
            ws.copy_(s)
            out = ops.linear_fp8(x, xs, w, ws, out_dtype=torch.float32)
        check_product(out, x, xs, w, ws)


def test_products_replayed_and_on_two_streams(ops):
    cases = [product_case(ops, M, 1024, 1024, "", M) for M in (2, 50, 1000)]
    want = [ops.linear_fp8(*c) for c in cases]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [ops.linear_fp8(*c) for c in cases]
        again = [ops.quantize_fp8(o)[0] for o in got]
    side = torch.cuda.Stream()
    for _ in range(3):
        for o in got:
            o.zero_()
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            other = [ops.linear_fp8(*c) for c in cases]
        torch.cuda.synchronize()
        for a, b, c, q in zip(got, want, other, again):
            assert torch.equal(a, b) and torch.equal(c, b)
            assert torch.equal(q.float(), ops.quantize_fp8(b)[0].float())
    ops.check_status()


def test_a_row_does_not_depend_on_the_batch(ops):
    """Within the sizes that run on one arrangement the sum over k has one order."""
    x, xs, w, ws = product_case(ops, 64, 1000, 4096, "", 21)
    full = ops.linear_fp8(x, xs, w, ws)
    assert torch.equal(ops.linear_fp8(x[40:], xs[40:], w, ws), full[40:])


def test_refusals(ops):
    x, xs, w, ws = product_case(ops, 4, 256, 256, "", 31)
    cpu = torch.zeros(4, 256)
    for call in (lambda: ops.quantize_fp8(cpu), lambda: ops.quantize_fp8(cpu.to(DEV).half()), lambda: ops.quantize_fp8(cpu.to(DEV), 64),
                 lambda: ops.quantize_fp8(cpu.to(DEV)[0]), lambda: ops.quantize_fp8(cpu.to(DEV).t()),
                 lambda: ops.quantize_fp8(torch.zeros(2, 4, 0, device=DEV)), lambda: ops.quantize_fp8(torch.zeros(2, 8, 4, device=DEV).transpose(1, 2)),
                 lambda: ops.linear_fp8(x.float(), xs, w, ws), lambda: ops.linear_fp8(x, xs, w.float(), ws),
                 lambda: ops.linear_fp8(x, xs[:3], w, ws), lambda: ops.linear_fp8(x, xs, w, ws[:1]),
                 lambda: ops.linear_fp8(x, xs, w, ws[:, :1]), lambda: ops.linear_fp8(x, xs.double(), w, ws),
                 lambda: ops.linear_fp8(x[:, :255], xs, w, ws), lambda: ops.linear_fp8(x[:, 1:], xs, w[:, 1:], ws),
                 lambda: ops.linear_fp8(x, xs, w, ws, out_dtype=torch.float16), lambda: ops.linear_fp8(x.cpu(), xs, w, ws),
                 lambda: ops.linear_fp8(x, xs, w.t(), ws), lambda: ops.linear_fp8(x[:, :100].contiguous(), xs[:, :1], w[:, :100], ws[:, :1])):
        with pytest.raises(ops.KernelError):
            call()
    assert ops.linear_fp8(x[:0], xs[:0], w, ws).shape == (0, 256)
