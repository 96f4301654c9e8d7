"""A whole routed feed-forward of a few tokens in two kernels, against 64-bit arithmetic, token by token.

The tokens' numbers are multiples of 1/8 and the router's of 1/256, so every logit is exact in float32 whatever the order of its
sum: the choice of experts is defined exactly, ties among equal logits included (the lower number first).

Tolerance of an output, from 64-bit magnitudes: u is rounded to bfloat16 (half a step, 2^-8 of it) after products whose float32 sums of
d numbers are off by at most 2 d 2^-24 of their magnitudes (the tensor core may cut off where float32 rounds) and an activation whose slope is
at most 1.2; the weighted sum over top * ff numbers likewise; a weight w is off by 2^-20 of it (float32 exp, a sum of at most 1,024 terms);
the result is rounded to bfloat16."""
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


def generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def experts_8bit(ops, w, scales, g):
    q, s = ops.quantize_fp8(w, 128)
    if scales == "float32":
        s = s.float() * (1 + torch.rand(s.shape, device=DEV, generator=g))
    values = q.double() * s.double().repeat_interleave(128, 1)[:, :w.shape[1]].repeat_interleave(128, 2)[:, :, :w.shape[2]]
    return q, s, values


def layer_case(ops, n, E, identity, top, d, ff, glu, weights, rule, groups, keep, shared, corrected, seed=0):
    g = generator(seed + 131 * n + E + d)
    many = E + identity
    h = (torch.randint(-8, 9, (n, d), device=DEV, generator=g) / 8).to(torch.bfloat16)
    router = (torch.randint(-4, 5, (many + int(shared == "gated"), d), device=DEV, generator=g) / 256).to(torch.bfloat16)
    correction = torch.randint(-8, 9, (many,), device=DEV, generator=g) / 64 if corrected else None
    up = torch.randn(E, (2 if glu else 1) * ff, d, device=DEV, generator=g) * d ** -0.5 * 2
    down = torch.randn(E, d, ff, device=DEV, generator=g) * ff ** -0.5
    add = torch.randn(n, d, device=DEV, generator=g).to(torch.bfloat16) if shared else None
    kw = dict(glu=glu, softmax_top=rule == "softmax_top", softmax=rule == "softmax", group_max=rule == "softmax",
              renormalise=rule == "softmax", add=add, add_gated=shared == "gated", identity=identity)
    if weights == "bfloat16":
        up, down = up.to(torch.bfloat16), down.to(torch.bfloat16)
        upv, downv = up.double(), down.double()
    else:
        up, kw["up_scale"], upv = experts_8bit(ops, up, weights, g)
        down, kw["down_scale"], downv = experts_8bit(ops, down, weights, g)
    scale = 2.5 if rule == "sigmoid" else 1.0
    args = (h, router, correction, groups, keep, top, scale, up, down)
    return args, kw, upv, downv


def choice_of(z, rule, correction, groups, keep, top, scale):
    """(numbers, weights) of one token's experts from its exact logits."""
    many = len(z)
    c = correction if correction is not None else [0.0] * many
    if rule == "softmax_top":
        choice = [a + b for a, b in zip(z, c)]
    elif rule == "sigmoid":
        s = [1 / (1 + math.exp(-a)) for a in z]
        choice = [a + b for a, b in zip(s, c)]
    else:
        m = max(z)
        t = sum(math.exp(a - m) for a in z)
        s = [math.exp(a - m) / t for a in z]
        choice = [a + b for a, b in zip(s, c)] if correction is not None else list(z)
    per = many // groups
    if groups > 1 and keep < groups:
        worth = []
        for k in range(groups):
            best = sorted(choice[k * per:(k + 1) * per], reverse=True)
            worth.append(best[0] if rule == "softmax" or per == 1 else best[0] + best[1])
        kept = sorted(range(groups), key=lambda k: (-worth[k], k))[:keep]
        choice = [v if e // per in kept else -math.inf for e, v in enumerate(choice)]
    ids = sorted(range(many), key=lambda e: (-choice[e], e))[:top]
    if rule == "softmax_top":
        w = [math.exp(choice[e] - choice[ids[0]]) for e in ids]
        return ids, [v / sum(w) * scale for v in w]
    w = [s[e] for e in ids]
    return ids, [v / (sum(w) if rule == "softmax" else 1.0) * scale for v in w]


def check_layer(out, args, kw, upv, downv, rule, rows=None):
    h, router, correction, groups, keep, top, scale, _, _ = args
    E, ff, d, many = upv.shape[0], downv.shape[2], h.shape[1], upv.shape[0] + kw["identity"]
    z, of_squares, all_squares = (h.double() @ router.double().t()), 0.0, 0.0
    corr = correction.double().tolist() if correction is not None else None
    assert out.dtype == torch.bfloat16 and out.shape == h.shape
    for t in rows if rows is not None else range(h.shape[0]):
        ids, w = choice_of(z[t, :many].tolist(), rule, corr, groups, keep, top, scale)
        want, room = torch.zeros(d, dtype=torch.float64, device=DEV), torch.zeros(d, dtype=torch.float64, device=DEV)
        x = h[t].double()
        for e, we in zip(ids, w):
            if e >= E:
                want += we * x
                room += we * x.abs() * 2.0 ** -19
                continue
            v, room_v = upv[e] @ x, (upv[e].abs() @ x.abs()) * 2 * d * 2.0 ** -24
            if kw["glu"]:
                a = torch.sigmoid(v[:ff]) * v[:ff]
                u = a * v[ff:]
                room_u = 1.2 * room_v[:ff] * v[ff:].abs() + a.abs() * room_v[ff:]
            else:
                u = 0.5 * v * torch.special.erfc(-v / math.sqrt(2))
                room_u = 1.2 * room_v
            room_u = room_u + u.abs() * (2.0 ** -8 + 2.0 ** -20) + 2.0 ** -20 * v[:ff].abs()       # erff and expf near zero: of the argument
            want += we * (downv[e] @ u)
            room += we * (downv[e].abs() @ room_u) + we * (downv[e].abs() @ u.abs()) * (2 * top * ff * 2.0 ** -24 + 2.0 ** -19)
        if kw["add"] is not None:
            a = kw["add"][t].double() * (torch.sigmoid(z[t, many]) if kw["add_gated"] else 1)
            want += a
            room += a.abs() * 2.0 ** -20
        room += want.abs() * 2.0 ** -8 + 2.0 ** -126
        off = (out[t].double() - want).abs()
        assert bool((off <= room).all()), (t, float((off / room).max()))
        of_squares, all_squares = of_squares + float((off ** 2).sum()), all_squares + float((want ** 2).sum())
    return math.sqrt(of_squares / max(all_squares, 1e-300))


CASES = [
    # n, E, identity, top, d, ff, glu, rule, groups, keep, shared, corrected
    (1, 8, 0, 2, 64, 32, True, "softmax_top", 1, 1, None, True),
    (1, 64, 0, 6, 2048, 1408, True, "softmax_top", 1, 1, None, True),
    (2, 5, 0, 5, 48, 16, False, "sigmoid", 1, 1, None, False),
    (3, 16, 4, 3, 272, 144, True, "softmax", 1, 1, "gated", True),
    (7, 64, 0, 4, 512, 96, False, "sigmoid", 8, 4, None, True),
    (8, 12, 0, 1, 1040, 720, True, "softmax", 4, 1, "plain", False),
    (9, 3, 2, 2, 128, 256, True, "softmax", 1, 1, None, False),
    (16, 2, 0, 2, 160, 400, False, "softmax_top", 1, 1, "plain", True),
    (17, 64, 0, 6, 768, 208, True, "sigmoid", 8, 4, "gated", True),
    (23, 20, 0, 3, 400, 528, True, "sigmoid", 4, 2, None, True),
    (40, 1, 0, 1, 96, 64, True, "softmax_top", 1, 1, None, False),
    (64, 1, 1, 2, 256, 128, False, "softmax", 1, 1, "gated", False),
    (61, 64, 16, 6, 2048, 1408, True, "softmax", 8, 4, "gated", True),
    (64, 100, 0, 8, 176, 80, False, "softmax_top", 1, 1, None, True),
    (5, 1000, 24, 8, 64, 16, True, "sigmoid", 1, 1, None, True),
    (4, 40, 0, 8, 4096, 1024, True, "softmax_top", 1, 1, None, True),
    (5, 3, 0, 1, 1024, 4096, False, "sigmoid", 1, 1, "plain", False),
    (33, 24, 8, 4, 1152, 896, True, "softmax", 1, 1, None, True),
    (48, 2, 0, 1, 512, 2048, True, "softmax_top", 1, 1, "gated", True),
    (64, 300, 0, 5, 2048, 160, True, "softmax_top", 1, 1, None, True),
    (64, 2, 0, 1, 128, 14336, True, "softmax_top", 1, 1, None, True),
    (20, 3, 0, 2, 256, 8336, False, "softmax_top", 1, 1, None, True),
    (2, 2, 0, 2, 9232, 4112, True, "softmax", 1, 1, "plain", True),
]


@pytest.mark.parametrize("weights", ["bfloat16", "e8m0", "float32"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_layer(ops, case, weights):
    n, E, identity, top, d, ff, glu, rule, groups, keep, shared, corrected = case
    args, kw, upv, downv = layer_case(ops, n, E, identity, top, d, ff, glu, weights, rule, groups, keep, shared, corrected)
    out = ops.moe_layer(*args, **kw)
    ops.check_status()
    check_layer(out, args, kw, upv, downv, rule, rows=range(0, n, max(1, n * d // 40000)))
    assert torch.equal(ops.moe_layer(*args, **kw), out), "the same call gives the same bits"


@pytest.mark.parametrize("glu,d,ff", [(True, 72, 40), (False, 200, 88), (False, 1032, 24), (True, 8, 8)])
def test_bfloat16_sizes_that_are_multiples_of_eight(ops, glu, d, ff):
    args, kw, upv, downv = layer_case(ops, 6, 9, 0, 3, d, ff, glu, "bfloat16", "softmax_top", 1, 1, None, True)
    check_layer(ops.moe_layer(*args, **kw), args, kw, upv, downv, "softmax_top")


def test_every_8bit_number(ops):
    """All finite codes, the smallest ones too, as weights of both products."""
    codes = torch.tensor([c for c in range(256) if c & 0x7F != 0x7F], dtype=torch.uint8, device=DEV)
    g = generator(9)
    E, d, ff = 2, 256, 128
    up = codes[torch.randint(0, 254, (E, ff, d), device=DEV, generator=g)].view(torch.float8_e4m3fn)
    down = codes[torch.randint(0, 254, (E, d, ff), device=DEV, generator=g)].view(torch.float8_e4m3fn)
    up[:, :16, :] = codes[(torch.arange(d, device=DEV) % 16)].view(torch.float8_e4m3fn)           # 0 to 2^-6: the subnormal ones alone
    su, sd = torch.full((E, 1, 2), 2.0 ** -9, device=DEV), torch.full((E, 2, 1), 2.0 ** -9, device=DEV)
    h = (torch.randint(-8, 9, (4, d), device=DEV, generator=g) / 8).to(torch.bfloat16)
    router = (torch.randint(-4, 5, (E, d), device=DEV, generator=g) / 256).to(torch.bfloat16)
    args = (h, router, None, 1, 1, 2, 1.0, up, down)
    kw = dict(glu=False, softmax_top=True, up_scale=su, down_scale=sd, add=None, add_gated=False, identity=0)
    check_layer(ops.moe_layer(*args, **kw), args, kw, up.double() * 2.0 ** -9, down.double() * 2.0 ** -9, "softmax_top")


@pytest.mark.parametrize("weights", ["bfloat16", "float32"])
def test_a_token_of_nan_stays_in_its_row(ops, weights):
    for n in (4, 30):
        args, kw, upv, downv = layer_case(ops, n, 16, 0, 4, 256, 64, True, weights, "softmax_top", 1, 1, None, True)
        want = ops.moe_layer(*args, **kw)
        args[0][1, 7] = math.nan
        out = ops.moe_layer(*args, **kw)
        assert bool(torch.isnan(out[1]).all())
        others = [t for t in range(n) if t != 1]
        check_layer(out, args, kw, upv, downv, "softmax_top", rows=others)
        assert not bool(torch.isnan(out[others].float()).any()) and out.shape == want.shape


def test_steps_whose_choices_are_all_identity_experts(ops):
    """No expert is read; tokens are weighted copies of themselves (and of ``add``)."""
    for n, shared in ((1, None), (7, "gated"), (40, "plain")):
        args, kw, upv, downv = layer_case(ops, n, 6, 10, 3, 144, 48, True, "bfloat16", "softmax", 1, 1, shared, True)
        args[2][:] = 0
        args[2][6:] = 4
        check_layer(ops.moe_layer(*args, **kw), args, kw, upv, downv, "softmax")


@pytest.mark.parametrize("weights", ["bfloat16", "e8m0"])
def test_tokens_of_very_different_sizes(ops, weights):
    """Tokens from 2^-100 to 2^60: a router that is zero for them makes the choice independent of the sizes."""
    args, kw, upv, downv = layer_case(ops, 20, 8, 0, 2, 256, 128, False, weights, "softmax_top", 1, 1, None, True)
    h, router = args[0], args[1]
    router.zero_()
    h *= torch.exp2(torch.linspace(-100, 60, 20, device=DEV).round())[:, None].to(torch.bfloat16)
    check_layer(ops.moe_layer(*args, **kw), args, kw, upv, downv, "softmax_top")


def test_a_nan_among_the_weights_shows_in_its_column(ops):
    for weights in ("bfloat16", "float32"):
        args, kw, upv, downv = layer_case(ops, 3, 2, 0, 2, 256, 128, True, weights, "softmax_top", 1, 1, None, True)
        down = args[8]
        if weights == "bfloat16":
            down[1, 77, 5] = math.nan
        else:
            down.view(torch.uint8)[1, 77, 5] = 0x7F
        out = ops.moe_layer(*args, **kw).float()
        assert bool(torch.isnan(out[:, 77]).all()) and int(torch.isnan(out).sum()) == 3


def test_experts_beyond_32_bits(ops):
    """Stacked weights of more than 2^31 numbers: the last experts."""
    E, d, ff = 72, 2048, 8192
    args, kw, _, _ = layer_case(ops, 3, 1, 0, 1, d, 64, True, "bfloat16", "softmax_top", 1, 1, None, False)
    g = generator(3)
    up, down = torch.zeros(E, 2 * ff, d, device=DEV, dtype=torch.bfloat16), torch.zeros(E, d, ff, device=DEV, dtype=torch.bfloat16)
    up[-2:] = torch.randn(2, 2 * ff, d, device=DEV, generator=g) * d ** -0.5
    down[-2:] = torch.randn(2, d, ff, device=DEV, generator=g) * ff ** -0.5
    correction = torch.zeros(E, device=DEV)
    correction[-2:] = torch.tensor([9.0, 8.5], device=DEV)
    router = torch.zeros(E, d, device=DEV, dtype=torch.bfloat16)
    args = (args[0], router, correction, 1, 1, 2, 1.0, up, down)
    out = ops.moe_layer(*args, **kw)
    small = (args[0], router[-2:].contiguous(), correction[-2:].contiguous(), 1, 1, 2, 1.0, up[-2:].contiguous(), down[-2:].contiguous())
    check_layer(out, small, kw, up[-2:].double(), down[-2:].double(), "softmax_top")


def test_agrees_with_the_separate_operators(ops):
    """moe_layer against moe_route and moe_experts: both round the same intermediate results to bfloat16."""
    args, kw, _, _ = layer_case(ops, 24, 64, 16, 6, 512, 256, True, "bfloat16", "softmax", 1, 1, "gated", True)
    h, router, correction, groups, keep, top, scale, up, down = args
    ids, wts, gate = ops.moe_route(h, router, correction, groups, keep, top, scale, softmax=True, group_max=True, renormalise=True, extra_rows=1)
    want = ops.moe_experts(h, ids, wts, up, down, h.dtype, glu=True, add=kw["add"], add_gate=gate, identity=True)
    torch.testing.assert_close(ops.moe_layer(*args, **kw).float(), want.float(), rtol=2e-2, atol=2e-2)


def test_layers_replayed_and_on_two_streams(ops):
    cases = [layer_case(ops, n, 32, 0, 4, 512, 256, True, w, "softmax_top", 1, 1, None, True)[:2] for n, w in ((1, "bfloat16"), (20, "e8m0"))]
    want = [ops.moe_layer(*a, **k) for a, k in cases]
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, [ops.moe_layer(*a, **k) for a, k in cases]))
    side = torch.cuda.Stream()
    for _ in range(5):
        for _, got in graphs:
            for o in got:
                o.zero_()
        torch.cuda.synchronize()
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
            other = [ops.moe_layer(*a, **k) for a, k in cases]
        torch.cuda.synchronize()
        for got in (graphs[0][1], graphs[1][1], other):
            for a, b in zip(got, want):
                assert torch.equal(a, b)
    ops.check_status()


def test_a_decode_step_of_8bit_products(ops):
    """As used together: quantise, project, gate, project, and the routed layer on the result, all in 8-bit weights."""
    g = generator(77)
    n, d, ff = 6, 512, 384
    x = torch.randn(n, d, device=DEV, generator=g).to(torch.bfloat16)
    w13, w2 = torch.randn(2 * ff, d, device=DEV, generator=g) * d ** -0.5, torch.randn(d, ff, device=DEV, generator=g) * ff ** -0.5
    (q13, s13), (q2, s2) = ops.quantize_fp8(w13, 128), ops.quantize_fp8(w2, 128)
    args, kw, upv, downv = layer_case(ops, n, 8, 0, 2, d, 128, True, "e8m0", "softmax_top", 1, 1, None, True)
    qx, sx = ops.quantize_fp8(x)
    u = ops.linear_fp8(qx, sx, q13, s13, w_is_parameter=True)
    m = torch.empty(n, ff, device=DEV, dtype=torch.bfloat16)
    ops.silu_mul(u, m)
    qm, sm = ops.quantize_fp8(m)
    y = ops.linear_fp8(qm, sm, q2, s2, w_is_parameter=True)
    # every link against the formula on the link before (each link's own tests hold the tolerances)
    v = lambda q, s, b: q.double() * s.double().repeat_interleave(b, 0)[:q.shape[0]].repeat_interleave(128, 1)[:, :q.shape[1]]
    torch.testing.assert_close(u.double(), v(qx, sx, 1) @ v(q13, s13, 128).t(), rtol=2.0 ** -7, atol=2.0 ** -10)
    torch.testing.assert_close(m.double(), torch.nn.functional.silu(u[:, :ff].double()) * u[:, ff:].double(), rtol=2.0 ** -7, atol=2.0 ** -10)
    torch.testing.assert_close(y.double(), v(qm, sm, 1) @ v(q2, s2, 128).t(), rtol=2.0 ** -7, atol=2.0 ** -10)
    h = (y.float() * 8).round().clamp(-16, 16) / 8          # exact logits
    args = (h.to(torch.bfloat16),) + args[1:]
    check_layer(ops.moe_layer(*args, **kw), args, kw, upv, downv, "softmax_top")


@pytest.mark.parametrize("weights", ["bfloat16", "e8m0", "float32"])
@pytest.mark.parametrize("n,E,top", [(16, 8, 3), (32, 24, 2), (60, 2, 1), (60, 30, 4)])
def test_activations_keep_their_precision(ops, weights, n, E, top):
    """What is left of the error is the result's rounding: 2^-8 at most at a significand of 1, evenly spread, 2^-8 / sqrt(3) / significand over
    significands of equal logarithms: 2^-8 sqrt(1/3) sqrt(3/8 / log 2) = 1.66e-3, over 8,192 numbers and more within 3 in 100.  8-bit experts: and two
    e4m3 numbers for each of u, at most 2^-9 off at a significand of 1, so half of that: 1.86e-3 in all; 16 bits of u add nothing to see
    (u rounded to bfloat16 would make it 2.3e-3)."""
    args, kw, upv, downv = layer_case(ops, n, E, 0, top, 512, 256, True, weights, "softmax_top", 1, 1, None, True)
    off = check_layer(ops.moe_layer(*args, **kw), args, kw, upv, downv, "softmax_top")
    assert off <= (1.66e-3 if weights == "bfloat16" else 1.86e-3) * 1.05


def test_more_choices_than_fit_are_refused(ops):
    h = torch.zeros(64, 64, device=DEV, dtype=torch.bfloat16)
    router, w_up = torch.zeros(512, 64, device=DEV, dtype=torch.bfloat16), torch.zeros(512, 32, 64, device=DEV, dtype=torch.bfloat16)
    w_down = torch.zeros(512, 64, 32, device=DEV, dtype=torch.bfloat16)
    with pytest.raises(ops.KernelError, match="do not fit"):
        ops.moe_layer(h, router, None, 1, 1, 512, 1.0, w_up, w_down)
    ops.check_status()


def test_refusals(ops):
    args, kw, _, _ = layer_case(ops, 4, 8, 0, 2, 64, 32, True, "e8m0", "softmax_top", 1, 1, "plain", True)
    assert ops.moe_layer(*args, **kw).shape == (4, 64)
    assert ops.moe_layer(args[0][:0], *args[1:], **dict(kw, add=kw["add"][:0])).shape == (0, 64)
    h, router, correction, groups, keep, top, scale, up, down = args

    def refused(new=None, **other):
        a = list(args)
        for i, v in (new or {}).items():
            a[i] = v
        with pytest.raises(ops.KernelError):
            ops.moe_layer(*a, **dict(kw, **other))

    refused({0: h.float()})
    refused({0: h.cpu()})
    refused({0: torch.zeros(65, 64, device=DEV, dtype=torch.bfloat16)}, add=None)
    refused({0: torch.zeros(4, 128, device=DEV, dtype=torch.bfloat16)[:, ::2]})
    refused({0: h[:, :48].contiguous()})
    refused({1: router[:7]})
    refused({1: router.float()})
    refused({2: correction[:7]})
    refused({3: 3})
    refused({4: 2})
    refused({5: 9})
    refused({5: 0})
    refused({7: up.to(torch.bfloat16)})
    refused({7: up[:, :62]})
    refused({8: down[:, :32]})
    refused(up_scale=None)
    refused(up_scale=kw["up_scale"].float())
    refused(down_scale=kw["down_scale"][:1])
    refused(add=kw["add"].float())
    refused(add=None, add_gated=True)
    refused(softmax=True)
    refused(identity=3)
    refused({7: torch.zeros(8, 64, 72, device=DEV, dtype=torch.float8_e4m3fn), 8: torch.zeros(8, 72, 32, device=DEV, dtype=torch.float8_e4m3fn),
             0: torch.zeros(4, 72, device=DEV, dtype=torch.bfloat16), 1: torch.zeros(8, 72, device=DEV, dtype=torch.bfloat16)}, add=None)
    bf = dict(kw, up_scale=None, down_scale=None)
    with pytest.raises(ops.KernelError):
        ops.moe_layer(h, router, correction, 1, 1, 2, 1.0, up.to(torch.bfloat16), down.to(torch.bfloat16), **dict(kw))
    assert ops.moe_layer(h, router, correction, 1, 1, 2, 1.0, up.to(torch.bfloat16), down.to(torch.bfloat16), **bf).shape == (4, 64)
