"""The choice of many experts and its options, for ``moe_route`` and ``moe_layer``, against 64-bit arithmetic.

Logits are exact in float32 (tokens in multiples of 1/8, routers of 1/256), and so are corrections where they are added to logits: the choice is
defined exactly, equal logits included.  A weight is off by 2^-19 of it at most (float32 exp, a division, a sum of at most 1,024 terms)."""
import math

import pytest
import test_moe_layer_gpu as layer
import torch
from test_moe_layer_gpu import generator, layer_case, ops  # noqa: F401  (ops: a fixture)

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def choice(z, rule, correction, groups, keep, top, scale, renormalise, group_max):
    """(numbers, weights) of one token's experts from its exact logits."""
    many = len(z)
    if rule == "softmax_top":
        score = by = [a + b for a, b in zip(z, correction or [0.0] * many)]
    elif rule == "sigmoid":
        score = by = [1 / (1 + math.exp(-a)) for a in z]
    else:
        e = [math.exp(a - max(z)) for a in z]
        score, by = [a / sum(e) for a in e], z
    per = many // groups
    worth = []
    for g in range(groups):
        best = sorted(by[g * per:(g + 1) * per], reverse=True)
        worth.append(best[0] if group_max or per == 1 else best[0] + best[1])
    kept = sorted(range(groups), key=lambda g: (-worth[g], g))[:keep]
    ids = sorted((e for e in range(many) if e // per in kept), key=lambda e: (-by[e], e))[:top]
    w = [score[e] for e in ids]
    if rule == "softmax_top":
        w = [math.exp(a - max(w)) for a in w]
    if rule == "softmax_top" or renormalise:
        w = [a / sum(w) for a in w]
    return ids, [a * scale for a in w]


RULES = [("sigmoid", False, 2.5), ("sigmoid", True, 1.0), ("sigmoid", True, 2.5), ("softmax", False, 1.5), ("softmax", True, 0.5),
         ("softmax_top", False, 0.75)]


@pytest.mark.parametrize("rule,renormalise,scale", RULES)
@pytest.mark.parametrize("E,groups,keep,top", [(64, 1, 1, 9), (64, 1, 1, 32), (64, 1, 1, 33), (64, 1, 1, 64), (128, 8, 4, 40), (1024, 1, 1, 40), (1000, 4, 2, 100)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [3, 70])
def test_route_to_many_experts(ops, n, dtype, E, groups, keep, top, rule, renormalise, scale):  # noqa: F811
    g = generator(E + top + n)
    h = (torch.randint(-8, 9, (n, 256), device=DEV, generator=g) / 8).to(dtype)
    router = (torch.randint(-4, 5, (E, 256), device=DEV, generator=g) / 256).to(dtype)
    ids, wts = ops.moe_route(h, router, None, groups, keep, top, scale, softmax_top=rule == "softmax_top", softmax=rule == "softmax",
                             renormalise=renormalise)[:2]
    z = (h.double() @ router.double().t()).tolist()
    for t in range(0, n, 23):
        want_ids, want = choice(z[t], rule, None, groups, keep, top, scale, renormalise, False)
        assert ids[t].tolist() == want_ids
        off = (wts[t].double().cpu() - torch.tensor(want, dtype=torch.float64)).abs()
        assert bool((off <= 2.0 ** -19 * torch.tensor(want)).all())


def checked(ops, monkeypatch, args, kw, upv, downv, rule, renormalise, rows):  # noqa: F811
    monkeypatch.setattr(layer, "choice_of", lambda z, r, c, groups, keep, top, scale:
                        choice(z, r, c, groups, keep, top, scale, renormalise, kw["group_max"]))
    out = ops.moe_layer(*args, **kw)
    ops.check_status()
    layer.check_layer(out, args, kw, upv, downv, rule, rows=rows)
    return out


@pytest.mark.parametrize("rule,renormalise,scale", RULES)
@pytest.mark.parametrize("n,E,identity,groups,keep,top,group_max", [(5, 32, 0, 4, 2, 4, False), (20, 24, 8, 4, 3, 5, True), (3, 64, 0, 1, 1, 9, False),
                                                                    (5, 64, 0, 1, 1, 40, False), (40, 40, 0, 1, 1, 33, False)])
def test_rules_of_the_layer(ops, monkeypatch, n, E, identity, groups, keep, top, group_max, rule, renormalise, scale):  # noqa: F811
    args, kw, upv, downv = layer_case(ops, n, E, identity, top, 256, 64, True, "bfloat16", rule, groups, keep, None, False)
    args = args[:6] + (scale,) + args[7:]
    kw.update(renormalise=renormalise, group_max=group_max)
    checked(ops, monkeypatch, args, kw, upv, downv, rule, renormalise, range(0, n, 7))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("top", [4, 35])
def test_corrections_of_either_type(ops, monkeypatch, top, dtype):  # noqa: F811
    args, kw, upv, downv = layer_case(ops, 6, 48, 0, top, 128, 64, True, "e8m0", "softmax_top", 1, 1, None, True)
    args = args[:2] + (args[2].to(dtype),) + args[3:]
    checked(ops, monkeypatch, args, kw, upv, downv, "softmax_top", False, range(6))
    ids, _ = ops.moe_route(args[0], args[1], args[2], 1, 1, top, 1.0, softmax_top=True)[:2]
    z = (args[0].double() @ args[1].double().t()).tolist()
    for t in range(6):
        assert ids[t].tolist() == choice(z[t], "softmax_top", args[2].tolist(), 1, 1, top, 1.0, False, False)[0]


@pytest.mark.parametrize("rule", ["sigmoid", "softmax", "softmax_top"])
def test_a_token_of_nan_among_many_choices(ops, monkeypatch, rule):  # noqa: F811
    """It still takes every expert at most once, so that no expert gets more entries than there are tokens."""
    for n, top in ((5, 40), (33, 36)):
        args, kw, upv, downv = layer_case(ops, n, 48, 0, top, 128, 64, False, "bfloat16", rule, 1, 1, None, False)
        args[0][2, 5] = math.nan
        out = checked(ops, monkeypatch, args, kw, upv, downv, rule, kw["renormalise"], [t for t in range(0, n, 8) if t != 2])
        assert bool(torch.isnan(out[2]).all()) and int(torch.isnan(out).sum()) == out.shape[1]


def test_as_many_choices_as_fit(ops, monkeypatch):  # noqa: F811
    """64 tokens, 64 experts in 8 bits with inner sizes of 4,096: lists of 60 choices fit beside three stages, of 61 they do not."""
    args, kw, upv, downv = layer_case(ops, 64, 64, 0, 60, 64, 4096, False, "e8m0", "softmax_top", 1, 1, None, True)
    checked(ops, monkeypatch, args, kw, upv, downv, "softmax_top", False, range(0, 64, 21))
    with pytest.raises(ops.KernelError, match="do not fit"):
        ops.moe_layer(*(args[:5] + (61,) + args[6:]), **kw)


@pytest.mark.parametrize("fp8,E,most", [(1, 64, 60), (1, 256, 55), (1, 1024, 37), (0, 64, 64), (0, 256, 167), (0, 1024, 149)])
def test_the_documented_numbers_of_choices(ops, fp8, E, most):  # noqa: F811
    size = ops.load_library(features=("moe",)).bspec_moe_layer_scratch
    for ff in (4096, 14336):
        assert size(64, 64, ff, most, fp8, E) > 0 and (most == E or size(64, 64, ff, most + 1, fp8, E) == 0)
        assert size(15, 64, ff, E, fp8, E) > 0


@pytest.mark.parametrize("weights", ["bfloat16", "e8m0"])
def test_a_longer_step_goes_as_its_refusal_says(ops, weights):  # noqa: F811
    args, kw, upv, downv = layer_case(ops, 150, 16, 0, 3, 128, 64, True, weights, "softmax_top", 1, 1, "plain", True)
    with pytest.raises(ops.KernelError, match="64 tokens at a time, or with bfloat16 experts through moe_route and moe_experts"):
        ops.moe_layer(*args, **kw)
    parts = [ops.moe_layer(args[0][i:i + 64], *args[1:], **dict(kw, add=kw["add"][i:i + 64])) for i in range(0, 150, 64)]
    layer.check_layer(torch.cat(parts), args, kw, upv, downv, "softmax_top", rows=range(0, 150, 13))
    with pytest.raises(ops.KernelError, match="fewer tokens at a time"):
        wide = torch.zeros(64, 64, device=DEV, dtype=torch.bfloat16)
        ops.moe_layer(wide, torch.zeros(512, 64, device=DEV, dtype=torch.bfloat16), None, 1, 1, 512, 1.0,
                      torch.zeros(512, 32, 64, device=DEV, dtype=torch.bfloat16), torch.zeros(512, 64, 32, device=DEV, dtype=torch.bfloat16))
