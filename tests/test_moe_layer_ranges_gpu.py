"""The routed layer of a few tokens at the ends of float32's range: tokens of any size, experts whose weights bring the result back.
The checks and their tolerances are those of ``test_moe_layer_gpu.py``."""
import pytest
import torch
from test_moe_layer_gpu import check_layer, layer_case, ops  # noqa: F401  (ops: a fixture)

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def scaled_case(ops, n, weights, up_exp, down_exp, ff=128):
    """GELU experts whose weights are moved by powers of two, tokens that all experts see alike (a router of zeros)."""
    args, kw, upv, downv = layer_case(ops, n, 8, 0, 2, 256, ff, False, weights, "softmax_top", 1, 1, None, True)
    args[1].zero_()
    for i, name, e in ((7, "up_scale", up_exp), (8, "down_scale", down_exp)):
        if weights == "bfloat16":
            args[i].mul_(2.0 ** e)
        else:
            kw[name] = (kw[name].float() * 2.0 ** e).to(kw[name].dtype)
    return args, kw, upv * 2.0 ** up_exp, downv * 2.0 ** down_exp


@pytest.mark.parametrize("weights", ["bfloat16", "e8m0", "float32"])
@pytest.mark.parametrize("h_exp,up_exp,down_exp", [(112, -30, 0), (118, -30, 0), (123, -110, 0), (90, 26, -60), (123, -5, -60), (-118, 40, 0)])
@pytest.mark.parametrize("n", [4, 20, 50])
def test_tokens_at_the_ends_of_the_range(ops, n, h_exp, up_exp, down_exp, weights):  # noqa: F811
    """u and the result are ordinary float32 numbers, whatever the sizes of the factors on the way."""
    args, kw, upv, downv = scaled_case(ops, n, weights, up_exp, down_exp)
    args[0].mul_(2.0 ** h_exp)
    check_layer(ops.moe_layer(*args, **kw), args, kw, upv, downv, "softmax_top")
    ops.check_status()


@pytest.mark.parametrize("weights", ["e8m0", "float32"])
def test_large_tokens_beside_ordinary_ones(ops, weights):  # noqa: F811
    """Also several windows of scales of u (more than 64 blocks of 64) and tokens of zeros."""
    args, kw, upv, downv = scaled_case(ops, 20, weights, -60, 0, ff=4352)
    args[0][3:] *= 2.0 ** 60
    args[0][9:] *= 2.0 ** 58
    args[0][15] = 0
    check_layer(ops.moe_layer(*args, **kw), args, kw, upv, downv, "softmax_top")
    ops.check_status()


@pytest.mark.parametrize("kind", ["e8m0", "float32"])
def test_a_block_of_nan_among_the_experts_shows_where_it_is_taken(ops, kind):  # noqa: F811
    for name in ("up_scale", "down_scale"):
        args, kw, upv, downv = layer_case(ops, 24, 8, 0, 2, 256, 128, True, kind, "softmax_top", 1, 1, None, False)
        ids, _ = ops.moe_route(args[0], args[1], args[2], 1, 1, 2, 1.0, softmax_top=True)
        e = int(ids[0, 0])
        if kind == "e8m0":
            kw[name].view(torch.uint8)[e, 0, 0] = 255
        else:
            kw[name][e, 0, 0] = float("nan")
        out = ops.moe_layer(*args, **kw)
        taken = (ids == e).any(dim=1)
        assert 0 < int(taken.sum()) < 24
        assert bool(torch.isnan(out[taken][:, :128]).all()) and not bool(torch.isnan(out[~taken]).any())
        check_layer(out, args, kw, upv, downv, "softmax_top", rows=torch.nonzero(~taken)[:, 0].tolist())
