"""What products with 8-bit weights and a routed feed-forward of a few tokens cost, as cases that can be timed and checked.

Three operators, each in its plain form (elementary torch operations in 32 bits) and as the call a user makes:

``quantize``  ``ops.quantize_fp8``: a matrix in 8-bit floating point (4 exponent bits, 3 of fraction) with a power of two for
              every 128 numbers of a row (activations) or every block of 128 x 128 (weights, once, at load).
``linear``    ``ops.linear_fp8``: x w^T of two such matrices; the scales are powers of two in 8 bits, or float32 numbers as
              checkpoints in this format often keep them.
``moe``       ``ops.moe_layer``: a whole routed feed-forward (router, choice, experts, weighted sum) for a few tokens, with
              experts in bfloat16 or in 8 bits with blocks of 128 x 128.

Sizes come from the configurations this package ships (Llama 8B: 4,096 wide, 14,336 inside; the 2,048 wide designs with 64
experts of 1,408, 6 per token), with ragged ones between them.
"""
import math

import torch

own = False
DEVICE = "cuda:0"
BLOCK = 128
LARGEST = 2 * 2048 * 28672 * 4096        # multiply-adds times two of the largest listed product


def listed():
    return [
        # one decoding request: the activations of one token before a product; latency alone
        dict(name="quantize-x1", kind="quantize", rows=1, cols=4096, dtype="bfloat16", block_rows=1),
        # a prompt's rows before the down projection at 8B sizes
        dict(name="quantize-prompt-2048", kind="quantize", rows=2048, cols=14336, dtype="bfloat16", block_rows=1),
        # float32 weights brought into 8 bits at load, sizes that end inside a block
        dict(name="quantize-weight-fp32", kind="quantize", rows=8200, cols=4100, dtype="float32", block_rows=128),
        # one user's decode step: the output projection of an attention layer at 8B sizes
        dict(name="linear-x1", kind="linear", m=1, n=4096, k=4096, scales="e8m0", out="bfloat16"),
        # a small batch's gate and up projection at 8B sizes, weights with float32 scales from a checkpoint
        dict(name="linear-x8-gate-up", kind="linear", m=8, n=28672, k=4096, scales="float32", out="bfloat16"),
        # a loaded server's logits: an odd batch, float32 out, vocabulary of the 2,048 wide designs
        dict(name="linear-x61-head", kind="linear", m=61, n=32000, k=2048, scales="e8m0", out="float32"),
        # a ragged prompt portion through the down projection, float32 scales
        dict(name="linear-x1537-down", kind="linear", m=1537, n=4096, k=14336, scales="float32", out="bfloat16"),
        # a 2,048-token prompt through gate and up at 8B sizes
        dict(name="linear-x2048-gate-up", kind="linear", m=2048, n=28672, k=4096, scales="e8m0", out="bfloat16"),
        # one request on gated experts chosen by the softmax over the best logits
        dict(name="moe-x1", kind="moe", n=1, d=2048, ff=1408, experts=64, identity=0, top=6, rule="softmax_top", groups=1,
             keep=1, gated=True, weights="bfloat16", shared=False),
        # a small batch: identity experts, a gated shared expert's result, 8-bit experts
        dict(name="moe-x8-8bit", kind="moe", n=8, d=2048, ff=1408, experts=64, identity=16, top=6, rule="softmax", groups=1,
             keep=1, gated=True, weights="e8m0", shared=True),
        # ragged sizes: few experts, inner sizes that end inside a block, float32 scales
        dict(name="moe-x23-ragged", kind="moe", n=23, d=1040, ff=720, experts=20, identity=0, top=3, rule="sigmoid", groups=4,
             keep=2, gated=True, weights="float32", shared=False),
        # the largest step: nearly every expert is read; GELU experts chosen by groups
        dict(name="moe-x61-gelu", kind="moe", n=61, d=2048, ff=1408, experts=64, identity=0, top=6, rule="sigmoid", groups=8,
             keep=4, gated=False, weights="bfloat16", shared=False),
    ]


def _spread(rng, lo, hi, step=1):
    """A multiple of ``step`` between lo and hi, spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step))


def draw(rng):
    kind = rng.choice(["quantize", "linear", "linear", "moe", "moe"])
    if kind == "quantize":
        cols = _spread(rng, 64, 14336)
        rows = _spread(rng, 1, max(1, min(8192, 2048 * 14336 // cols)))
        return dict(kind=kind, rows=rows, cols=cols, dtype=rng.choice(["bfloat16", "float32"]), block_rows=rng.choice([1, 1, 128]))
    if kind == "linear":
        n, k = _spread(rng, 128, 28672), _spread(rng, 128, 14336, rng.choice([1, 16, 128]))
        m = _spread(rng, 1, min(4096, max(1, LARGEST // (2 * n * k))))
        return dict(kind=kind, m=m, n=n, k=k, scales=rng.choice(["e8m0", "float32"]), out=rng.choice(["bfloat16", "bfloat16", "float32"]))
    groups = rng.choice([1, 1, 2, 4])
    experts = groups * rng.randint(max(2, 4 // groups), 64 // groups)
    top = rng.randint(1, min(8, max(1, experts // 2)))
    rule = rng.choice(["sigmoid", "softmax", "softmax_top"])
    if rule == "softmax_top":
        groups = 1
    per = experts // groups
    keep = rng.randint(min(groups, -(-top // per)), groups)
    return dict(kind=kind, n=_spread(rng, 1, 61), d=_spread(rng, 256, 2048, 16), ff=_spread(rng, 128, 1408, 16), experts=experts,
                identity=rng.choice([0, 0, 5]) if groups == 1 and rule == "softmax" else 0, top=top, rule=rule, groups=groups, keep=keep,
                gated=rng.choice([True, True, False]), weights=rng.choice(["bfloat16", "e8m0", "float32"]),
                shared=rng.choice([False, True]))


# ---------------------------------------------------------------------------- inputs

def _blocks(n):
    return -(-n // BLOCK)


def _padded(x, rows, cols):
    return torch.nn.functional.pad(x, (0, cols - x.shape[-1], 0, rows - x.shape[-2]))


def _amax(x, block_rows):
    """[..., R, C] largest magnitudes of blocks of block_rows x 128."""
    r, c = -(-x.shape[-2] // block_rows), _blocks(x.shape[-1])
    p = _padded(x.abs(), r * block_rows, c * BLOCK)
    return p.reshape(*x.shape[:-2], r, block_rows, c, BLOCK).amax(dim=(-3, -1))


def _spread_out(s, block_rows, rows, cols):
    """The scale of every number from the blocks' scales."""
    return s.repeat_interleave(block_rows, dim=-2)[..., :rows, :].repeat_interleave(BLOCK, dim=-1)[..., :cols]


def _power_of_two(amax):
    """The exponent j of the smallest power of two, at least 2^-127, with amax <= 448 * 2^j; 0 where amax is 0."""
    m, e = torch.frexp(amax)
    j = torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-127)
    return torch.where(amax == 0, torch.zeros_like(j), j)


def _to_8bit(x, block_rows, scales):
    """(e4m3 numbers with rows that start on 16 bytes, scales) of float32 x."""
    rows, cols = x.shape[-2:]
    amax = _amax(x, block_rows)
    if scales == "e8m0":
        j = _power_of_two(amax)
        # exact: both factors are powers of two within float32's range
        s, inverse = torch.ldexp(torch.ones_like(amax), j), torch.ldexp(torch.ones_like(amax), -j)
        v = x * _spread_out(inverse, block_rows, rows, cols)
        s = s.to(torch.float8_e8m0fnu)
    else:
        s = torch.where(amax == 0, torch.ones_like(amax), amax / 448)
        v = (x / _spread_out(s, block_rows, rows, cols)).clamp(-448, 448)
    q = torch.empty((*x.shape[:-1], -(-cols // 16) * 16), dtype=torch.float8_e4m3fn, device=x.device)[..., :cols]
    q.copy_(v.to(torch.float8_e4m3fn))
    return q, s.contiguous()


def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed) * 2654435761 % (1 << 62) + 17)
    return g


def _activations(g, rows, cols):
    """Normed rows: unit scale, some channels much larger than the others."""
    x = torch.randn((rows, cols), device=DEVICE, generator=g)
    return x * torch.exp(0.8 * torch.randn((cols,), device=DEVICE, generator=g))


def prepare(case, seed):
    g = _generator(seed)
    if case["kind"] == "quantize":
        x = _activations(g, case["rows"], case["cols"]).to(getattr(torch, case["dtype"]))
        return dict(case=case, x=x)
    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        x, xs = _to_8bit(_activations(g, m, k), 1, case["scales"])
        w, ws = _to_8bit(torch.randn((n, k), device=DEVICE, generator=g) * k ** -0.5, BLOCK, case["scales"])
        return dict(case=case, x=x, xs=xs, w=w, ws=ws)
    n, d, ff, E = case["n"], case["d"], case["ff"], case["experts"]
    rows = E + case["identity"] + (1 if case["shared"] else 0)
    bf = torch.bfloat16
    s = dict(case=case, h=torch.randn((n, d), device=DEVICE, generator=g).to(bf))
    s["router"] = (torch.randn((rows, d), device=DEVICE, generator=g) * d ** -0.5).to(bf)
    s["correction"] = 0.05 * torch.randn((E + case["identity"],), device=DEVICE, generator=g)
    s["add"] = torch.randn((n, d), device=DEVICE, generator=g).to(bf) if case["shared"] else None
    up = torch.randn((E, (2 if case["gated"] else 1) * ff, d), device=DEVICE, generator=g) * d ** -0.5
    down = torch.randn((E, d, ff), device=DEVICE, generator=g) * ff ** -0.5
    if case["weights"] == "bfloat16":
        s.update(up=up.to(bf), down=down.to(bf), up_scale=None, down_scale=None)
    else:
        s["up"], s["up_scale"] = _to_8bit(up, BLOCK, case["weights"])
        s["down"], s["down_scale"] = _to_8bit(down, BLOCK, case["weights"])
    return s


# ---------------------------------------------------------------------------- the plain forms, in 32 bits

def _values(q, s, block_rows, dtype=torch.float32):
    """The numbers that 8-bit numbers and their scales stand for."""
    return q.to(dtype) if s is None else q.to(dtype) * _spread_out(s.to(dtype), block_rows, *q.shape[-2:])


def _chosen(case, z, correction):
    """(expert numbers, weights) of every token from its logits; ties go to the lower number."""
    E, G, top = z.shape[1], case["groups"], case["top"]
    if case["rule"] == "softmax_top":
        choice = z + correction
    else:
        s = torch.sigmoid(z) if case["rule"] == "sigmoid" else torch.softmax(z, dim=1)
        choice = s + correction
    masked = choice
    if G > 1:
        by = choice.reshape(-1, G, E // G).sort(dim=2, descending=True).values
        score = by[:, :, 0] if case["rule"] == "softmax" or E == G else by[:, :, 0] + by[:, :, 1]
        kept = torch.zeros_like(score).scatter(1, score.sort(dim=1, descending=True, stable=True).indices[:, :case["keep"]], 1.0)
        masked = torch.where(kept.repeat_interleave(E // G, dim=1) > 0, choice, torch.full_like(choice, -math.inf))
    ids = masked.sort(dim=1, descending=True, stable=True).indices[:, :top]
    if case["rule"] == "softmax_top":
        return ids, torch.softmax(choice.gather(1, ids), dim=1)
    w = s.gather(1, ids)
    return ids, (w / (w.sum(dim=1, keepdim=True) + 1e-20) if case["rule"] == "softmax" else w * 2.5)


def _layer(state, dtype):
    """The routed feed-forward in ``dtype``, not rounded: every expert on every token where most are chosen, else the chosen ones."""
    case, h = state["case"], state["h"].to(dtype)
    E, ff, (n, d) = case["experts"], case["ff"], h.shape
    z = h @ state["router"].to(dtype).t()
    ids, wts = _chosen(case, z[:, :E + case["identity"]], state["correction"].to(dtype))

    def act(u):
        if case["gated"]:
            return u[..., :ff] * torch.sigmoid(u[..., :ff]) * u[..., ff:]
        return 0.5 * u * (1 + torch.erf(u * 0.5 ** 0.5))

    if n * case["top"] < E:
        at = ids.reshape(-1).clamp(max=E - 1)
        pick = [None if t is None else t.view(torch.uint8)[at].view(t.dtype) if t.element_size() == 1 else t[at]
                for t in (state["up"], state["up_scale"], state["down"], state["down_scale"])]
        u = act((_values(pick[0], pick[1], BLOCK, dtype) @ h.repeat_interleave(case["top"], dim=0)[:, :, None])[:, :, 0])
        y = (_values(pick[2], pick[3], BLOCK, dtype) @ u[:, :, None])[:, :, 0].reshape(n, case["top"], d)
        out = (y * (wts * (ids < E))[:, :, None]).sum(dim=1)
    else:
        u = act(h @ _values(state["up"], state["up_scale"], BLOCK, dtype).transpose(1, 2))
        y = u @ _values(state["down"], state["down_scale"], BLOCK, dtype).transpose(1, 2)
        share = torch.zeros((n, E + case["identity"]), dtype=dtype, device=h.device).scatter_add(1, ids, wts)
        out = (y * share[:, :E].t()[:, :, None]).sum(dim=0)
    out = out + (wts * (ids >= E)).sum(dim=1, keepdim=True) * h
    if state["add"] is not None:
        out = out + torch.sigmoid(z[:, -1:]) * state["add"].to(dtype)
    return out


def run(state):
    case = state["case"]
    if own:
        return _run_own(state)
    if case["kind"] == "quantize":
        return list(_to_8bit(state["x"].float(), case["block_rows"], "e8m0"))
    if case["kind"] == "linear":
        x, w = _values(state["x"], state["xs"], 1), _values(state["w"], state["ws"], BLOCK)
        return (x @ w.t()).to(getattr(torch, case["out"]))
    return _layer(state, torch.float32).to(torch.bfloat16)


def _run_own(state):
    from batchspec_b200.kernels import ops
    case = state["case"]
    if case["kind"] == "quantize":
        return list(ops.quantize_fp8(state["x"], block_rows=case["block_rows"]))
    if case["kind"] == "linear":
        return ops.linear_fp8(state["x"], state["xs"], state["w"], state["ws"], out_dtype=getattr(torch, case["out"]),
                              w_is_parameter=True)
    rule = case["rule"]
    return ops.moe_layer(state["h"], state["router"], state["correction"], case["groups"], case["keep"], case["top"],
                         2.5 if rule == "sigmoid" else 1.0, state["up"], state["down"], up_scale=state["up_scale"],
                         down_scale=state["down_scale"], glu=case["gated"], softmax_top=rule == "softmax_top",
                         softmax=rule == "softmax", group_max=rule == "softmax", renormalise=rule == "softmax",
                         add=state["add"], add_gated=case["shared"], identity=case["identity"])


# ---------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "quantize":
        x = state["x"].double()
        rows, cols = x.shape
        b, c = case["block_rows"], _blocks(cols)
        r = -(-rows // b)
        whole = torch.zeros((r * b, c * BLOCK), dtype=torch.float64, device=x.device)
        whole[:rows, :cols] = x
        tiles = whole.view(r, b, c, BLOCK).permute(0, 2, 1, 3)
        top = tiles.abs().flatten(2).max(dim=2).values
        s = torch.exp2(torch.floor(torch.log2(top.clamp(min=1e-300) / 448)).clamp(min=-127))
        s = torch.where(s * 448 < top, 2 * s, s)                  # the logarithm may have landed one lower
        s = torch.where((s > 2.0 ** -127) & (s * 224 >= top), s / 2, s)
        s = torch.where(top == 0, torch.ones_like(s), s)
        v = tiles / s[:, :, None, None]
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
        q = (torch.round(v / step) * step).permute(0, 2, 1, 3).reshape(r * b, c * BLOCK)[:rows, :cols]
        return [q, s]
    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        row, col = torch.arange(n, device=DEVICE) // BLOCK, torch.arange(k, device=DEVICE) // BLOCK
        x = state["x"].double() * state["xs"].double()[:, col]
        w = state["w"].double() * state["ws"].double()[row][:, col]
        return torch.einsum("mk,nk->mn", x, w)
    return _exact_layer(case, state)


def _exact_layer(case, s):
    """Token by token and expert by expert."""
    h, z = s["h"].double(), torch.einsum("nd,ed->ne", s["h"].double(), s["router"].double())
    E, ff, d, many = case["experts"], case["ff"], case["d"], case["experts"] + case["identity"]
    score, corr = z[:, :many].clone(), s["correction"].double()
    if case["rule"] == "sigmoid":
        score = 1 / (1 + torch.exp(-score))
    elif case["rule"] == "softmax":
        score = torch.exp(score - torch.logsumexp(score, dim=1, keepdim=True))
    choice, score, out = (score + corr).tolist(), score.tolist(), []
    taken = []
    for t in range(case["n"]):
        c, per = choice[t], many // case["groups"]
        best = [sorted(c[g * per:(g + 1) * per], reverse=True) for g in range(case["groups"])]
        worth = [b[0] if case["rule"] == "softmax" or per == 1 else b[0] + b[1] for b in best]
        kept = set(sorted(range(case["groups"]), key=lambda g: (-worth[g], g))[:case["keep"]])
        ids = sorted((e for e in range(many) if e // per in kept), key=lambda e: (-c[e], e))[:case["top"]]
        if case["rule"] == "softmax_top":
            w = [math.exp(c[e] - c[ids[0]]) for e in ids]
            w = [v / sum(w) for v in w]
        elif case["rule"] == "softmax":
            w = [score[t][e] for e in ids]
            w = [v / sum(w) for v in w]
        else:
            w = [2.5 * score[t][e] for e in ids]
        taken.append(dict(zip(ids, w)))
    out = torch.zeros((case["n"], d), dtype=torch.float64, device=DEVICE)
    for e in sorted({e for t in taken for e in t}):
        rows = [t for t in range(case["n"]) if e in taken[t]]
        weight = torch.tensor([taken[t][e] for t in rows], dtype=torch.float64, device=DEVICE)[:, None]
        x = h[rows]
        if e < E:
            up, down = s["up"][e].double(), s["down"][e].double()
            if s["up_scale"] is not None:
                col = torch.arange(d, device=DEVICE) // BLOCK
                inner = torch.arange(ff, device=DEVICE) // BLOCK
                up = up * s["up_scale"][e].double()[torch.arange(up.shape[0], device=DEVICE) // BLOCK][:, col]
                down = down * s["down_scale"][e].double()[col][:, inner]
            u = torch.einsum("td,fd->tf", x, up)
            if case["gated"]:
                u = u[:, :ff] / (1 + torch.exp(-u[:, :ff])) * u[:, ff:]
            else:
                u = u / 2 * torch.special.erfc(-u / math.sqrt(2))
            x = torch.einsum("tf,df->td", u, down)
        out[rows] += weight * x
    if s["add"] is not None:
        out += s["add"].double() / (1 + torch.exp(-z[:, many:]))
    return out


# ---------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case["kind"] == "quantize":
        n = case["rows"] * case["cols"]
        scales = -(-case["rows"] // case["block_rows"]) * _blocks(case["cols"])
        return {"bytes": n * (5 if case["dtype"] == "float32" else 3) + scales, "flops": 2 * n}
    one = 4 if case["kind"] == "linear" and case["scales"] == "float32" or case.get("weights") == "float32" else 1
    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        scales = (m + _blocks(n)) * _blocks(k) * one
        return {"bytes": m * k + n * k + scales + m * n * (4 if case["out"] == "float32" else 2), "flops": 2 * m * n * k}
    n, d, ff, E, top = case["n"], case["d"], case["ff"], case["experts"], case["top"]
    many = E + case["identity"]
    read = E * (1 - (1 - top / many) ** n)                      # experts that some token chooses, when all are as likely
    inner = (3 if case["gated"] else 2) * ff
    each = inner * d * (2 if case["weights"] == "bfloat16" else 1)
    if case["weights"] != "bfloat16":
        each += ((_blocks(inner - ff)) * _blocks(d) + _blocks(d) * _blocks(ff)) * one
    rows = many + (1 if case["shared"] else 0)
    return {"bytes": read * each + rows * d * 2 + 2 * n * d * (3 if case["shared"] else 2),
            "flops": 2 * n * (top * E / many * inner * d + rows * d)}
