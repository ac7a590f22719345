"""Matrix products on 8-bit floating point (FP8: e4m3 values, one fp32 scale for each block of 128) and the routing of tokens to
experts that hold such matrices, as a program that serves a language model makes them, over the range of sizes it meets.

  round    ops.quantize_fp8 and ops.dequantize: activations (a scale per row and 128 k) or weights (per 128 rows and 128 k) to 8 bits and back
  linear   ops.qlinear on a QWeightFP8: y = x @ dequant(W).T, from one decoded token to a long prompt; x is bf16 or, "fp8", activations that
           ops.quantize_fp8 has just made 8-bit ones
  grouped  ops.qgemm_grouped on QExpertsFP8: rows sorted by expert, each group times its own expert's matrix, x as in linear
  route    ops.moe_route: softmax or sigmoid scores, a bias that balances the experts' load, groups of experts, top-k, renormalised weights
  moe      ops.moe_ffn on QExpertsFP8: routing as in route, gate and up, SiLU, down, the weighted sum; x as in linear, and where it is
           8-bit the hidden activations become it too

Values: sign, 4 bits of exponent, 3 of mantissa, largest 448.  Quantisation: r = 448 / amax and scale = amax / 448 of a block's largest
magnitude (2^-126 * 448 at least), each one fp32 division; a value goes to the nearest of x * r, one fp32 product, ties to the even one.
Routing: an expert is chosen by its score plus bias in 64 bits (by its logit where there is neither bias nor a sum over a group), ties go
to the lowest index; one whose logit is -infinity or NaN comes behind all others and has the score 0.  A group of consecutive experts
counts as much as the sum of its `group_sum` largest choices; the experts of the `top_groups` largest groups may be chosen.
"""
import math

import torch

own = False

DEV = "cuda:0"
BLOCK = 128
LARGEST = 448.0
LEAST = 448.0 * 2.0 ** -126
LAST = -1e300  # the choice value of a masked expert

SOFTMAX = dict(score="softmax", bias=False, groups=1, top_groups=1, group_sum=1, scale=1.0)
GROUPED = dict(score="sigmoid", bias=True, groups=8, top_groups=4, group_sum=2, scale=2.5)


def _round(what, rows, k, dtype, **more):
    return dict(more, op="round", what=what, rows=rows, k=k, dtype=dtype)


def _linear(m, n, k, x="bf16", out="native", **more):
    return dict(more, op="linear", m=m, n=n, k=k, x=x, out=out)


def _grouped(rows, experts, n, k, x="fp8", **more):
    return dict(more, op="grouped", rows=rows, experts=experts, n=n, k=k, x=x)


def _route(tokens, experts, top_k, renorm=True, how=SOFTMAX, **more):
    return dict(more, op="route", tokens=tokens, experts=experts, top_k=top_k, renorm=renorm, **how)


def _moe(tokens, h, f, experts, top_k, x="bf16", how=SOFTMAX, **more):
    return dict(more, op="moe", tokens=tokens, h=h, f=f, experts=experts, top_k=top_k, renorm=True, x=x, **how)


def listed():
    return [
        # the activations of 16 sequences decoded together: launches and host time decide
        _round("rows", 16, 4096, "bf16", name="round rows bf16 16x4096"),
        # a feed-forward matrix of a 7B-sized model, quantised as it is loaded
        _round("weights", 14336, 4096, "fp32", name="round weights fp32 14336x4096"),
        # the feed-forward projection of a 7B-sized model, one decoded token
        _linear(1, 14336, 4096, name="linear 1x14336x4096"),
        # six sequences decoded together, 8-bit activations, results wanted in bf16, a width that fits no tile
        _linear(6, 11008, 4096, x="fp8", out="bf16", name="linear fp8 6x11008x4096 bf16"),
        # a prompt of a thousand tokens, down projection; no multiple of a tile
        _linear(1000, 4096, 14336, name="linear 1000x4096x14336"),
        # several prompts packed together: the largest product
        _linear(4096, 14336, 4096, x="fp8", name="linear fp8 4096x14336x4096"),
        # 16 decoding tokens, two experts each, through one matrix of every expert: some experts get none
        _grouped(32, 8, 14336, 4096, x="bf16", name="grouped 32 rows, 8 of 14336x4096"),
        # a prompt's rows through smaller experts
        _grouped(2048, 16, 4096, 2048, name="grouped fp8 2048 rows, 16 of 4096x2048"),
        # the router of a layer of many small experts, 16 sequences decoded together
        _route(16, 256, 8, how=GROUPED, name="route 16 tokens to 8 of 256"),
        # the same for several prompts packed together
        _route(8192, 256, 8, how=GROUPED, name="route 8192 tokens to 8 of 256"),
        # four decoding tokens through a mixture of experts
        _moe(4, 4096, 14336, 8, 2, name="moe 4 tokens"),
        # a prompt of a thousand tokens through a layer of many small experts, everything in 8 bits
        _moe(1000, 2048, 1408, 64, 6, x="fp8", how=GROUPED, name="moe fp8 1000 tokens, 64 experts"),
    ]


def _log(rng, lo, hi):
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi))))


def _size(rng, lo, hi, step, odd):
    """lo .. hi, spread over the logarithm: multiples of `step`, one in three of them only of `odd`."""
    step = odd if rng.random() < 1 / 3 else step
    return max(lo, _log(rng, lo, hi) // step * step)


def _how(rng, experts, top_k):
    """A way of routing to `experts`, as models do it."""
    groups = rng.choice([g for g in (1, 1, 2, 4, 8) if experts % g == 0 and experts // g >= 2])
    per = experts // groups
    least = -(-top_k // per)
    return dict(score=rng.choice(("softmax", "sigmoid")), bias=rng.random() < 0.5, groups=groups, top_groups=rng.randint(least, groups),
                group_sum=rng.choice((1, 2)) if groups > 1 else 1, scale=rng.choice((1.0, 2.5)))


def draw(rng):
    op = rng.choices(("round", "linear", "grouped", "route", "moe"), (2, 7, 3, 3, 3))[0]
    x = rng.choice(("bf16", "fp8"))
    if op == "round":
        return _round(rng.choice(("rows", "weights")), _log(rng, 1, 14336), _size(rng, 128, 4096, 128, 16), rng.choice(("bf16", "fp16", "fp32")))
    if op == "linear":
        m = rng.choice((1, rng.randint(2, 16), _log(rng, 17, 256), _log(rng, 256, 4096)))
        n, k = _size(rng, 256, 14336, 128, 1), _size(rng, 256, 14336, 128, 16)
        while m * n * k > 4096 * 14336 * 4096:
            n, k = _size(rng, 256, 14336, 128, 1), _size(rng, 256, 14336, 128, 16)
        return _linear(m, n, k, x, rng.choice(("native", "bf16")) if m <= 16 else "native")
    if op == "grouped":
        experts, rows = _log(rng, 2, 64), _log(rng, 1, 4096)
        n, k = _size(rng, 256, 14336, 128, 1), _size(rng, 256, 14336, 128, 16)
        while experts * n * k > 8 * 14336 * 4096 or rows * n * k > 4096 * 14336 * 4096:
            n, k = _size(rng, 256, 14336, 128, 1), _size(rng, 256, 14336, 128, 16)
        return _grouped(rows, experts, n, k, x)
    if op == "route":
        experts = rng.choice((8, 16, 32, 60, 64, 128, 160, 256, 384))
        top_k = rng.choice((1, 2, 4, 6, 8))
        return _route(_log(rng, 1, 8192), experts, top_k, rng.random() < 0.7, _how(rng, experts, top_k))
    experts = rng.choice((4, 8, 16, 32, 64))
    h, f = _size(rng, 256, 4096, 128, 16), _size(rng, 256, 14336, 128, 16)
    while experts * h * f > 8 * 14336 * 4096:
        h, f = _size(rng, 256, 4096, 128, 16), _size(rng, 256, 14336, 128, 16)
    top_k = rng.choice([k for k in (1, 2, 2, 4, 6) if k <= experts])
    return _moe(_log(rng, 1, 1000), h, f, experts, top_k, x, rng.choice((SOFTMAX, _how(rng, experts, top_k))))


# ---- the plain form: 32-bit torch operations ----------------------------------------------------------------------------
def _padded(x, rows):
    """fp32 x with zeros up to whole blocks along K and, `rows`, along the rows too."""
    return torch.nn.functional.pad(x.to(torch.float32), (0, -x.shape[-1] % BLOCK, 0, -x.shape[-2] % BLOCK if rows else 0))


def _quantize_rows(x):
    """[M,K] -> values of 8 bits [M,K], scales fp32 [M,ceil(K/128)]."""
    blocks = _padded(x, False).unflatten(-1, (-1, BLOCK))
    amax = blocks.abs().amax(-1).clamp(min=LEAST)
    largest = torch.full_like(amax, LARGEST)
    q = (blocks * (largest / amax)[..., None]).flatten(-2)[..., :x.shape[-1]].to(torch.float8_e4m3fn)
    return q.contiguous(), amax / largest


def _quantize_weights(w):
    """[..,N,K] -> values of 8 bits [..,N,K], scales fp32 [..,ceil(N/128),ceil(K/128)]."""
    n, k = w.shape[-2:]
    blocks = _padded(w, True).unflatten(-1, (-1, BLOCK)).unflatten(-3, (-1, BLOCK))  # [..,N/128,128,K/128,128]
    amax = blocks.abs().amax((-1, -3)).clamp(min=LEAST)
    largest = torch.full_like(amax, LARGEST)
    q = (blocks * (largest / amax)[..., None, :, None]).flatten(-2).flatten(-3, -2)[..., :n, :k].to(torch.float8_e4m3fn)
    return q.contiguous(), amax / largest


def _row_values(q, scale):
    return q.to(torch.float32) * scale.repeat_interleave(BLOCK, -1)[..., :q.shape[-1]]


def _weight_values(q, scale):
    return _row_values(q, scale.repeat_interleave(BLOCK, -2)[..., :q.shape[-2], :])


def _rows(state, case):
    """The activations of a product in 32 bits."""
    return _row_values(*_quantize_rows(state["x"])) if case["x"] == "fp8" else state["x"].to(torch.float32)


def _by_group(x, offsets, most):
    """Rows [R,K] and group bounds -> (rows [E,most,K], the row that each place of it holds, whether it holds one)."""
    place = offsets[:-1, None].long() + torch.arange(most, device=x.device)
    held = place < offsets[1:, None]
    place = place.clamp(max=x.shape[0] - 1)
    return x[place], place, held


def _grouped_product(x, w, offsets, most):
    """fp32 rows [R,K], weights [E,N,K] -> [R,N]: each row times its group's matrix."""
    rows, place, held = _by_group(x, offsets, most)
    y = torch.bmm(rows, w.transpose(1, 2).contiguous())
    out = torch.zeros(x.shape[0], w.shape[1], device=x.device)
    out[place[held]] = y[held]
    return out


def _plain_route(logits, bias, case):
    """-> experts int32 [T,top_k], weights fp32 [T,top_k]"""
    t, e, top_k = *logits.shape, case["top_k"]
    masked = torch.isnan(logits) | (logits == -math.inf)
    z = logits.to(torch.float64).masked_fill(masked, -math.inf)
    score = torch.softmax(z, -1) if case["score"] == "softmax" else 1 / (1 + torch.exp(-z))
    score = score.masked_fill(masked, 0.0)
    by = z if bias is None and case["group_sum"] == 1 else score + (0 if bias is None else bias.to(torch.float64))
    by = by.masked_fill(masked, LAST)
    if case["groups"] > 1:
        per = e // case["groups"]
        value = by.view(t, case["groups"], per).sort(dim=-1, descending=True).values[..., :case["group_sum"]].sum(-1)
        group = value.sort(dim=-1, descending=True, stable=True).indices[:, :case["top_groups"]]
        open_ = (group[:, :, None] == torch.arange(e, device=logits.device) // per).any(1)
        by = by.masked_fill(~open_, -math.inf)
    chosen = by.sort(dim=-1, descending=True, stable=True).indices[:, :top_k]
    w = torch.gather(score, 1, chosen)
    if case["renorm"]:
        total = w.sum(-1, keepdim=True)
        w = w / torch.where(total > 0, total, torch.ones_like(total))
    return chosen.to(torch.int32), (w * case["scale"]).to(torch.float32)


def _plain_moe(state, case):
    top_k = case["top_k"]
    choice, p = _plain_route(state["logits"], state.get("bias"), case)
    order = choice.flatten().sort(stable=True).indices  # (token, slot) pairs by expert
    counts = (choice.flatten()[:, None] == torch.arange(case["experts"], device=DEV)).sum(0)
    offsets = torch.cat((counts.new_zeros(1), counts.cumsum(0)))
    x = _rows(state, case)[order // top_k]
    gate = _grouped_product(x, _weight_values(*state["gate"]), offsets, case["tokens"])
    up = _grouped_product(x, _weight_values(*state["up"]), offsets, case["tokens"])
    hidden = gate / (1 + torch.exp(-gate)) * up
    if case["x"] == "fp8":
        hidden = _row_values(*_quantize_rows(hidden))
    down = _grouped_product(hidden, _weight_values(*state["down"]), offsets, case["tokens"])
    y = torch.empty_like(down)
    y[order] = down
    return (y.view(case["tokens"], top_k, -1) * p[..., None]).sum(1).to(torch.bfloat16)


def _plain(state):
    case = state["case"]
    if case["op"] == "round":
        return _row_values(*_quantize_rows(state["x"])) if case["what"] == "rows" else _weight_values(*_quantize_weights(state["x"]))
    if case["op"] == "linear":
        y = _rows(state, case) @ _weight_values(state["w8"], state["scale"]).T
        return y if _result(case) == torch.float32 else y.to(torch.bfloat16)
    if case["op"] == "grouped":
        return _grouped_product(_rows(state, case), _weight_values(state["w8"], state["scale"]), state["offsets"], state["most"]).to(torch.bfloat16)
    if case["op"] == "route":
        return _plain_route(state["logits"], state.get("bias"), case)
    return _plain_moe(state, case)


# ---- the framework's operators ------------------------------------------------------------------------------------------
def _routing(state, case):
    return dict(top_k=case["top_k"], renorm=case["renorm"], score=case["score"], bias=state.get("bias"), groups=case["groups"],
                top_groups=case["top_groups"], group_sum=case["group_sum"], scale=case["scale"])


def _own(state):
    from chadslab_amd import QExpertsFP8, QWeightFP8, ops

    case = state["case"]
    if case["op"] == "round":
        return ops.dequantize(ops.quantize_fp8(state["x"], rows=case["what"] == "rows"))
    if case["op"] == "route":
        return ops.moe_route(state["logits"], **_routing(state, case))
    if "w" not in state:  # the containers of the loaded weights
        if case["op"] == "moe":
            state["w"] = tuple(QExpertsFP8(*state[m]) for m in ("gate", "up", "down"))
        else:
            state["w"] = (QExpertsFP8 if case["op"] == "grouped" else QWeightFP8)(state["w8"], state["scale"])
    x = ops.quantize_fp8(state["x"]) if case["x"] == "fp8" else state["x"]
    if case["op"] == "linear":
        return ops.qlinear(x, state["w"], out_dtype=torch.bfloat16 if case["out"] == "bf16" else None)
    if case["op"] == "grouped":
        return ops.qgemm_grouped(x, state["w"], state["offsets"])
    return ops.moe_ffn(x, state["logits"], state["w"], **_routing(state, case))


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# ---- inputs -------------------------------------------------------------------------------------------------------------
def _result(case):
    """The type of a product's result: fp32 for up to 16 rows unless bf16 is asked for."""
    return torch.float32 if case["m"] <= 16 and case["out"] == "native" else torch.bfloat16


def _weights(g, *shape):
    """Normal weights, every row with a spread of its own, as values of 8 bits and scales."""
    spread = torch.exp(torch.randn(*shape[:-1], 1, device=DEV, generator=g) * 0.5 - 4.0)
    return _quantize_weights(torch.randn(*shape, device=DEV, generator=g) * spread)


def _activations(g, rows, k):
    """Normal activations, some channels of which are many times larger than the others, as in a decoder's hidden state."""
    gain = torch.exp(torch.randn(k, device=DEV, generator=g) * 0.7)
    return torch.randn(rows, k, device=DEV, generator=g) * gain


def _router(g, state, case):
    """Logits, some experts liked more than others, and the bias that makes up for it."""
    liked = torch.randn(case["experts"], device=DEV, generator=g) * 0.5
    state["logits"] = torch.randn(case["tokens"], case["experts"], device=DEV, generator=g) + liked
    if case["bias"]:
        state["bias"] = (0.1 if case["score"] == "sigmoid" else 0.2 / case["experts"]) * -liked


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    state = {"case": case}
    if case["op"] == "round":
        dtype = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[case["dtype"]]
        state["x"] = _activations(g, case["rows"], case["k"]).to(dtype)
    elif case["op"] == "linear":
        state["x"] = _activations(g, case["m"], case["k"]).to(torch.bfloat16)
        state["w8"], state["scale"] = _weights(g, case["n"], case["k"])
    elif case["op"] == "grouped":
        rows, experts = case["rows"], case["experts"]
        share = torch.softmax(torch.randn(experts, device=DEV, generator=g), 0)  # some experts are liked more than others
        choice = torch.multinomial(share, rows, replacement=True, generator=g)
        counts = torch.bincount(choice, minlength=experts)
        state["offsets"] = torch.cat((counts.new_zeros(1), counts.cumsum(0))).to(torch.int32)
        state["most"] = int(counts.max())
        state["x"] = _activations(g, rows, case["k"]).to(torch.bfloat16)
        state["w8"], state["scale"] = _weights(g, experts, case["n"], case["k"])
    elif case["op"] == "route":
        _router(g, state, case)
    else:
        e, h, f = case["experts"], case["h"], case["f"]
        state["x"] = _activations(g, case["tokens"], h).to(torch.bfloat16)
        _router(g, state, case)
        state["gate"], state["up"], state["down"] = _weights(g, e, f, h), _weights(g, e, f, h), _weights(g, e, h, f)
    return state


# ---- what a pass cannot do without --------------------------------------------------------------------------------------
def _ceil(n):
    return -(-n // BLOCK)


def _held(n, k):
    """Bytes of an N x K matrix with its scales."""
    return n * k + 4 * _ceil(n) * _ceil(k)


def work(case):
    if case["op"] == "round":
        r, k = case["rows"], case["k"]
        held = r * k + 4 * r * _ceil(k) if case["what"] == "rows" else _held(r, k)
        return {"bytes": r * k * (4 if case["dtype"] == "fp32" else 2) + held + 4 * r * k, "flops": 3 * r * k}
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": _held(n, k) + 2 * m * k + m * n * (4 if _result(case) == torch.float32 else 2), "flops": 2 * m * n * k}
    if case["op"] == "grouped":
        r, e, n, k = case["rows"], case["experts"], case["n"], case["k"]
        hit = e * (1 - (1 - 1 / e) ** r)  # experts that have a row, on average
        return {"bytes": hit * _held(n, k) + 2 * r * k + 2 * r * n + 4 * (e + 1), "flops": 2 * r * n * k}
    t, e, top_k = case["tokens"], case["experts"], case["top_k"]
    if case["op"] == "route":
        return {"bytes": 4 * t * e + 8 * t * top_k + (4 * e if case["bias"] else 0), "flops": t * e * (4 + top_k)}
    h, f = case["h"], case["f"]
    hit = e * (1 - (1 - top_k / e) ** t)
    return {"bytes": hit * (2 * _held(f, h) + _held(h, f)) + 4 * t * h + 4 * t * e, "flops": 6 * t * top_k * h * f}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------
def _exact_values(bits, scale, by_row):
    """(-1)^s 2^(e - 7) (1 + m/8), or (-1)^s 2^-6 m/8 where e is 0, times the block's scale."""
    b = bits.view(torch.uint8).to(torch.int64)
    e, m = b // 8 % 16, (b % 8).double() / 8
    v = (1.0 - 2.0 * (b // 128).double()) * torch.where(e == 0, 2.0 ** -6 * m, torch.exp2((e - 7).double()) * (1 + m))
    k = torch.arange(v.shape[1], device=DEV) // BLOCK
    r = torch.arange(v.shape[0], device=DEV)
    return v * scale.double()[r if by_row else r // BLOCK][:, k]


def _exact_rounded(x, high):
    """The values in 64 bits that x becomes: in a block of `high` rows and 128 columns the nearest multiple of the spacing at each value."""
    x = x.double()
    y = torch.empty_like(x)
    for c in range(0, x.shape[1], BLOCK):
        part = x[:, c:c + BLOCK]
        largest = part.abs().max(1, keepdim=True).values
        if high > 1:
            largest = torch.cat([largest[r:r + high].max().expand(min(high, x.shape[0] - r), 1) for r in range(0, x.shape[0], high)])
        scale = largest.clamp(min=LEAST) / 448
        v = (part * (LARGEST / largest.clamp(min=LEAST)).float()).float().double()  # (the definition's two roundings to fp32)
        spacing = torch.exp2((torch.frexp(v).exponent - 4).clamp(min=-9).double())  # 2^-9 below 2^-6, then an eighth of the power of two
        y[:, c:c + BLOCK] = (v / spacing).round() * spacing * scale
    return y


def _exact_route(logits, bias, case):
    """Experts by counting those that go before each; scores as 1 / sums of exponentials."""
    z = logits.double()
    t, e = z.shape
    per, top_k = e // case["groups"], case["top_k"]
    if case["score"] == "softmax":
        up = torch.exp(z - z.max(1, keepdim=True).values)
        score = up / up.sum(1, keepdim=True)
    else:
        score = torch.sigmoid(z)
    by = z if bias is None and case["group_sum"] == 1 else score if bias is None else score + bias.double()

    def first(v, count):  # whether so many at most go before each: larger ones, and equal ones in front of it
        place = torch.arange(v.shape[1], device=DEV)
        out = torch.empty(v.shape, dtype=torch.int64, device=DEV)
        for i in range(v.shape[1]):
            out[:, i] = ((v > v[:, i:i + 1]) | ((v == v[:, i:i + 1]) & (place < i))).sum(1)
        return out < count, out

    if case["groups"] > 1:
        inside = by.reshape(t * case["groups"], per)
        value = torch.where(first(inside, case["group_sum"])[0], inside, torch.zeros_like(inside)).sum(1).reshape(t, case["groups"])
        kept = first(value, case["top_groups"])[0].repeat_interleave(per, 1)
        by = torch.where(kept, by, torch.full_like(by, -math.inf))
    taken, rank = first(by, top_k)
    chosen = torch.zeros(t, top_k, dtype=torch.int64, device=DEV)
    at = taken.nonzero()
    chosen[at[:, 0], rank[taken]] = at[:, 1]
    w = torch.gather(score, 1, chosen)
    if case["renorm"]:
        w = w / w.sum(1, keepdim=True)
    return chosen.to(torch.int32), w * case["scale"]


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "round":
        return _exact_rounded(state["x"], 1 if case["what"] == "rows" else BLOCK)
    if case["op"] == "route":
        return _exact_route(state["logits"], state.get("bias"), case)
    x = _exact_rounded(state["x"], 1) if case["x"] == "fp8" else state["x"].double()
    if case["op"] == "linear":
        return torch.mm(x, _exact_values(state["w8"], state["scale"], False).t())
    if case["op"] == "grouped":
        y = torch.zeros(case["rows"], case["n"], dtype=torch.float64, device=DEV)
        bounds = state["offsets"].tolist()
        for e, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
            y[lo:hi] = x[lo:hi] @ _exact_values(state["w8"][e], state["scale"][e], False).t()
        return y
    y = torch.zeros(case["tokens"], case["h"], dtype=torch.float64, device=DEV)
    chosen, weight = _exact_route(state["logits"], state.get("bias"), case)
    for e in range(case["experts"]):
        gate, up, down = (_exact_values(state[m][0][e], state[m][1][e], False) for m in ("gate", "up", "down"))
        token, slot = (chosen == e).nonzero(as_tuple=True)
        g = x[token] @ gate.t()
        hidden = g * torch.sigmoid(g) * (x[token] @ up.t())
        if case["x"] == "fp8":
            hidden = _exact_rounded(hidden, 1)
        y.index_add_(0, token, weight[token, slot][:, None] * (hidden @ down.t()))
    return y
