"""Matrix products on microscaled 4-bit floating point (MXFP4: e2m1 values, one power-of-two scale per 32 of them along
K), as a program that serves a language model makes them, over the range of sizes it meets.

  round    ops.quantize_mxfp4 and ops.dequantize: a matrix to 4 bits and back
  linear   ops.qlinear on a QWeightMXFP4: y = x @ dequant(W).T for bf16 activations, from one decoded token to a long prompt
  linear4  ops.quantize_mxfp4 of the activations and ops.qlinear of the two 4-bit matrices
  grouped  ops.qgemm_grouped: rows sorted by expert, each group times its own expert's matrix, groups of any size; the rows are
           bf16 or, "mxfp4", 4-bit ones
  moe      ops.moe_ffn on MXFP4 experts: router, gate and up, SiLU, down, the weighted sum

Codes: sign in bit 3, then 0, 0.5, 1, 1.5, 2, 3, 4, 6; two to a byte, the even k in the low nibble.  Scale byte e: 2^(e - 127).
Quantisation: the scale of a block is 2^(floor(log2(largest magnitude)) - 2), its values go to the nearest code, ties to the
even one, what lies beyond 6 to 6.
"""
import math

import torch

own = False

DEV = "cuda:0"
BLOCK = 32


def _round(rows, k, dtype, **more):
    return dict(more, op="round", rows=rows, k=k, dtype=dtype)


def _linear(m, n, k, op="linear", out="native", **more):
    return dict(more, op=op, m=m, n=n, k=k, out=out)


def _grouped(rows, experts, n, k, x="bf16", **more):
    return dict(more, op="grouped", rows=rows, experts=experts, n=n, k=k, x=x)


def _moe(tokens, h, f, experts, top_k, **more):
    return dict(more, op="moe", tokens=tokens, h=h, f=f, experts=experts, top_k=top_k)


def listed():
    return [
        # the activations of 16 sequences decoded together: launches and host time decide
        _round(16, 4096, "bf16", name="round bf16 16x4096"),
        # a feed-forward matrix of a 7B-sized model, quantised as it is loaded
        _round(14336, 4096, "fp32", name="round fp32 14336x4096"),
        # the smallest projection of the 2B decoder (attention output), one token
        _linear(1, 2048, 2048, name="linear 1x2048x2048"),
        # the feed-forward projection of a 7B-sized model, one decoded token
        _linear(1, 14336, 4096, name="linear 1x14336x4096"),
        # six sequences decoded together, results wanted in the activations' own type, a width that fits no tile
        _linear(6, 11008, 4096, out="bf16", name="linear 6x11008x4096 bf16"),
        # a serving batch of 48 sequences, one token each: between decoding and prompts
        _linear(48, 14336, 4096, name="linear 48x14336x4096"),
        # a prompt of a thousand tokens, down projection; no multiple of a tile
        _linear(1000, 4096, 14336, name="linear 1000x4096x14336"),
        # several prompts packed together, activations in 4 bits too: the largest product
        _linear(4096, 14336, 4096, op="linear4", name="linear4 4096x14336x4096"),
        # 16 decoding tokens, two experts each, through one matrix of every expert: some experts get none
        _grouped(32, 8, 14336, 4096, name="grouped 32 rows, 8 of 14336x4096"),
        # a prompt's rows, 4-bit ones, through smaller experts
        _grouped(2048, 16, 4096, 2048, x="mxfp4", name="grouped mxfp4 2048 rows, 16 of 4096x2048"),
        # four decoding tokens through a mixture of experts
        _moe(4, 4096, 14336, 8, 2, name="moe 4 tokens"),
        # a prompt of 256 tokens through the same layer
        _moe(256, 4096, 14336, 8, 2, name="moe 256 tokens"),
    ]


def _log(rng, lo, hi):
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi))))


def _size(rng, lo, hi, step, odd):
    """lo .. hi, spread over the logarithm: multiples of `step`, one in three of them only of `odd`."""
    step = odd if rng.random() < 1 / 3 else step
    return max(lo, _log(rng, lo, hi) // step * step)


def draw(rng):
    op = rng.choices(("round", "linear", "linear4", "grouped", "moe"), (2, 6, 2, 3, 2))[0]
    if op == "round":
        return _round(_log(rng, 1, 14336), _size(rng, 32, 4096, 256, 32), rng.choice(("bf16", "fp16", "fp32")))
    if op in ("linear", "linear4"):
        m = rng.choice((1, rng.randint(2, 16), _log(rng, 17, 256), _log(rng, 256, 4096)))
        n, k = _size(rng, 256, 14336, 128, 1), _size(rng, 256, 14336, 256, 32)
        while m * n * k > 4096 * 14336 * 4096:
            n, k = _size(rng, 256, 14336, 128, 1), _size(rng, 256, 14336, 256, 32)
        return _linear(m, n, k, op, rng.choice(("native", "bf16")) if m <= 16 else "native")
    if op == "grouped":
        experts, rows = _log(rng, 2, 64), _log(rng, 1, 4096)
        n, k = _size(rng, 256, 14336, 128, 1), _size(rng, 256, 14336, 256, 32)
        while experts * n * k > 8 * 14336 * 4096 or rows * n * k > 4096 * 14336 * 4096:
            n, k = _size(rng, 256, 14336, 128, 1), _size(rng, 256, 14336, 256, 32)
        return _grouped(rows, experts, n, k, rng.choice(("bf16", "mxfp4")))
    experts = rng.choice((4, 8, 16))
    h, f = _size(rng, 256, 4096, 256, 32), _size(rng, 256, 14336, 256, 32)
    while experts * h * f > 8 * 14336 * 4096:
        h, f = _size(rng, 256, 4096, 256, 32), _size(rng, 256, 14336, 256, 32)
    return _moe(_log(rng, 1, 512), h, f, experts, rng.choice((1, 2, 2, 4)))


# ---- the plain form: 32-bit torch operations ----------------------------------------------------------------------------
def _quantize(x):
    """[.., K] -> packed codes uint8 [.., K/2], scale bytes uint8 [.., K/32]."""
    blocks = x.to(torch.float32).unflatten(-1, (-1, BLOCK))
    exponent = (blocks.abs().amax(-1, keepdim=True).view(torch.int32) >> 23) - 2  # of the scale, as its byte
    exponent = exponent.clamp(min=0)
    v = blocks * ((254 - exponent) << 23).view(torch.float32)  # times 2^(127 - byte): exact
    a = v.abs()
    # the codes' midpoints; where a midpoint itself goes is its even neighbour's
    code = (a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    code = (code + 8 * torch.signbit(v)).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), exponent.squeeze(-1).to(torch.uint8)


def _values(packed, scale):
    """The fp32 values that codes and scales stand for."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=packed.device)
    table = torch.cat((table, -table))
    code = torch.stack((packed & 15, packed >> 4), -1).flatten(-2)
    v = table[code.to(torch.int32)].unflatten(-1, (-1, BLOCK))
    return (v * torch.exp2(scale.to(torch.float32) - 127.0)[..., None]).flatten(-2)


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


def _plain(state):
    case = state["case"]
    if case["op"] == "round":
        return _values(*_quantize(state["x"]))
    if case["op"] in ("linear", "linear4"):
        x = _values(*_quantize(state["x"])) if case["op"] == "linear4" else state["x"].to(torch.float32)
        y = x @ _values(state["packed"], state["scale"]).T
        return y if _result(case) == torch.float32 else y.to(torch.bfloat16)
    if case["op"] == "grouped":
        x = _values(state["x_packed"], state["x_scale"]) if case["x"] == "mxfp4" else state["x"].to(torch.float32)
        return _grouped_product(x, _values(state["packed"], state["scale"]), state["offsets"], state["most"]).to(torch.bfloat16)
    t, top_k = case["tokens"], case["top_k"]
    p, choice = torch.softmax(state["logits"], -1).sort(dim=-1, descending=True, stable=True)
    p, choice = p[:, :top_k], choice[:, :top_k]
    p = p / p.sum(-1, keepdim=True)
    order = choice.flatten().sort(stable=True).indices  # (token, slot) pairs by expert
    counts = (choice.flatten()[:, None] == torch.arange(case["experts"], device=DEV)).sum(0)
    offsets = torch.cat((counts.new_zeros(1), counts.cumsum(0)))
    x = state["x"].to(torch.float32)[order // top_k]
    gate = _grouped_product(x, _values(*state["gate"]), offsets, t)
    up = _grouped_product(x, _values(*state["up"]), offsets, t)
    down = _grouped_product(gate / (1 + torch.exp(-gate)) * up, _values(*state["down"]), offsets, t)
    y = torch.empty_like(down)
    y[order] = down
    return (y.view(t, top_k, -1) * p[..., None]).sum(1).to(torch.bfloat16)


# ---- the framework's operators ------------------------------------------------------------------------------------------
def _own(state):
    from chadslab_amd import QExpertsMXFP4, QWeightMXFP4, ops

    case = state["case"]
    if case["op"] == "round":
        return ops.dequantize(ops.quantize_mxfp4(state["x"]))
    if "w" not in state:  # the containers of the loaded weights
        if case["op"] == "moe":
            state["w"] = tuple(QExpertsMXFP4(*state[m]) for m in ("gate", "up", "down"))
        else:
            state["w"] = (QExpertsMXFP4 if case["op"] == "grouped" else QWeightMXFP4)(state["packed"], state["scale"])
    if case["op"] in ("linear", "linear4"):
        x = ops.quantize_mxfp4(state["x"]) if case["op"] == "linear4" else state["x"]
        return ops.qlinear(x, state["w"], out_dtype=torch.bfloat16 if case["out"] == "bf16" else None)
    if case["op"] == "grouped":
        x = QWeightMXFP4(state["x_packed"], state["x_scale"]) if case["x"] == "mxfp4" else state["x"]
        return ops.qgemm_grouped(x, state["w"], state["offsets"])
    return ops.moe_ffn(state["x"], state["logits"], state["w"], top_k=case["top_k"])


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# ---- inputs -------------------------------------------------------------------------------------------------------------
def _result(case):
    """The type of a product's result: fp32 for up to 16 rows unless bf16 is asked for."""
    return torch.float32 if case["m"] <= 16 and case["out"] == "native" else torch.bfloat16


def _weights(g, *shape):
    """Normal weights, every row with a spread of its own, as codes and scales."""
    spread = torch.exp(torch.randn(*shape[:-1], 1, device=DEV, generator=g) * 0.5 - 4.0)
    return _quantize(torch.randn(*shape, device=DEV, generator=g) * spread)


def _activations(g, rows, k):
    """Normal activations, some channels of which are many times larger than the others, as in a decoder's hidden state."""
    gain = torch.exp(torch.randn(k, device=DEV, generator=g) * 0.7)
    return torch.randn(rows, k, device=DEV, generator=g) * gain


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    state = {"case": case}
    if case["op"] == "round":
        dtype = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[case["dtype"]]
        state["x"] = _activations(g, case["rows"], case["k"]).to(dtype)
    elif case["op"] in ("linear", "linear4"):
        state["x"] = _activations(g, case["m"], case["k"]).to(torch.bfloat16)
        state["packed"], state["scale"] = _weights(g, case["n"], case["k"])
    elif case["op"] == "grouped":
        rows, experts = case["rows"], case["experts"]
        share = torch.softmax(torch.randn(experts, device=DEV, generator=g), 0)  # some experts are liked more than others
        choice = torch.multinomial(share, rows, replacement=True, generator=g)
        counts = torch.bincount(choice, minlength=experts)
        state["offsets"] = torch.cat((counts.new_zeros(1), counts.cumsum(0))).to(torch.int32)
        state["most"] = int(counts.max())
        x = _activations(g, rows, case["k"])
        if case["x"] == "mxfp4":
            state["x_packed"], state["x_scale"] = _quantize(x)
        else:
            state["x"] = x.to(torch.bfloat16)
        state["packed"], state["scale"] = _weights(g, experts, case["n"], case["k"])
    else:
        e, h, f = case["experts"], case["h"], case["f"]
        state["x"] = _activations(g, case["tokens"], h).to(torch.bfloat16)
        state["logits"] = torch.randn(case["tokens"], e, device=DEV, generator=g)
        state["gate"], state["up"], state["down"] = _weights(g, e, f, h), _weights(g, e, f, h), _weights(g, e, h, f)
    return state


# ---- what a pass cannot do without --------------------------------------------------------------------------------------
def _bytes(*shape):
    return math.prod(shape) // 2 + math.prod(shape) // BLOCK


def work(case):
    if case["op"] == "round":
        r, k = case["rows"], case["k"]
        return {"bytes": r * k * (4 if case["dtype"] == "fp32" else 2) + _bytes(r, k) + 4 * r * k, "flops": 2 * r * k}
    if case["op"] in ("linear", "linear4"):
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": _bytes(n, k) + 2 * m * k + m * n * (4 if _result(case) == torch.float32 else 2), "flops": 2 * m * n * k}
    if case["op"] == "grouped":
        r, e, n, k = case["rows"], case["experts"], case["n"], case["k"]
        hit = e * (1 - (1 - 1 / e) ** r)  # experts that have a row, on average
        return {"bytes": hit * _bytes(n, k) + (_bytes(r, k) if case["x"] == "mxfp4" else 2 * r * k) + 2 * r * n + 4 * (e + 1), "flops": 2 * r * n * k}
    t, h, f, e, top_k = case["tokens"], case["h"], case["f"], case["experts"], case["top_k"]
    hit = e * (1 - (1 - top_k / e) ** t)
    return {"bytes": hit * 3 * _bytes(f, h) + 4 * t * h + 4 * t * e, "flops": 6 * t * top_k * h * f}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------
def _exact_values(packed, scale):
    """(-1)^s 2^(e - 1) (1 + m/2), or (-1)^s m/2 where e is 0, times 2^(byte - 127)."""
    nibbles = torch.empty(*packed.shape[:-1], packed.shape[-1] * 2, dtype=torch.uint8, device=packed.device)
    nibbles[..., 0::2], nibbles[..., 1::2] = packed % 16, packed // 16
    sign = 1.0 - 2.0 * (nibbles // 8).double()
    e, m = (nibbles // 2 % 4).double(), (nibbles % 2).double()
    magnitude = torch.where(e == 0, m / 2, torch.exp2(e - 1) * (1 + m / 2))
    return sign * magnitude * torch.exp2(scale.double() - 127).repeat_interleave(BLOCK, -1)


def _exact_rounded(x):
    """The values in 64 bits that x becomes in 4 bits: the nearest multiple of the spacing at each value, ties to the even one."""
    blocks = x.double().reshape(*x.shape[:-1], -1, BLOCK)
    largest = blocks.abs().max(-1, keepdim=True).values
    top = torch.where(largest > 0, torch.frexp(largest).exponent - 1, -125).clamp(min=-125)  # floor(log2(largest))
    scale = torch.exp2((top - 2).double())
    v = blocks / scale
    spacing = torch.exp2((torch.frexp(v).exponent - 2).clamp(min=-1).double())  # 1/2 below 2, 1 below 4, 2 beyond
    return ((v / spacing).round() * spacing).clamp(-6, 6).mul(scale).reshape(x.shape)


def _exact_silu(gate):
    return gate * torch.sigmoid(gate)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "round":
        return _exact_rounded(state["x"])
    if case["op"] in ("linear", "linear4"):
        x = _exact_rounded(state["x"]) if case["op"] == "linear4" else state["x"].double()
        return torch.mm(x, _exact_values(state["packed"], state["scale"]).t())
    if case["op"] == "grouped":
        x = _exact_values(state["x_packed"], state["x_scale"]) if case["x"] == "mxfp4" else state["x"].double()
        y = torch.zeros(case["rows"], case["n"], dtype=torch.float64, device=DEV)
        bounds = state["offsets"].tolist()
        for e, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
            y[lo:hi] = x[lo:hi] @ _exact_values(state["packed"][e], state["scale"][e]).t()
        return y
    x, logits, top_k = state["x"].double(), state["logits"].double(), case["top_k"]
    y = torch.zeros_like(x)
    rank = (logits[:, :, None] < logits[:, None, :]).sum(-1)  # how many experts a token likes more
    same = (logits[:, :, None] == logits[:, None, :]) & torch.ones(case["experts"], case["experts"], device=DEV).tril(-1).bool()
    taken = rank + same.sum(-1) < top_k
    share = torch.exp(logits - logits.max(-1, keepdim=True).values) * taken
    share = share / share.sum(-1, keepdim=True)
    for e in range(case["experts"]):
        gate, up, down = (_exact_values(state[m][0][e], state[m][1][e]) for m in ("gate", "up", "down"))
        y += share[:, e:e + 1] * ((_exact_silu(x @ gate.t()) * (x @ up.t())) @ down.t())
    return y
