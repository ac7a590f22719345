"""Routing to experts on the GPU against the oracle in 64 bits: the same experts in the same order, weights within fp32 roundings (the scores are formed in
64 bits, or in 32 by an exponential of at most 2 steps and sums of at most 512 terms by halving: 2^-23 * (2 + 9 + 4) at most)."""
import numpy as np
import pytest
import torch

from oracle import chadq_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BOUND = 15 * 2.0 ** -23


@pytest.fixture(scope="module")
def ops():
    from chadslab_amd import _lib, ops as _ops

    assert torch.cuda.is_available(), "these tests need the GPU"
    _lib.load()
    return _ops


def check(ops, z, bias=None, **how):
    idx, w = ops.moe_route(torch.from_numpy(z).to(DEV), bias=None if bias is None else torch.from_numpy(bias).to(DEV), **how)
    want, ww = O.moe_route_experts(z, bias=bias, **how)
    assert idx.dtype == torch.int32 and w.dtype == torch.float32 and idx.shape == w.shape == want.shape
    assert np.array_equal(idx.cpu().numpy(), want)
    assert (np.abs(w.cpu().numpy() - ww) <= BOUND * np.abs(ww) + 2.0 ** -126).all()


HOWS = [dict(), dict(renorm=False), dict(score="sigmoid"), dict(score="sigmoid", renorm=False, scale=2.5)]
SIZES = [(1, 1), (3, 1), (7, 3), (8, 8), (9, 2), (16, 4), (17, 6), (32, 32), (33, 8), (60, 4), (64, 32), (100, 5), (128, 8), (160, 6), (256, 8), (300, 32), (384, 8), (512, 1)]


@pytest.mark.parametrize("how", HOWS)
@pytest.mark.parametrize("experts,top_k", SIZES)
def test_sizes(ops, experts, top_k, how):
    r = np.random.Generator(np.random.PCG64(experts * 100 + top_k))
    bias = (r.standard_normal(experts) * 0.1).astype(np.float32)
    for tokens in (1, 5, 130):
        z = (r.standard_normal((tokens, experts)) * 2).astype(np.float32)
        if len(how) or experts > 16:
            check(ops, z, top_k=top_k, **how)
        check(ops, z, bias, top_k=top_k, **how)


@pytest.mark.parametrize("experts,groups", [(8, 8), (8, 2), (12, 3), (16, 4), (60, 4), (64, 64), (64, 8), (160, 8), (256, 8), (384, 8), (500, 5), (512, 64)])
def test_groups(ops, experts, groups):
    r = np.random.Generator(np.random.PCG64(experts + groups))
    per = experts // groups
    for score in ("softmax", "sigmoid"):
        for bias in (None, (r.standard_normal(experts) * 0.1).astype(np.float32)):
            for group_sum in (1, 2)[:per]:
                for top_groups in {1, (groups + 1) // 2, groups}:
                    top_k = min(8, top_groups * per)
                    z = (r.standard_normal((37, experts)) * 2).astype(np.float32)
                    check(ops, z, bias, top_k=top_k, score=score, groups=groups, top_groups=top_groups, group_sum=group_sum)


@pytest.mark.parametrize("experts,groups,top_k", [(8, 2, 4), (16, 1, 16), (33, 3, 8), (40, 1, 6), (60, 4, 4), (64, 8, 8), (64, 1, 17), (100, 5, 12), (128, 8, 8), (160, 8, 6), (160, 20, 6),
                                                  (256, 8, 8), (256, 1, 16), (300, 6, 8), (384, 8, 8), (512, 16, 16), (512, 1, 8)])
def test_many_tokens(ops, experts, groups, top_k):
    """As many as take fewer lanes each; ties and masked experts among them."""
    r = np.random.Generator(np.random.PCG64(experts + groups))
    z = (r.standard_normal((2500, experts)) * 2).astype(np.float32)
    z[::7] = np.rint(z[::7])
    z[::11][r.random(z[::11].shape) < 0.3] = -np.inf
    bias = (r.standard_normal(experts) * 0.1).astype(np.float32)
    top_groups = max(1, -(-top_k // (experts // groups)), groups // 2)
    for how in (dict(), dict(score="sigmoid", renorm=False, scale=2.5)):
        check(ops, z, None, top_k=top_k, groups=groups, top_groups=top_groups, **how)
        check(ops, z, bias, top_k=top_k, groups=groups, top_groups=top_groups, group_sum=2 if groups > 1 and experts // groups > 1 else 1, **how)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("experts,groups", [(8, 1), (16, 4), (40, 1), (64, 8), (256, 8), (400, 1)])
def test_ties_go_to_the_lowest_index(ops, experts, groups, wide):
    """Logits of few different values, -0 and 0 among them; groups of the same value too."""
    r = np.random.Generator(np.random.PCG64(experts))
    z = r.choice(np.array([0.0, -0.0, 1.0, 1.5], np.float32), (200, experts))
    z[0] = 0.25
    check(ops, z, np.zeros(experts, np.float32) if wide else None, top_k=8, groups=groups, top_groups=max(1, groups // 2), score="sigmoid")


def test_near_ties_are_told_apart(ops):
    """Scores that 32 bits would round to the same number: sigmoid near 1, and a bias below its last bit."""
    z = np.zeros((1, 64), np.float32)
    z[0] = 20 + np.arange(64, dtype=np.float32) * 2.0 ** -18  # sigmoid: steps of 2^-18 * 2^-28.8
    check(ops, z, np.zeros(64, np.float32), top_k=8, score="sigmoid")
    bias = np.arange(64, dtype=np.float32) * np.float32(2.0 ** -40)
    check(ops, np.zeros((1, 64), np.float32), bias, top_k=8, score="sigmoid")


@pytest.mark.parametrize("how", HOWS[:3])
@pytest.mark.parametrize("biased", [False, True])
def test_masked_experts_and_rows(ops, how, biased):
    """-infinity and NaN come last with the score 0, also where a bias speaks for them; a row with nothing else gets the first ones with weights of 0; the
    type's lowest value is a number like others."""
    r = np.random.Generator(np.random.PCG64(4))
    z = r.standard_normal((60, 40)).astype(np.float32)
    z[r.random(z.shape) < 0.5] = -np.inf
    z[r.random(z.shape) < 0.1] = np.nan
    z[0], z[1], z[2], z[3] = -np.inf, np.nan, -np.inf, np.finfo(np.float32).min
    z[2, 33] = 0.5
    z[4, :39] = np.finfo(np.float32).min
    bias = (r.standard_normal(40)).astype(np.float32) if biased else None
    for groups in (1, 5):
        check(ops, z, bias, top_k=6, groups=groups, top_groups=(groups + 1) // 2, **how)


@pytest.mark.parametrize("how", HOWS)
def test_large_logits(ops, how):
    r = np.random.Generator(np.random.PCG64(5))
    z = (r.standard_normal((50, 48)) * 60).astype(np.float32)
    check(ops, z, top_k=4, **how)
    z = (np.abs(r.standard_normal((50, 48))) * -60 - 100).astype(np.float32)
    check(ops, z, top_k=4, **how)


def test_many_tokens_strides_and_none(ops):
    r = np.random.Generator(np.random.PCG64(6))
    z, bias = r.standard_normal((3000, 256)).astype(np.float32), (r.standard_normal(256) * 0.05).astype(np.float32)
    check(ops, z, bias, top_k=8, score="sigmoid", groups=8, top_groups=4, group_sum=2, scale=2.5)
    t = torch.from_numpy(z).to(DEV)
    a, b = ops.moe_route(t[::3, :128], 4, score="sigmoid"), ops.moe_route(t[::3, :128].contiguous(), 4, score="sigmoid")
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    idx, w = ops.moe_route(t[:0], 4, score="sigmoid")
    assert idx.shape == w.shape == (0, 4)
    # 2^32 bytes and more of logits: the last token is the first one again
    big = torch.zeros(2 ** 31 // 512 + 8, 512, device=DEV)
    big[-1, :256] = t[0] + 9
    idx, w = ops.moe_route(big, 8, score="sigmoid")
    assert torch.equal(idx[-1], ops.moe_route(t[:1] + 9, 8, score="sigmoid")[0][0]) and bool((idx[0] == torch.arange(8, device=DEV)).all())


def test_replays(ops):
    r = np.random.Generator(np.random.PCG64(7))
    z, bias = torch.from_numpy(r.standard_normal((70, 160)).astype(np.float32)).to(DEV), torch.zeros(160, device=DEV)
    how = dict(top_k=6, score="sigmoid", bias=bias, groups=8, top_groups=3, group_sum=2)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.moe_route(z, **how)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        got = ops.moe_route(z, **how)
    for turn in range(3):
        z.copy_(torch.randn_like(z))
        bias.copy_(torch.randn_like(bias) * 0.1)
        want = ops.moe_route(z, **how)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals(ops):
    z = torch.zeros(3, 64, device=DEV)
    for call, match in ((lambda: ops.moe_route(z, 33), "top_k"), (lambda: ops.moe_route(z, 0, score="sigmoid"), "top_k"), (lambda: ops.moe_route(z, -1, score="sigmoid"), "top_k"),
                        (lambda: ops.moe_route(z, 2, groups=5), "groups"), (lambda: ops.moe_route(z, 2, groups=8, top_groups=9), "top_groups"),
                        (lambda: ops.moe_route(z, 2, groups=64, group_sum=2), "group_sum"), (lambda: ops.moe_route(z, 9, groups=8, top_groups=1), "top_k"),
                        (lambda: ops.moe_route(z.double(), 2, score="sigmoid"), "float32"), (lambda: ops.moe_route(z[0], 2, score="sigmoid"), r"\[T,E\]"),
                        (lambda: ops.moe_route(torch.zeros(3, 513, device=DEV), 2), "E"), (lambda: ops.moe_route(z, 2, bias=z[0, :5]), "bias must"),
                        (lambda: ops.moe_route(z, 2, bias=z[0].cpu()), "GPU tensor"), (lambda: ops.moe_route(z, 2, bias=z[0].half()), "float32")):
        with pytest.raises(ValueError, match=match):
            call()


def test_switched_off_experts_come_before_masked_ones(ops):
    z = np.array([[0, -np.inf, 1, -np.inf]], np.float32)
    bias = np.array([-np.inf, 0, 0, 0], np.float32)
    idx, _ = ops.moe_route(torch.from_numpy(z).to(DEV), 2, score="sigmoid", bias=torch.from_numpy(bias).to(DEV))
    assert idx.tolist() == [[2, 0]]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,groups", [(8, 1), (8, 2), (12, 3), (16, 4), (40, 5), (64, 1), (64, 8), (64, 32), (160, 20), (256, 8), (300, 6), (512, 64)])
def test_bias_that_is_not_finite(ops, experts, groups, score):
    """Experts switched off (-infinity, NaN) and always taken (+infinity), beside masked ones, in groups that have none, one or more of each; as many chosen as there may be."""
    r = np.random.Generator(np.random.PCG64(experts + groups))
    per = experts // groups
    for kind in (0.3, 0.9, 1.0):
        bias = (r.standard_normal(experts) * 0.1).astype(np.float32)
        bias[r.random(experts) < kind] = -np.inf
        bias[r.random(experts) < 0.1] = np.nan
        if kind < 1:
            bias[r.random(experts) < 0.1] = np.inf
        z = (r.standard_normal((70, experts)) * 2).astype(np.float32)
        z[::2][r.random(z[::2].shape) < 0.5] = -np.inf
        z[::5][r.random(z[::5].shape) < 0.1] = np.nan
        z[0], z[1] = -np.inf, 0.5
        for top_groups in {1, (groups + 1) // 2, groups}:
            for group_sum in (1, 2)[:per]:
                check(ops, z, bias, top_k=min(32, top_groups * per), score=score, groups=groups, top_groups=top_groups, group_sum=group_sum, renorm=False)


@pytest.mark.parametrize("tokens", [3, 70, 3000])
def test_layer_with_experts_switched_off(ops, tokens):
    """-infinity is the least of all biases: the layer is the one with a very low finite one, bit for bit, also where no more experts are left but masked ones."""
    r = np.random.Generator(np.random.PCG64(tokens))
    triple = [ops.quantize_fp8(torch.from_numpy(r.standard_normal(shape).astype(np.float32)).to(DEV), rows=False) for shape in ((8, 48, 64), (8, 48, 64), (8, 64, 48))]
    x = torch.from_numpy(r.standard_normal((tokens, 64)).astype(np.float32)).to(DEV).bfloat16()
    z = torch.from_numpy(r.standard_normal((tokens, 8)).astype(np.float32)).to(DEV)
    z[:, 5:] = -np.inf
    bias = torch.zeros(8, device=DEV)
    for off in ([0, 1], [0, 1, 2, 3], list(range(8))):
        for how in (dict(score="sigmoid"), dict(groups=4, top_groups=3, group_sum=2)):
            bias[off] = -1e30
            want = ops.moe_ffn(x, z, triple, top_k=4, bias=bias, **how)
            bias[off] = -np.inf
            assert torch.equal(ops.moe_ffn(x, z, triple, top_k=4, bias=bias, **how), want)


@pytest.mark.parametrize("experts,tokens", [(33, 2 ** 26 + 5), (2, 2 ** 29 + 70)])
def test_more_tokens_than_a_launch_has_threads_for(ops, experts, tokens):
    """2^32 lanes and more: every token is somebody's, and the ones at the borders are right."""
    r = np.random.Generator(np.random.PCG64(experts))
    z = torch.from_numpy(r.standard_normal((7, experts)).astype(np.float32)).to(DEV)
    at = torch.tensor([0, 2 ** 24 - 1, 2 ** 24, 2 ** 26 - 1, 2 ** 26, tokens // 2, tokens - 1], device=DEV)
    logits = torch.zeros(tokens, experts, device=DEV)
    logits[at] = z
    bias = torch.zeros(experts, device=DEV)
    bias[1] = 0.25  # (so that no token's answer is what fresh memory may hold)
    idx, w = ops.moe_route(logits, 1, score="sigmoid", bias=bias, renorm=False)
    want = ops.moe_route(z, 1, score="sigmoid", bias=bias, renorm=False)
    assert torch.equal(idx[at], want[0]) and torch.equal(w[at], want[1])
    idx[at], w[at] = 1, 0.5
    assert bool((idx == 1).all()) and bool((w == 0.5).all())


@pytest.mark.parametrize("experts,top_k", [(1, 1), (3, 2), (8, 2), (8, 8), (16, 1), (16, 8)])
def test_plain_routing_goes_the_short_way(ops, experts, top_k):
    """Softmax over at most 16: chadq_moe_route's bits from the native call, NaN and rows of nothing but -infinity as they are there."""
    from chadslab_amd import _lib

    r = np.random.Generator(np.random.PCG64(experts + top_k))
    z = torch.from_numpy(r.standard_normal((33, experts)).astype(np.float32)).to(DEV)
    z[3], z[5, 0], z[7] = -np.inf, np.nan, 0.25
    for renorm in (True, False):
        idx, w = torch.empty(33, top_k, dtype=torch.int32, device=DEV), torch.empty(33, top_k, device=DEV)
        _lib.check(_lib.load().chadq_moe_route(z.data_ptr(), idx.data_ptr(), w.data_ptr(), 33, experts, top_k, int(renorm), torch.cuda.current_stream().cuda_stream), "chadq_moe_route")
        for got in (_lib.native().route(z, None, False, renorm, 1, 1, 1, top_k, 1.0), ops.moe_route(z, top_k, renorm), ops.moe_route(z, top_k, np.bool_(renorm))):
            assert torch.equal(got[0], idx) and torch.equal(got[1].view(torch.int32), w.view(torch.int32))
