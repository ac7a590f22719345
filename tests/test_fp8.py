"""FP8 by blocks of 128 and routing, on the CPU: the oracle against the formats' own definitions, containers, refusals, the weight file."""
import numpy as np
import pytest
import torch

from chadslab_amd import QExpertsFP8, QRowsFP8, QWeightFP8, wfile
from oracle import chadq_oracle as O

FP8 = torch.float8_e4m3fn


def test_every_byte_is_what_torch_reads():
    want = torch.arange(256, dtype=torch.uint8).view(FP8).double().numpy()
    assert np.array_equal(O.e4m3_values(), want, equal_nan=True)


def test_quantiser_rounds_as_torch_does():
    """With a = 448 the factor is 1 and what is left is the rounding: every border between two values, what lies beside it, and random numbers."""
    v = O.e4m3_values()[:127].astype(np.float32)
    mid = (v[1:] + v[:-1]) / 2
    x = np.concatenate([v, mid, np.nextafter(mid, np.float32(0)), np.nextafter(mid, np.float32(1000)), np.random.default_rng(1).uniform(0, 448, 1000).astype(np.float32)])
    x = np.concatenate([x, -x])
    x = np.pad(x, (0, -len(x) % 127)).reshape(-1, 127)
    x = np.concatenate([np.full((len(x), 1), 448, np.float32), x], 1)
    b, s = O.quantize_fp8(x, 1)
    assert (s == 1).all() and np.array_equal(b, torch.from_numpy(x).to(FP8).view(torch.uint8).numpy())


@pytest.mark.parametrize("high", [1, 128])
def test_quantiser_scales(high):
    r = np.random.default_rng(2)
    x = (r.standard_normal((200, 272)) * np.exp(r.standard_normal((200, 1)) * 3)).astype(np.float32)
    x[128:, 128:] = 0  # (whole blocks of either kind)
    b, s = O.quantize_fp8(x, high)
    assert s.shape == (200 if high == 1 else 2, 3)
    back = O.dequant_fp8(b, s, high)
    i, j = np.arange(200)[:, None] // high, np.arange(272)[None] // 128
    # half a step of a normal value, or of the smallest, and two fp32 roundings
    assert (np.abs(back - x) <= np.maximum(np.abs(x) * 2.0 ** -4, s[i, j] * 2.0 ** -10) * (1 + 2.0 ** -20)).all()
    assert s.min() == np.float32(2.0 ** -126)


def test_quantiser_blocks_that_are_not_finite():
    x = np.ones((3, 256), np.float32)
    x[0, 5], x[1, 200] = np.nan, np.inf
    b, s = O.quantize_fp8(x, 1)
    assert np.isnan(s[0, 0]) and np.isnan(s[1, 1]) and np.isfinite(s[[0, 1, 2, 2], [1, 0, 0, 1]]).all() and not b[0, :128].any()


# ---- routing --------------------------------------------------------------------------------------------------------------
def test_routing_is_the_softmax_one():
    z = np.random.default_rng(3).standard_normal((40, 12)).astype(np.float32)
    z[5, 3] = z[5, 7] = z[5].max() + 1
    for renorm in (True, False):
        idx, w = O.moe_route_experts(z, 3, renorm)
        want, ww = O.moe_route(z, 3, renorm)
        assert np.array_equal(idx, want) and np.allclose(w, ww, rtol=1e-6)


def test_routing_bias_chooses_and_does_not_weigh():
    z = np.array([[0.0, 1.0, 2.0, 3.0]])
    idx, w = O.moe_route_experts(z, 2, False, "sigmoid", bias=np.array([1.0, 0.0, 0.0, 0.0]), scale=2.0)
    assert idx.tolist() == [[0, 3]] and np.allclose(w, [[1.0, 2 / (1 + np.exp(-3.0))]])


def test_routing_groups():
    z = np.array([[3.0, -9, 2, 1.9, 1, 1, 2.5, -9]])
    assert O.moe_route_experts(z, 2, groups=4, top_groups=1)[0].tolist() == [[0, 1]]
    assert O.moe_route_experts(z, 2, groups=4, top_groups=2)[0].tolist() == [[0, 6]]
    assert O.moe_route_experts(z, 2, score="sigmoid", groups=4, top_groups=1, group_sum=2)[0].tolist() == [[2, 3]]


def test_routing_masked_experts():
    z = np.full((2, 6), -np.inf)
    z[0, 4], z[0, 1] = 1.0, np.nan
    idx, w = O.moe_route_experts(z, 2, bias=np.ones(6))
    assert idx.tolist() == [[4, 0], [0, 1]] and w.tolist() == [[1, 0], [0, 0]]


# ---- containers -----------------------------------------------------------------------------------------------------------
def test_containers():
    w = QWeightFP8(torch.zeros(300, 272).to(FP8), torch.zeros(3, 3))
    assert (w.N, w.K) == (300, 272)
    e = QExpertsFP8(torch.zeros(4, 130, 16).to(FP8), torch.zeros(4, 2, 1))
    assert (e.E, e.N, e.K) == (4, 130, 16) and e.expert(2).scale.shape == (2, 1)
    x = QRowsFP8(torch.zeros(5, 144).to(FP8), torch.zeros(5, 2))
    assert (x.M, x.K) == (5, 144) and type(x.to("cpu")) is QRowsFP8
    for make in (lambda: QWeightFP8(w.w.view(torch.uint8), w.scale), lambda: QWeightFP8(w.w, w.scale[:2]), lambda: QWeightFP8(w.w, w.scale.double()),
                 lambda: QWeightFP8(w.w[:, :8], w.scale[:, :1]), lambda: QExpertsFP8(e.w, e.scale[:3]), lambda: QExpertsFP8(w.w, w.scale),
                 lambda: QRowsFP8(x.w, x.scale[:1]), lambda: QRowsFP8(e.w, e.scale)):
        with pytest.raises(ValueError):
            make()


def test_weight_file(tmp_path):
    r = np.random.default_rng(4)
    w = QWeightFP8(torch.from_numpy(r.integers(0, 127, (130, 144), dtype=np.uint8)).view(FP8), torch.from_numpy(r.random((2, 2), np.float32)))
    e = QExpertsFP8(torch.from_numpy(r.integers(0, 127, (3, 20, 16), dtype=np.uint8)).view(FP8), torch.from_numpy(r.random((3, 1, 1), np.float32)))
    path = str(tmp_path / "w")
    wfile.save(path, {"w": w, "e": e})
    got = wfile.load(path)
    for a, b in ((w, got["w"]), (e, got["e"])):
        assert type(a) is type(b) and torch.equal(a.w.view(torch.uint8), b.w.view(torch.uint8)) and torch.equal(a.scale, b.scale)


def test_what_the_operators_refuse_without_a_gpu():
    """Everything that can be said before a device is needed; nothing computes on the CPU."""
    from chadslab_amd import ops

    x = torch.zeros(3, 32)
    for call, error in ((lambda: ops.quantize_fp8(x), "GPU tensor"), (lambda: ops.quantize_fp8(x.double()), "float32, bfloat16"), (lambda: ops.quantize_fp8(x[:, :8]), "multiple of 16"),
                        (lambda: ops.quantize_fp8(x[None]), r"\[M,K\]"), (lambda: ops.quantize_fp8(x[0], rows=False), r"\[N,K\]"),
                        (lambda: ops.moe_route(x, score="max"), "softmax"), (lambda: ops.moe_route(x, 2, groups=2), "GPU tensor")):
        with pytest.raises(ValueError, match=error):
            call()
    w = QWeightFP8(torch.zeros(32, 32).to(FP8), torch.zeros(1, 1))
    with pytest.raises(ValueError, match=r"\[M,32\]"):
        ops.qlinear(x[:, :16].bfloat16(), w)
    with pytest.raises(TypeError, match="bias"):
        ops.moe_route(x, bias=3.0)
    with pytest.raises(TypeError, match="FP8 activations"):
        from chadslab_amd import QWeightInt8
        ops.qlinear(QRowsFP8(torch.zeros(3, 32).to(FP8), torch.zeros(3, 1)), QWeightInt8(torch.zeros(8, 32, dtype=torch.int8), torch.zeros(8)))


def test_routing_bias_that_is_not_finite():
    """Switched off: behind all others, in front of masked ones.  NaN as -infinity; a group's +infinity + -infinity as +infinity."""
    z = np.array([[0, -np.inf, 1, -np.inf]])
    inf = np.inf
    assert O.moe_route_experts(z, 2, score="sigmoid", bias=np.array([-inf, 0, 0, 0]))[0].tolist() == [[2, 0]]
    assert O.moe_route_experts(z, 3, score="sigmoid", bias=np.array([np.nan, 0, 0, 0]))[0].tolist() == [[2, 0, 1]]
    z = np.array([[0.0, 1, 2, 3, 4, 5]])
    assert O.moe_route_experts(z, 2, groups=3, group_sum=2, bias=np.array([inf, -inf, -inf, 0, -inf, -inf]))[0].tolist() == [[0, 1]]
    assert O.moe_route_experts(z, 2, groups=3, group_sum=2, bias=np.array([-inf, -inf, -inf, 0, -inf, -inf]))[0].tolist() == [[0, 1]]  # (all sums alike)
