"""MXFP4 on the GPU, through chadslab_amd.ops, against the oracle in 64 bits.  Quantisation and its inverse bit for bit.

Products.  bf16 x e2m1 and e2m1 x e2m1 are exact in fp32 and so are the scales, so what is off is the sums.  With S = sum_k |x w| of
an element, every fp32 addition is off by at most 2^-24 S; a matrix instruction adds 32 (bf16) or 128 products and its operand C in
at most 4 roundings' worth (2^-22 S), an element takes at most K/16 of them, and at most 64 partial sums are joined:
|y - exact| <= (K/16 * 4 + 64) 2^-24 S; a result in bf16 adds half a step, 2^-8 |y|.  (And 2^-126 for what is below the normal numbers.)"""
import numpy as np
import pytest
import torch

from oracle import chadq_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from chadslab_amd import _lib, ops as _ops

    assert torch.cuda.is_available(), "these tests need the GPU"
    _lib.load()
    return _ops


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def weights(r, *shape, spread=1.0):
    """Any codes; scales around 2^-6."""
    *lead, k = shape
    codes = r.integers(0, 256, (*lead, k // 2), dtype=np.uint8)
    scale = np.clip(np.rint(r.standard_normal((*lead, k // 32)) * spread + 121), 0, 254).astype(np.uint8)
    return codes, scale


def activations(r, m, k, x4):
    """-> (what the operators take, the same values in 64 bits)"""
    from chadslab_amd import QWeightMXFP4

    if x4:
        c, s = weights(r, m, k)
        return QWeightMXFP4(dev(c), dev(s)), torch.from_numpy(O.dequant_mxfp4(c, s)).to(DEV)
    x = torch.from_numpy(r.standard_normal((m, k)).astype(np.float32)).to(torch.bfloat16).to(DEV)
    return x, x.double()


def check(y, x64, w64):
    """Element by element, with the bound above; x64 [M,K], w64 [N,K] in 64 bits."""
    exact, s = x64 @ w64.T, x64.abs() @ w64.abs().T
    bound = (x64.shape[1] / 4 + 64) * 2.0 ** -24 * s + 2.0 ** -126
    if y.dtype == torch.bfloat16:
        bound = bound + 2.0 ** -8 * exact.abs()
    off = (y.double() - exact).abs()
    assert torch.isfinite(y).all() and bool((off <= bound).all()), "off by %.3g bounds" % float((off / bound).max())


# ---- quantisation --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,k", [(1, 32), (3, 96), (7, 4096), (129, 2080), (1000, 64)])
def test_quantize_is_the_oracles(ops, rows, k, dtype):
    r = np.random.Generator(np.random.PCG64(rows + k))
    x = r.standard_normal((rows, k)) * np.exp(r.standard_normal((rows, 1)) * 3)
    x[r.random((rows, k)) < 0.1] = 0.0
    edge = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.75, -0.25, -0.75, -1.25, -2.5, -5.0, -0.0])
    x[0, :16] = edge
    xt = torch.from_numpy(x).to(dtype)
    q = ops.quantize_mxfp4(xt.to(DEV))
    codes, scale = O.quantize_mxfp4(xt.double().numpy())
    assert np.array_equal(q.packed.cpu().numpy(), codes) and np.array_equal(q.scale.cpu().numpy(), scale)
    back = ops.dequantize(q)
    assert back.dtype == torch.float32 and np.array_equal(back.cpu().double().numpy(), O.dequant_mxfp4(codes, scale))


def test_quantize_every_bf16_beside_every_binade(ops):
    """Every finite bf16 as the second value of a block whose first is a power of two: scales from the smallest to the largest, codes at every border."""
    bits = np.arange(65536, dtype=np.uint16)
    v = O.bf16_to_f32(bits)
    v = v[np.isfinite(v)]
    x = np.zeros((len(v), 32), np.float32)
    x[:, 1] = v
    x[:, 0] = np.ldexp(1.0, (np.arange(len(v)) * 7) % 254 - 126).astype(np.float32)
    q = ops.quantize_mxfp4(dev(x).to(torch.bfloat16))
    codes, scale = O.quantize_mxfp4(x)
    assert np.array_equal(q.packed.cpu().numpy(), codes) and np.array_equal(q.scale.cpu().numpy(), scale)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_quantize_extremes(ops, dtype):
    info = torch.finfo(dtype)
    tiny = float(torch.tensor(info.smallest_normal * info.eps, dtype=dtype))
    x = np.zeros((8, 64))
    x[0, 3], x[0, 40] = np.nan, 1.0
    x[1, 5], x[1, 41] = np.inf, -2.0
    x[2, 6], x[2, 42] = -np.inf, 0.3
    x[3, 0], x[3, 1] = info.max, -info.max
    x[4, 0], x[4, 1], x[4, 32] = tiny, -tiny, info.smallest_normal
    x[5] = -0.0
    x[6, :32], x[6, 32:] = 1e-3, 7.0
    xt = torch.from_numpy(x).to(dtype)
    q = ops.quantize_mxfp4(xt.to(DEV))
    codes, scale = O.quantize_mxfp4(xt.double().numpy())
    assert np.array_equal(q.packed.cpu().numpy(), codes) and np.array_equal(q.scale.cpu().numpy(), scale)
    back, want = ops.dequantize(q).cpu().double().numpy(), O.dequant_mxfp4(codes, scale)
    assert np.array_equal(back, want, equal_nan=True) and np.isnan(back[0, :32]).all() and back[0, 40 - 8] == want[0, 32]


def test_dequantize_every_code_with_every_scale(ops):
    from chadslab_amd import QExpertsMXFP4

    codes = np.tile((np.arange(16, dtype=np.uint8)[0::2] | (np.arange(16, dtype=np.uint8)[1::2] << 4)), (2, 128, 2))
    scale = np.arange(256, dtype=np.uint8).reshape(2, 128, 1)
    got = ops.dequantize(QExpertsMXFP4(dev(codes), dev(scale))).cpu().numpy()
    with np.errstate(over="ignore"):
        assert np.array_equal(got, O.dequant_mxfp4(codes, scale).astype(np.float32), equal_nan=True)  # (6 x 2^127 is infinite)


def test_quantize_views_and_experts(ops):
    r = np.random.Generator(np.random.PCG64(3))
    x = dev(r.standard_normal((4, 6, 128)).astype(np.float32))
    q = ops.quantize_mxfp4(x.transpose(0, 1))  # a strided view: [6,4,128]
    codes, scale = O.quantize_mxfp4(x.transpose(0, 1).reshape(24, 128).cpu().numpy())
    assert q.E == 6 and np.array_equal(q.packed.cpu().numpy().reshape(24, 64), codes) and np.array_equal(q.scale.cpu().numpy().reshape(24, 4), scale)
    assert ops.quantize_mxfp4(x[:, :, :0]).K == 0 and ops.quantize_mxfp4(x[:0]).E == 0
    assert ops.dequantize(ops.quantize_mxfp4(x[0, :0])).shape == (0, 128)
    with pytest.raises(ValueError, match="aligned"):
        ops.quantize_mxfp4(torch.zeros(1 + 64, device=DEV)[1:].view(2, 32))


# ---- products ------------------------------------------------------------------------------------------------------------
MS = [1, 2, 3, 5, 8, 9, 16, 17, 31, 33, 48, 64, 65, 100, 129, 200, 257]
NKS = [(1, 32), (16, 128), (33, 160), (250, 96), (64, 2080), (130, 4096), (515, 544), (96, 7200)]


@pytest.mark.parametrize("x4", [False, True], ids=["bf16", "mxfp4"])
@pytest.mark.parametrize("n,k", NKS)
def test_products(ops, n, k, x4):
    from chadslab_amd import QWeightMXFP4

    r = np.random.Generator(np.random.PCG64(n * 10007 + k))
    c, s = weights(r, n, k)
    qw, w64 = QWeightMXFP4(dev(c), dev(s)), dev(O.dequant_mxfp4(c, s))
    for m in MS:
        x, x64 = activations(r, m, k, x4)
        y = ops.qlinear(x, qw)
        assert y.shape == (m, n) and y.dtype == (torch.float32 if m <= 16 else torch.bfloat16)
        check(y, x64, w64)
        if m <= 16:
            check(ops.qgemv(x, qw), x64, w64)
            yb = ops.qlinear(x, qw, out_dtype=torch.bfloat16)
            assert yb.dtype == torch.bfloat16 and torch.equal(yb, y.to(torch.bfloat16))  # the same sums, rounded once
        y = ops.qgemm(x, qw)
        assert y.dtype == torch.bfloat16
        check(y, x64, w64)


@pytest.mark.parametrize("x4", [False, True], ids=["bf16", "mxfp4"])
@pytest.mark.parametrize("m,n,k", [(1, 14336, 4096), (16, 1000, 14368), (40, 4100, 1056), (300, 2064, 1184), (512, 4096, 4096), (1030, 777, 2048), (2050, 520, 352)])
def test_larger_products(ops, m, n, k, x4):
    from chadslab_amd import QWeightMXFP4

    r = np.random.Generator(np.random.PCG64(m + n + k))
    c, s = weights(r, n, k)
    x, x64 = activations(r, m, k, x4)
    check(ops.qlinear(x, QWeightMXFP4(dev(c), dev(s))), x64, dev(O.dequant_mxfp4(c, s)))


@pytest.mark.parametrize("x4", [False, True], ids=["bf16", "mxfp4"])
@pytest.mark.parametrize("m", [1, 7, 40, 200])
def test_integer_products_are_exact(ops, m, x4):
    """Small integers: every partial sum is an integer below 2^24, so any order gives the same."""
    from chadslab_amd import QWeightMXFP4

    r = np.random.Generator(np.random.PCG64(m))
    n, k = 100, 512
    w = r.choice([0, 1, 2, 3, 4, 6, -1, -2, -3, -4, -6], (n, k)).astype(np.float64)
    w[:, ::32] = 4
    x = r.choice([0, 1, 2, 3, 4, -1, -2, -3, -4], (m, k)).astype(np.float64)
    x[:, ::32] = 4
    c, s = O.quantize_mxfp4(w)
    assert np.array_equal(O.dequant_mxfp4(c, s), w)
    qw = QWeightMXFP4(dev(c), dev(s))
    xq = ops.quantize_mxfp4(dev(x.astype(np.float32))) if x4 else dev(x.astype(np.float32)).to(torch.bfloat16)
    y = ops.qgemv(xq, qw) if m <= 16 else ops.qgemm(xq, qw)
    assert np.array_equal(y.double().cpu().numpy(), torch.from_numpy(x @ w.T).to(y.dtype).double().numpy())


@pytest.mark.parametrize("x4", [False, True], ids=["bf16", "mxfp4"])
@pytest.mark.parametrize("m", [2, 40, 200])
def test_nan_blocks_stay_in_their_row_and_column(ops, m, x4):
    from chadslab_amd import QWeightMXFP4

    r = np.random.Generator(np.random.PCG64(m + 1))
    n, k = 70, 224  # K ends inside a unit: what lies behind it must not leak in
    c, s = weights(r, n, k)
    s[3, 6], s[50, 0] = 255, 255  # the last and the first block of a row
    x, x64 = activations(r, m, k, x4)
    if x4:
        x.scale[1, 2] = 255
    else:
        x[1, 65] = float("nan")
    y = ops.qlinear(x, QWeightMXFP4(dev(c), dev(s)))
    want = torch.zeros(m, n, dtype=torch.bool)
    want[1], want[:, 3], want[:, 50] = True, True, True
    assert torch.equal(torch.isnan(y).cpu(), want)
    s[3, 6] = s[50, 0] = 120
    w64 = dev(O.dequant_mxfp4(c, s))
    keep_m, keep_n = [i for i in range(m) if i != 1], [i for i in range(n) if i not in (3, 50)]
    check(y[keep_m][:, keep_n], x64[keep_m], w64[keep_n])


@pytest.mark.parametrize("m", [2, 40, 200])
def test_infinite_activations(ops, m):
    """As IEEE has it: infinity times a weight that is 0 is NaN, else infinite."""
    from chadslab_amd import QWeightMXFP4

    c = np.zeros((3, 32), np.uint8)
    s = np.full((3, 2), 127, np.uint8)
    c[0, 0], c[1, 0] = 2, 10  # k = 0: 1, -1, 0
    x = torch.zeros(m, 64, dtype=torch.bfloat16, device=DEV)
    x[1, 0] = float("inf")
    y = ops.qlinear(x, QWeightMXFP4(dev(c), dev(s)))
    assert y[1, 0] == float("inf") and y[1, 1] == -float("inf") and torch.isnan(y[1, 2]) and bool((y[0] == 0).all())


@pytest.mark.parametrize("k", [32, 96, 288, 800, 1056, 4128])
@pytest.mark.parametrize("m", [1, 3, 16, 40])
def test_weights_beyond_bf16_in_the_last_block(ops, m, k):
    """They count as infinite, and the activations behind the row's end, zeros, may not meet them: infinity times zero is NaN."""
    from chadslab_amd import QExpertsMXFP4, QWeightMXFP4

    c = np.zeros((2, 24, k // 2), np.uint8)
    s = np.full((2, 24, k // 32), 127, np.uint8)
    s[0, 5, -1], s[1, 7, -1] = 254, 253
    c[0, 5, -16:], c[1, 7, -16:] = 0x44, 0x77  # 2 x 2^127, 6 x 2^126
    x = torch.ones(m, k, dtype=torch.bfloat16, device=DEV)
    want = torch.zeros(2, m, 24, device=DEV)
    want[0, :, 5] = want[1, :, 7] = float("inf")
    for e in range(2):
        assert torch.equal(ops.qlinear(x, QWeightMXFP4(dev(c[e]), dev(s[e]))).float(), want[e])
    half = m // 2
    y = ops.qgemm_grouped(x, QExpertsMXFP4(dev(c), dev(s)), torch.tensor([0, half, m], dtype=torch.int32, device=DEV))
    assert torch.equal(y.float(), torch.cat((want[0, :half], want[1, half:])))


@pytest.mark.parametrize("m", [1, 33, 150])
def test_extreme_scales(ops, m):
    """Scales at both ends of the bytes; 2^-100 against 2^100 has to come out as if neither were there."""
    from chadslab_amd import QWeightMXFP4

    r = np.random.Generator(np.random.PCG64(m + 9))
    n, k = 40, 256
    c, _ = weights(r, n, k)
    xc, _ = weights(r, m, k)
    w64 = dev(O.dequant_mxfp4(c, np.full((n, k // 32), 127, np.uint8)))
    x64 = dev(O.dequant_mxfp4(xc, np.full((m, k // 32), 127, np.uint8)))
    for a, b in ((27, 227), (227, 27), (1, 253), (127, 127), (0, 254)):
        qw, xq = (QWeightMXFP4(dev(v), torch.full((v.shape[0], k // 32), e, dtype=torch.uint8, device=DEV)) for v, e in ((c, a), (xc, b)))
        check(ops.qlinear(xq, qw) * 2.0 ** (254 - a - b), x64, w64)


def test_strides_outputs_and_refusals(ops):
    from chadslab_amd import QWeightMXFP4

    r = np.random.Generator(np.random.PCG64(17))
    n, k = 48, 128
    c, s = weights(r, n, k)
    qw, w64 = QWeightMXFP4(dev(c), dev(s)), dev(O.dequant_mxfp4(c, s))
    for m in (4, 80):
        x, x64 = activations(r, m, 2 * k, False)
        check(ops.qlinear(x[:, k:], qw), x64[:, k:], w64)
        check(ops.qlinear(x.view(2, m, k), qw).view(2 * m, n), x64.view(2 * m, k), w64)
        wide = QWeightMXFP4(dev(np.repeat(c, 2, 0))[::2], dev(np.repeat(s, 2, 0))[::2])  # strided weights
        check(ops.qlinear(x[:, :k], wide), x64[:, :k], w64)
        out = torch.full((m, n), 7.0, dtype=torch.bfloat16, device=DEV)
        assert ops.qgemm(x[:, :k].contiguous(), qw, out=out) is out
        check(out, x64[:, :k], w64)
    assert ops.qlinear(x[:0, :k], qw).shape == (0, n) and ops.qgemm(x[:0, :k], qw).dtype == torch.bfloat16
    assert ops.qlinear(x[:, :k], QWeightMXFP4(qw.packed[:0], qw.scale[:0])).shape == (80, 0)
    assert ops.qlinear(x[:5, :k], qw, out_dtype=torch.float16).dtype == torch.float16
    with pytest.raises(ValueError, match="bfloat16"):
        ops.qlinear(x[:, :k].float(), qw)
    with pytest.raises(ValueError, match="out must"):
        ops.qgemm(x[:, :k].contiguous(), qw, out=torch.empty(80, n, device=DEV))
    with pytest.raises(ValueError, match="aligned"):
        ops.qlinear(torch.zeros(1 + k, dtype=torch.bfloat16, device=DEV)[1:].view(1, k), qw)
    with pytest.raises(ValueError, match="must live on"):
        ops.qgemm(x[:, :k].contiguous(), qw, out=out.cpu())


# ---- products by group ---------------------------------------------------------------------------------------------------
def grouped_case(seed, counts, n, k, x4):
    from chadslab_amd import QExpertsMXFP4

    r = np.random.Generator(np.random.PCG64(seed))
    e, rows = len(counts), int(sum(counts))
    c, s = weights(r, e, n, k)
    x, x64 = activations(r, rows, k, x4)
    offsets = torch.tensor([0, *np.cumsum(counts)], dtype=torch.int32, device=DEV)
    return x, x64, QExpertsMXFP4(dev(c), dev(s)), dev(O.dequant_mxfp4(c, s)), offsets


def check_groups(y, x64, w64, bounds):
    for e in range(w64.shape[0]):
        if bounds[e + 1] > bounds[e]:
            check(y[bounds[e]:bounds[e + 1]], x64[bounds[e]:bounds[e + 1]], w64[e])


@pytest.mark.parametrize("x4", [False, True], ids=["bf16", "mxfp4"])
@pytest.mark.parametrize("counts,n,k", [([1], 40, 64), ([0, 3, 0, 0, 17, 1, 0], 130, 160), ([16, 16, 16], 64, 256), ([5, 0, 70, 33, 128, 1, 0, 2], 257, 288),
                                        ([1] * 70, 33, 96), ([0] * 130 + [9] + [0] * 69, 64, 128), ([300, 2, 0, 513], 200, 544), ([0, 700, 0, 0], 96, 2080)])
def test_grouped(ops, counts, n, k, x4):
    x, x64, w, w64, offsets = grouped_case(len(counts) * 31 + n, counts, n, k, x4)
    y = ops.qgemm_grouped(x, w, offsets)
    assert y.dtype == torch.bfloat16 and y.shape == (sum(counts), n)
    check_groups(y, x64, w64, offsets.tolist())


@pytest.mark.parametrize("x4", [False, True], ids=["bf16", "mxfp4"])
@pytest.mark.parametrize("rows", [40, 700])
def test_grouped_rows_of_no_group(ops, rows, x4):
    """In front of the first group and behind the last: 0 in a fresh result, left alone in a given one."""
    n, k = 72, 160
    x, x64, w, w64, _ = grouped_case(rows, [rows, 0, 0], n, k, x4)
    for bounds in ([3, 3, 9, rows - 4], [0, 0, 0, 0], [rows] * 4, [0, 1, 1, 1], [rows - 1, rows - 1, rows, rows], [0, 5, 5, rows]):
        offsets = torch.tensor(bounds, dtype=torch.int32, device=DEV)
        y = ops.qgemm_grouped(x, w, offsets)
        check_groups(y, x64, w64, bounds)
        assert not y[:bounds[0]].any() and not y[bounds[-1]:].any()
        out = torch.full((rows, n), 5.0, dtype=torch.bfloat16, device=DEV)
        assert ops.qgemm_grouped(x, w, offsets, out=out) is out
        assert torch.equal(out[bounds[0]:bounds[-1]], y[bounds[0]:bounds[-1]])
        assert bool((out[:bounds[0]] == 5).all()) and bool((out[bounds[-1]:] == 5).all())


@pytest.mark.parametrize("rows", [30, 500])
def test_grouped_offsets_out_of_order_lead_nowhere_else(ops, rows):
    """Clamped into the rows, a descending one counts as the largest before it."""
    n, k = 64, 96
    x, x64, w, w64, _ = grouped_case(rows, [rows, 0, 0, 0], n, k, False)
    for given, meant in (([-5, 4, 2, 9, 2 ** 31 - 1], [0, 4, 4, 9, rows]), ([rows + 7, 0, 0, 0, 0], [rows] * 5), ([2, -2 ** 31, 20, 10, 25], [2, 2, 20, 20, 25])):
        y = ops.qgemm_grouped(x, w, torch.tensor(given, dtype=torch.int32, device=DEV))
        check_groups(y, x64, w64, meant)
        assert not y[:meant[0]].any() and not y[meant[-1]:].any()


def test_grouped_refusals_and_empty(ops):
    x, _, w, _, offsets = grouped_case(1, [3, 2], 32, 64, False)
    assert ops.qgemm_grouped(x[:0], w, offsets).shape == (0, 32)
    for bad in (offsets[:2], offsets.to(torch.int64), offsets.view(1, 3)):
        with pytest.raises(ValueError, match="offsets must"):
            ops.qgemm_grouped(x, w, bad)
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.qgemm_grouped(x, w, offsets.cpu())
    with pytest.raises(ValueError, match="out must"):
        ops.qgemm_grouped(x, w, offsets, out=torch.empty(5, 31, dtype=torch.bfloat16, device=DEV))
    with pytest.raises(ValueError, match="bfloat16"):
        ops.qgemm_grouped(x.float(), w, offsets)


# ---- streams and graphs ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("m", [3, 48, 300])
def test_captured_products_replay(ops, m):
    """Two graphs of different products and eager work in between: every replay is the eager result of the inputs it finds."""
    from chadslab_amd import QWeightMXFP4

    r = np.random.Generator(np.random.PCG64(m))
    n, k = 512, 4096
    cases = []
    side = torch.cuda.Stream()
    for i in range(2):
        c, s = weights(r, n, k)
        qw = QWeightMXFP4(dev(c), dev(s))
        x, _ = activations(r, m, k, False)
        with torch.cuda.stream(side):
            ops.qlinear(ops.quantize_mxfp4(x), qw)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            y = ops.qlinear(x, qw), ops.qlinear(ops.quantize_mxfp4(x), qw)
        cases.append((g, x, qw, y))
    for turn in range(3):
        for g, x, qw, y in cases:
            x.copy_(activations(r, m, k, False)[0])
            want = ops.qlinear(x, qw), ops.qlinear(ops.quantize_mxfp4(x), qw)
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y[0], want[0]) and torch.equal(y[1], want[1])


def test_same_call_gives_the_same_bits_on_any_stream(ops):
    from chadslab_amd import QWeightMXFP4

    r = np.random.Generator(np.random.PCG64(2))
    c, s = weights(r, 600, 4096)
    qw = QWeightMXFP4(dev(c), dev(s))
    for m in (1, 16, 60, 260):
        x, _ = activations(r, m, 4096, False)
        want = ops.qlinear(x, qw)
        torch.cuda.synchronize()
        streams, got = [torch.cuda.Stream() for _ in range(3)], []
        for st in streams:
            with torch.cuda.stream(st):
                got += [ops.qlinear(x, qw) for _ in range(4)]
        torch.cuda.synchronize()
        assert all(torch.equal(g, want) for g in got)


# ---- together -------------------------------------------------------------------------------------------------------------
def test_weights_and_activations_quantised_and_multiplied(ops):
    """Load time and serving in a row: weights quantised on the GPU, activations quantised per call, both products."""
    r = np.random.Generator(np.random.PCG64(8))
    w, x = r.standard_normal((300, 512)).astype(np.float32) * 0.05, r.standard_normal((50, 512)).astype(np.float32)
    qw = ops.quantize_mxfp4(dev(w))
    w64 = dev(O.dequant_mxfp4(*O.quantize_mxfp4(w)))
    xb = dev(x).to(torch.bfloat16)
    check(ops.qlinear(xb, qw), xb.double(), w64)
    check(ops.qlinear(ops.quantize_mxfp4(xb), qw), dev(O.dequant_mxfp4(*O.quantize_mxfp4(xb.double().cpu().numpy()))), w64)


# ---- mixture of experts ---------------------------------------------------------------------------------------------------
def moe_oracle(x64, logits, gate, up, down, top_k, renorm):
    idx, w = O.moe_route(logits, top_k, renorm)
    y = np.zeros_like(x64)
    for t in range(len(x64)):
        for j in range(top_k):
            g, u = gate[idx[t, j]] @ x64[t], up[idx[t, j]] @ x64[t]
            y[t] += float(w[t, j]) * (down[idx[t, j]] @ (g / (1 + np.exp(-g)) * u))
    return y


@pytest.mark.parametrize("tokens,h,f,experts,top_k,renorm", [(1, 32, 64, 4, 2, True), (4, 256, 512, 8, 2, True), (7, 96, 160, 3, 3, False), (33, 288, 352, 16, 4, True),
                                                             (100, 512, 1056, 8, 2, False), (300, 256, 224, 5, 1, True), (64, 64, 32, 1, 1, True)])
def test_moe(ops, tokens, h, f, experts, top_k, renorm):
    """Against 64 bits without rounding in between: what is rounded is h, half a step of bf16 (2^-8), and the result; the errors of h are
    independent, so the norm of the result's error is at most 2^-8 (h) + 2^-8 (y) of its own and the fp32 sums' and weights' 2^-18."""
    from chadslab_amd import QExpertsMXFP4

    r = np.random.Generator(np.random.PCG64(tokens + h + f))
    mats = [weights(r, experts, *shape, spread=0.5) for shape in ((f, h), (f, h), (h, f))]
    x, x64 = activations(r, tokens, h, False)
    logits = r.standard_normal((tokens, experts)).astype(np.float32)
    if experts > 3:
        logits[:, 1] = -50.0  # nobody's choice, as long as there are enough others
        logits[0, 2] = logits[0, 0]
    triple = tuple(QExpertsMXFP4(dev(c), dev(s)) for c, s in mats)
    y = ops.moe_ffn(x, dev(logits), triple, top_k=top_k, renorm=renorm)
    want = moe_oracle(x64.cpu().numpy(), logits, *(O.dequant_mxfp4(c, s) for c, s in mats), top_k, renorm)
    assert y.dtype == torch.bfloat16 and O.rel_l2(y.double().cpu().numpy(), want) <= 2 * 2.0 ** -8 + 2.0 ** -18


def test_moe_is_its_parts_and_replays(ops):
    """The layer against its own operators in a row (route, sort, products by group, gate, down, weighted sum), eager and from a graph."""
    from chadslab_amd import QExpertsMXFP4

    r = np.random.Generator(np.random.PCG64(77))
    tokens, h, f, experts, top_k = 90, 256, 320, 8, 2
    gate, up, down = (QExpertsMXFP4(*(dev(a) for a in weights(r, experts, *shape))) for shape in ((f, h), (f, h), (h, f)))
    x, _ = activations(r, tokens, h, False)
    logits = dev(r.standard_normal((tokens, experts)).astype(np.float32))

    def parts():
        idx, w = ops.moe_route(logits, top_k)
        order = torch.sort(idx.flatten().long(), stable=True).indices
        offsets = torch.searchsorted(idx.flatten().long().sort().values, torch.arange(experts + 1, device=DEV)).to(torch.int32)
        xs = x[order // top_k]
        g, u = ops.qgemm_grouped(xs, gate, offsets).float(), ops.qgemm_grouped(xs, up, offsets).float()
        d = ops.qgemm_grouped((g * torch.sigmoid(g) * u).to(torch.bfloat16), down, offsets).float()
        y = torch.empty_like(d)
        y[order] = d
        return (y.view(tokens, top_k, h) * w[..., None]).sum(1)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.moe_ffn(x, logits, (gate, up, down), top_k=top_k)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y = ops.moe_ffn(x, logits, (gate, up, down), top_k=top_k)
    for turn in range(3):
        x.copy_(activations(r, tokens, h, False)[0])
        logits.copy_(torch.randn_like(logits))
        eager, want = ops.moe_ffn(x, logits, (gate, up, down), top_k=top_k), parts()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eager)
        # gate and up (half a step of bf16 each, silu's slope is at most 1.1), h and the result are rounded here, h and the result there
        assert float((eager.double() - want.double()).norm() / want.double().norm()) <= (1.1 + 1 + 2 * 2) * 2.0 ** -8


def test_moe_refusals(ops):
    from chadslab_amd import QExpertsMXFP4

    r = np.random.Generator(np.random.PCG64(1))
    gate, up, down = (QExpertsMXFP4(*(dev(a) for a in weights(r, 4, *shape))) for shape in ((64, 32), (64, 32), (32, 64)))
    x, z = torch.zeros(3, 32, dtype=torch.bfloat16, device=DEV), torch.zeros(3, 4, device=DEV)
    assert not ops.moe_ffn(x, z, (gate, up, down)).any()
    with pytest.raises(TypeError, match="triple"):
        ops.moe_ffn(x, z, (gate, up))
    with pytest.raises(ValueError, match="gate and up"):
        ops.moe_ffn(x, z, (gate, down, up))
    with pytest.raises(ValueError, match="logits"):
        ops.moe_ffn(x, z[:, :3], (gate, up, down))
    for bad in (0, 5):
        with pytest.raises(ValueError, match="unsupported"):
            ops.moe_ffn(x, z, (gate, up, down), top_k=bad)


# ---- sizes for which the rule takes each of the tiles, with K that ends inside a step -------------------------------------
@pytest.mark.parametrize("x4,m,n,k", [(False, 19, 32, 608), (False, 135, 3466, 576), (False, 2919, 139, 640), (False, 2798, 2060, 608), (False, 523, 3762, 576),
                                      (False, 1063, 2698, 576), (False, 803, 4884, 608), (False, 2340, 1553, 640), (True, 2864, 146, 640), (True, 2524, 1594, 608),
                                      (True, 18, 36, 608), (True, 331, 2753, 576), (True, 2887, 652, 704), (True, 2358, 1683, 608), (True, 1608, 1183, 608),
                                      (True, 2347, 1550, 608), (True, 2188, 3702, 608)])
def test_every_tile(ops, x4, m, n, k):
    from chadslab_amd import QWeightMXFP4

    r = np.random.Generator(np.random.PCG64(m + n))
    c, s = weights(r, n, k)
    x, x64 = activations(r, m, k, x4)
    check(ops.qlinear(x, QWeightMXFP4(dev(c), dev(s))), x64, dev(O.dequant_mxfp4(c, s)))


@pytest.mark.parametrize("x4,m,n,k,e", [(False, 17, 32, 608, 2), (False, 69, 4062, 800, 8), (False, 115, 1277, 640, 13), (False, 88, 3552, 608, 10), (False, 129, 1436, 800, 11),
                                        (False, 202, 4169, 640, 15), (False, 710, 4513, 800, 13), (False, 2827, 1386, 608, 2), (True, 17, 33, 672, 2), (True, 67, 2089, 576, 8),
                                        (True, 113, 2567, 608, 14), (True, 348, 4184, 736, 15), (True, 18, 36, 2176, 2), (True, 1958, 3084, 576, 11), (True, 245, 4573, 1568, 7),
                                        (True, 209, 4216, 1056, 15), (True, 79, 3988, 928, 8)])
def test_every_tile_by_group(ops, x4, m, n, k, e):
    """Groups of any sizes, the first one empty."""
    r = np.random.Generator(np.random.PCG64(m * 3 + n))
    counts = [0, *r.multinomial(m, r.dirichlet(np.ones(e - 1)))]
    x, x64, w, w64, offsets = grouped_case(m + n + k, counts, n, k, x4)
    check_groups(ops.qgemm_grouped(x, w, offsets), x64, w64, offsets.tolist())


@pytest.mark.parametrize("tokens,h,f,experts", [(19, 1568, 64, 2), (22, 704, 32, 2), (92, 576, 1824, 11), (200, 672, 2080, 15), (303, 640, 2848, 11)])
def test_every_tile_of_gate_and_up(ops, tokens, h, f, experts):
    test_moe(ops, tokens, h, f, experts, 1, False)


# ---- the ends of the ranges ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("m", [1, 12, 40, 300])
def test_subnormal_activations_and_weights(ops, m):
    """bf16's subnormal numbers, as activations and as weights times their scale, count: 2^-130 against 2^100 is 2^-30."""
    from chadslab_amd import QWeightMXFP4

    r = np.random.Generator(np.random.PCG64(m + 3))
    n, k = 40, 256
    c, _ = weights(r, n, k)
    w64 = dev(O.dequant_mxfp4(c, np.full((n, k // 32), 127, np.uint8)))
    x = r.integers(-8, 9, (m, k)).astype(np.float64)
    for xe, we in ((-133, 227), (100, 0), (100, 2), (-120, 230)):
        xt = torch.from_numpy(x * 2.0 ** xe).to(torch.bfloat16).to(DEV)
        y = ops.qlinear(xt, QWeightMXFP4(dev(c), torch.full((n, k // 32), we, dtype=torch.uint8, device=DEV)))
        check((y.double() * 2.0 ** (127 - we - xe)).to(y.dtype), dev(x), w64)  # (of y's own type: the bound counts its rounding)


@pytest.mark.parametrize("x4", [False, True], ids=["bf16", "mxfp4"])
@pytest.mark.parametrize("m,n,k", [(1, 1, 32), (16, 1, 4096), (17, 1, 96), (500, 1, 352), (3, 5, 20000), (33, 3, 20000), (20000, 2, 64), (1, 70000, 32), (40, 70000, 32)])
def test_thin_products(ops, m, n, k, x4):
    from chadslab_amd import QWeightMXFP4

    r = np.random.Generator(np.random.PCG64(m + n + k))
    c, s = weights(r, n, k)
    x, x64 = activations(r, m, k, x4)
    check(ops.qlinear(x, QWeightMXFP4(dev(c), dev(s))), x64, dev(O.dequant_mxfp4(c, s)))


@pytest.mark.parametrize("m", [2, 48, 300])
def test_scales_at_any_address(ops, m):
    """Scales are bytes and may begin anywhere; codes want 16 bytes' alignment and are refused without."""
    from chadslab_amd import QWeightMXFP4

    r = np.random.Generator(np.random.PCG64(m))
    n, k = 100, 1056
    c, s = weights(r, n, k)
    x, x64 = activations(r, m, k, False)
    for shift in (1, 2, 7):
        buf = torch.zeros(n * k // 32 + shift, dtype=torch.uint8, device=DEV)
        buf[shift:] = dev(s).flatten()
        check(ops.qlinear(x, QWeightMXFP4(dev(c), buf[shift:].view(n, k // 32))), x64, dev(O.dequant_mxfp4(c, s)))
    codes = torch.zeros(n * k // 2 + 8, dtype=torch.uint8, device=DEV)[8:].view(n, k // 2)
    with pytest.raises(ValueError, match="aligned"):
        ops.qlinear(x, QWeightMXFP4(codes, dev(s)))


def test_without_the_host_module(ops, monkeypatch):
    """The Python road to the same kernels: the same bits."""
    from chadslab_amd import QExpertsMXFP4, QWeightMXFP4, _lib

    r = np.random.Generator(np.random.PCG64(5))
    c, s = weights(r, 4, 128, 256)
    qw, qe = QWeightMXFP4(dev(c[0]), dev(s[0])), QExpertsMXFP4(dev(c), dev(s))
    down = QExpertsMXFP4(*(dev(a) for a in weights(r, 4, 256, 128)))
    x, _ = activations(r, 40, 256, False)
    z, offsets = dev(r.standard_normal((40, 4)).astype(np.float32)), torch.tensor([0, 7, 7, 30, 40], dtype=torch.int32, device=DEV)

    def calls():
        q = ops.quantize_mxfp4(x)
        e = ops.quantize_mxfp4(x.float().view(2, 20, 256))
        assert type(q) is QWeightMXFP4 and type(e) is QExpertsMXFP4 and repr(q) and (q.N, q.K, e.E) == (40, 256, 2)
        return [q.packed, q.scale, e.packed, e.scale, ops.dequantize(q), ops.dequantize(e), ops.qlinear(x, qw), ops.qlinear(x[:3], qw), ops.qlinear(q, qw),
                ops.qlinear(x[:3], qw, out_dtype=torch.bfloat16), ops.qgemm_grouped(x, qe, offsets), ops.qgemm_grouped(q, qe, offsets), ops.moe_ffn(x, z, (qe, qe, down))]

    native = calls()
    monkeypatch.setattr(_lib, "_native", _lib._NoHostModule)
    for a, b in zip(native, calls()):
        assert a.dtype == b.dtype and torch.equal(a, b)


@pytest.mark.parametrize("rows,x4", [(30, False), (400, False), (400, True)])
def test_captured_groups_follow_their_offsets(ops, rows, x4):
    """A captured product by group reads the offsets of the replay, not those of the capture."""
    n, k = 96, 288
    x, x64, w, w64, offsets = grouped_case(rows, [rows // 4] * 4, n, k, x4)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.qgemm_grouped(x, w, offsets)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        y = ops.qgemm_grouped(x, w, offsets)
    rows = x64.shape[0]
    for bounds in ([0, 0, 0, 0, rows], [2, 9, 9, rows - 1, rows - 1], [0, 5, rows // 2, rows, rows], [0, rows // 4, rows // 2, rows - 3, rows]):
        offsets.copy_(torch.tensor(bounds, dtype=torch.int32))
        eager = ops.qgemm_grouped(x, w, offsets)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eager)
        check_groups(y, x64, w64, bounds)
        assert not y[:bounds[0]].any() and not y[bounds[-1]:].any()


@pytest.mark.parametrize("m,n,k", [(48, 512, 8192), (100, 2048, 8192), (20, 130, 14368), (300, 256, 14336)])
def test_products_in_parts_of_k(ops, m, n, k):
    """Few tiles and a long K: summed in parts, by the C entry point with its workspace and without, and with one too small."""
    from chadslab_amd import QWeightMXFP4, _lib

    lib = _lib.load()
    need = lib.chadq_product_mxfp4_workspace_bytes(m, n, k, 0)
    assert need > 0 and need % (4 * m * n) == 0
    r = np.random.Generator(np.random.PCG64(m))
    c, s = weights(r, n, k)
    qw, w64 = QWeightMXFP4(dev(c), dev(s)), dev(O.dequant_mxfp4(c, s))
    x, x64 = activations(r, m, k, False)
    check(ops.qlinear(x, qw), x64, w64)
    for size in (0, need - 1, need):
        ws = torch.full((need,), 255, dtype=torch.uint8, device=DEV)
        for dtype in (torch.float32, torch.bfloat16):
            y = torch.full((m, n), float("nan"), dtype=dtype, device=DEV)
            rc = lib.chadq_product_mxfp4(x.data_ptr(), None, qw.packed.data_ptr(), qw.scale.data_ptr(), y.data_ptr(), int(dtype == torch.bfloat16), m, n, k, ws.data_ptr() if size else None,
                                         size, torch.cuda.current_stream().cuda_stream)
            assert rc == 0
            check(y, x64, w64)


def test_library_refuses(ops):
    """The C entry points' own checks: status and message, no launch."""
    from chadslab_amd import _lib

    lib = _lib.load()
    a = torch.zeros(4096, dtype=torch.uint8, device=DEV).data_ptr()
    for call, status in (((a, None, a, a, a, 0, 1, 1, 48, None, 0, None), -2), ((a, None, a, a, a, 0, -1, 1, 32, None, 0, None), -2), ((a, None, a, a, a, 0, 1, 1, 2 ** 26 + 32, None, 0, None), -2),
                         ((None, None, a, a, a, 0, 1, 1, 32, None, 0, None), -1), ((a, None, a, None, a, 0, 1, 1, 32, None, 0, None), -1), ((a + 8, None, a, a, a, 0, 1, 1, 32, None, 0, None), -3),
                         ((a, None, a + 4, a, a, 0, 1, 1, 32, None, 0, None), -3), ((a, None, a, a, a, 0, 20, 1, 32, a + 4, 64, None), -3), ((a, None, a, a, a, 0, 2 ** 31 - 1, 2 ** 31 - 1, 32, None, 0, None), -2)):
        assert lib.chadq_product_mxfp4(*call) == status, call
    assert lib.chadq_product_mxfp4(None, None, None, None, None, 0, 0, 5, 32, None, 0, None) == 0
    for call, status in (((a, None, a, a, a, a, 4, 0, 1, 32, 1, None), -2), ((a, None, a, a, None, a, 4, 1, 1, 32, 1, None), -1), ((a, None, a, a, a + 2, a, 4, 1, 1, 32, 1, None), -3),
                         ((a, None, a, a, a, a, 4, 1, 1, 33, 1, None), -2)):
        assert lib.chadq_product_mxfp4_grouped(*call) == status, call
    for call, status in (((a, 3, a, a, 1, 32, None), -2), ((a, 0, a, a, 1, 33, None), -2), ((a, 0, a, a, -1, 32, None), -2), ((a, 0, None, a, 1, 32, None), -1), ((a + 4, 0, a, a, 1, 32, None), -3),
                         ((a, 0, a + 1, a, 1, 32, None), -3), ((a, 0, a, a, 2 ** 62, 32, None), -2)):
        assert lib.chadq_quantize_mxfp4(*call) == status, call
    assert lib.chadq_dequant_mxfp4(a, a, a + 4, 1, 32, None) == -3 and lib.chadq_dequant_mxfp4(a, a, a, 1, 31, None) == -2
    assert lib.chadq_moe_ffn_mxfp4_workspace_bytes(4, 64, 64, 17, 2) == 0 and lib.chadq_moe_ffn_mxfp4_workspace_bytes(4, 64, 48, 4, 2) == 0
    assert lib.chadq_moe_ffn_mxfp4_workspace_bytes(4, 64, 64, 4, 2) > 0
