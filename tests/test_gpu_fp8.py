"""FP8 by blocks of 128 on the GPU, through chadslab_amd.ops, against the oracle in 64 bits.  Quantisation and its inverse bit for bit.

Products.  bf16 x e4m3 and e4m3 x e4m3 are exact in fp32; what is off is the sums and the scales.  With S = sum_k |x w scales| of an
element: inside a block of 128 an fp32 addition is off by at most 2^-24 of the block's own S, and a matrix instruction adds 32 to 128
products and its operand C in at most 4 roundings' worth, so a block takes at most 128/16 * 4 = 32 of them; the scales' product and its
FMA are two more; the G = ceil(K/128) blocks are joined by G additions, and at most 64 partial sums:
|y - exact| <= (32 + 2 + G + 64) 2^-24 S;  a result in bf16 adds half a step, 2^-8 |y|.

8-bit activations of more rows than are streamed (16, or 8 of a group on average; results in bf16) meet the 8-bit matrix instruction, which adds the products of
eight k as multiples of 2^-13 of the power of two that is the largest one's exponents' sum, cutting off what lies below (measured with one large product of
either sign beside a small one: all its forms alike).  The largest is exact; the other seven are each off by less than 2^-13 of it, so eight products by less than
7 * 2^-13 times their own S, and so is the sum of all: `cut` adds 7 * 2^-13 S.  Values of the four binades from 1 to 15 (`narrow`) are exact there
too: their products are multiples of 2^-6, and the largest exponents' sum is 6, so that multiples of 2^-7 are kept: these are held to the tight bound."""
import numpy as np
import pytest
import torch

from oracle import chadq_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FP8 = torch.float8_e4m3fn
KINDS = pytest.mark.parametrize("x8", [False, True], ids=["bf16", "fp8"])


@pytest.fixture(scope="module")
def ops():
    from chadslab_amd import _lib, ops as _ops

    assert torch.cuda.is_available(), "these tests need the GPU"
    _lib.load()
    return _ops


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def blocks(n):
    return -(-n // 128)


def values(r, *shape):
    """Any finite values of 8 bits, small ones and zeros among them."""
    b = r.integers(0, 127, shape, dtype=np.uint8)
    return dev(b | (r.integers(0, 2, shape, dtype=np.uint8) << 7)).view(FP8)


def narrow(r, *shape):
    """Values from 1 to 15 and 0, of either sign."""
    b = r.integers(0x38, 0x38 + 32, shape, dtype=np.uint8)
    b[r.random(shape) < 0.1] = 0
    return dev(b | (r.integers(0, 2, shape, dtype=np.uint8) << 7)).view(FP8)


def scales(r, *shape):
    return dev(np.exp(r.standard_normal(shape) - 7).astype(np.float32))


def weights(r, n, k, experts=None, values=values):
    from chadslab_amd import QExpertsFP8, QWeightFP8

    if experts is None:
        return QWeightFP8(values(r, n, k), scales(r, blocks(n), blocks(k)))
    return QExpertsFP8(values(r, experts, n, k), scales(r, experts, blocks(n), blocks(k)))


def w64(q):
    """float64 of a matrix or, [E,N,K], of experts."""
    *_, n, k = q.w.shape
    s = q.scale.double().repeat_interleave(128, -1)[..., :k].repeat_interleave(128, -2)[..., :n, :]
    return q.w.double() * s


def x64(x):
    return x.double() if isinstance(x, torch.Tensor) else x.w.double() * x.scale.double().repeat_interleave(128, -1)[:, :x.K]


def activations(r, m, k, x8, values=values):
    from chadslab_amd import QRowsFP8

    if x8:
        return QRowsFP8(values(r, m, k), scales(r, m, blocks(k)))
    return dev(r.standard_normal((m, k)).astype(np.float32)).to(torch.bfloat16)


def rows_of(x, index):
    from chadslab_amd import QRowsFP8

    return x[index] if isinstance(x, torch.Tensor) else QRowsFP8(x.w.view(torch.uint8)[index].view(FP8), x.scale[index])


def check(y, a, b, cut=False):
    """Element by element, with the bound above; a [M,K], b [N,K] in 64 bits."""
    exact, s = a @ b.T, a.abs() @ b.abs().T
    bound = (98 + blocks(a.shape[1])) * 2.0 ** -24 * s + 2.0 ** -126
    if y.dtype == torch.bfloat16:
        bound = bound + 2.0 ** -8 * exact.abs()
    if cut and y.dtype == torch.bfloat16:
        bound = bound + 7 * 2.0 ** -13 * s
    off = (y.double() - exact).abs()
    assert torch.isfinite(y).all() and bool((off <= bound).all()), "off by %.3g bounds" % float((off / bound).max())


# ---- quantisation ---------------------------------------------------------------------------------------------------------
def check_quantised(ops, x, rows):
    q = ops.quantize_fp8(x, rows=rows)
    flat = x.float().cpu().numpy()
    if x.dim() == 2:
        b, s = O.quantize_fp8(flat, 1 if rows else 128)
    else:
        b, s = (np.stack(v) for v in zip(*(O.quantize_fp8(m, 128) for m in flat)))
    assert np.array_equal(q.w.view(torch.uint8).cpu().numpy(), b) and np.array_equal(q.scale.cpu().numpy(), s, equal_nan=True)
    back = ops.dequantize(q)
    with np.errstate(invalid="ignore", over="ignore"):
        want = (q.w.float() * q.scale.repeat_interleave(128, -1)[..., :x.size(-1)] if rows else
                q.w.float() * q.scale.repeat_interleave(128, -1)[..., :x.size(-1)].repeat_interleave(128, -2)[..., :x.size(-2), :])
    assert back.dtype == torch.float32 and torch.equal(torch.nan_to_num(back, nan=7e9), torch.nan_to_num(want, nan=7e9))
    return q


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [True, False])
@pytest.mark.parametrize("n,k", [(1, 16), (3, 144), (127, 128), (130, 272), (300, 4096), (1025, 48), (129, 16400)])
def test_quantize_is_the_oracles(ops, n, k, rows, dtype):
    r = np.random.Generator(np.random.PCG64(n + k))
    x = r.standard_normal((n, k)) * np.exp(r.standard_normal((n, 1)) * 2)
    x[r.random((n, k)) < 0.1] = 0.0
    check_quantised(ops, torch.from_numpy(x).to(dtype).to(DEV), rows)


@pytest.mark.parametrize("rows", [True, False])
def test_quantize_every_border(ops, rows):
    """The largest of every block is 448, so that the factor is 1: every value, every middle between two and its neighbours."""
    v = O.e4m3_values()[:127].astype(np.float32)
    mid = (v[1:] + v[:-1]) / 2
    x = np.concatenate([v, mid, np.nextafter(mid, np.float32(0)), np.nextafter(mid, np.float32(1000))])
    x = np.concatenate([x, -x])
    x = np.pad(x, (0, -len(x) % 127)).reshape(-1, 127)
    check_quantised(ops, dev(np.concatenate([np.full((len(x), 1), 448, np.float32), x], 1)), rows)


@pytest.mark.parametrize("rows", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_quantize_extremes(ops, dtype, rows):
    info = torch.finfo(dtype)
    tiny = float(torch.tensor(info.smallest_normal * info.eps, dtype=dtype))
    x = np.zeros((1024, 256))
    for i, (a, b) in enumerate(((np.nan, 1.0), (np.inf, -2.0), (-np.inf, 0.3), (info.max, -info.max), (tiny, info.smallest_normal), (-0.0, -0.0), (1e-3, 7.0))):
        x[i * 128 + 3, 5], x[i * 128 + 3, 200] = a, b
        x[i * 128 + 4, 6], x[i * 128 + 4, 201] = b, a
    check_quantised(ops, torch.from_numpy(x).to(dtype).to(DEV), rows)


def test_quantize_views_experts_and_nothing(ops):
    r = np.random.Generator(np.random.PCG64(3))
    x = dev(r.standard_normal((4, 140, 272)).astype(np.float32))
    assert check_quantised(ops, x, False).E == 4
    assert check_quantised(ops, x.transpose(0, 1)[:, :, 16:160], False).E == 140
    check_quantised(ops, x[1, ::3, :256:2], True)
    assert ops.quantize_fp8(x[0, :0]).M == 0 and ops.quantize_fp8(x[:0], rows=False).E == 0 and ops.quantize_fp8(x[0, :, :0]).K == 0
    assert ops.dequantize(ops.quantize_fp8(x[0, :0])).shape == (0, 272)
    with pytest.raises(ValueError, match="aligned"):
        ops.quantize_fp8(torch.zeros(1 + 64, device=DEV)[1:].view(2, 32))


def test_dequantize_every_byte(ops):
    from chadslab_amd import QRowsFP8

    w = torch.arange(256, dtype=torch.uint8, device=DEV).repeat(9, 1)
    s = torch.tensor([1.0, 2.0 ** -126, 2.0 ** -140, 2.0 ** 119, 3.3e38, float("inf"), float("nan"), 0.0, 0.7], device=DEV)[:, None].repeat(1, 2)
    got, want = ops.dequantize(QRowsFP8(w.view(FP8), s)), w.view(FP8).float() * s[:, :1]
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.nan_to_num(got, nan=0.0), torch.nan_to_num(want, nan=0.0))


# ---- products -------------------------------------------------------------------------------------------------------------
MS = [1, 2, 3, 5, 8, 9, 16, 17, 31, 33, 48, 64, 65, 100, 129, 200, 257]
NKS = [(1, 16), (16, 128), (33, 144), (250, 80), (129, 2064), (130, 4096), (515, 528), (96, 7216)]


@KINDS
@pytest.mark.parametrize("n,k", NKS)
def test_products(ops, n, k, x8):
    r = np.random.Generator(np.random.PCG64(n * 10007 + k))
    qw = weights(r, n, k)
    b = w64(qw)
    for m in MS:
        x = activations(r, m, k, x8)
        a = x64(x)
        y = ops.qlinear(x, qw)
        assert y.shape == (m, n) and y.dtype == (torch.float32 if m <= 16 else torch.bfloat16)
        check(y, a, b, x8)
        if m <= 16:
            check(ops.qgemv(x, qw), a, b)
            yb = ops.qlinear(x, qw, out_dtype=torch.bfloat16)
            assert yb.dtype == torch.bfloat16 and torch.equal(yb, y.to(torch.bfloat16))  # the same sums, rounded once
        y = ops.qgemm(x, qw)
        assert y.dtype == torch.bfloat16
        check(y, a, b, x8 and m > 16)


@KINDS
@pytest.mark.parametrize("m,n,k", [(1, 14336, 4096), (16, 1000, 14352), (40, 4100, 1040), (300, 2064, 1168), (512, 4096, 4096), (1030, 777, 2048), (2050, 520, 336)])
def test_larger_products(ops, m, n, k, x8):
    r = np.random.Generator(np.random.PCG64(m + n + k))
    qw, x = weights(r, n, k), activations(r, m, k, x8)
    check(ops.qlinear(x, qw), x64(x), w64(qw), x8)


@KINDS
@pytest.mark.parametrize("n,k", [(1, 16), (33, 144), (250, 80), (129, 2064), (260, 4096), (515, 528)])
def test_products_of_narrow_values(ops, n, k, x8):
    r = np.random.Generator(np.random.PCG64(n * 10007 + k))
    qw = weights(r, n, k, values=narrow)
    b = w64(qw)
    for m in MS + [300, 515]:
        x = activations(r, m, k, x8, values=narrow)
        check(ops.qgemm(x, qw), x64(x), b)


@KINDS
@pytest.mark.parametrize("counts,n,k", [([0, 3, 0, 0, 17, 1, 0], 130, 144), ([5, 0, 70, 33, 128, 1, 0, 2], 257, 272), ([300, 2, 0, 513], 200, 528), ([0, 700, 0, 0], 96, 2064)])
def test_groups_of_narrow_values(ops, counts, n, k, x8):
    r = np.random.Generator(np.random.PCG64(n))
    w, x = weights(r, n, k, len(counts), values=narrow), activations(r, sum(counts), k, x8, values=narrow)
    bounds = [0, *np.cumsum(counts)]
    check_groups(ops.qgemm_grouped(x, w, torch.tensor(bounds, dtype=torch.int32, device=DEV)), x, w, bounds, cut=False)


@KINDS
@pytest.mark.parametrize("m", [1, 7, 40, 200])
def test_integer_products_are_exact(ops, m, x8):
    """Small integers and powers of two for scales: every partial sum is exact, so any order gives the same."""
    from chadslab_amd import QRowsFP8, QWeightFP8

    r = np.random.Generator(np.random.PCG64(m))
    n, k = 300, 528
    w, x = (dev(r.integers(-8, 9, s).astype(np.float32)) for s in ((n, k), (m, k)))
    ws, xs = (dev(np.exp2(r.integers(0, 3, s)).astype(np.float32)) for s in ((3, 5), (m, 5)))
    qw = QWeightFP8(w.to(FP8), ws)
    xq = QRowsFP8(x.to(FP8), xs) if x8 else x.to(torch.bfloat16)
    y = ops.qgemv(xq, qw) if m <= 16 else ops.qgemm(xq, qw)
    assert torch.equal(y, (x64(xq) @ w64(qw).T).to(y.dtype))


@KINDS
@pytest.mark.parametrize("m", [2, 40, 200])
def test_nan_stays_in_its_row_and_column(ops, m, x8):
    """NaN values and scales; K ends inside a block: what lies behind it must not leak in."""
    r = np.random.Generator(np.random.PCG64(m + 1))
    n, k = 270, 208
    qw, x = weights(r, n, k), activations(r, m, k, x8)
    qw.w.view(torch.uint8)[3, 207], qw.w.view(torch.uint8)[50, 0] = 0x7F, 0xFF
    qw.scale[1, 1] = float("nan")
    if x8:
        x.scale[1, 0] = float("nan")
    else:
        x[1, 65] = float("nan")
    y = ops.qlinear(x, qw)
    want = torch.zeros(m, n, dtype=torch.bool, device=DEV)
    want[1], want[:, 3], want[:, 50], want[:, 128:256] = True, True, True, True
    assert torch.equal(torch.isnan(y), want)
    keep_m, keep_n = [i for i in range(m) if i != 1], [i for i in range(n) if i not in (3, 50) and not 128 <= i < 256]
    check(y[keep_m][:, keep_n], x64(rows_of(x, keep_m)), w64(qw)[keep_n], x8)


@pytest.mark.parametrize("m", [2, 40, 200])
def test_infinite_activations(ops, m):
    """As IEEE has it: infinity times a weight that is 0 is NaN, else infinite."""
    from chadslab_amd import QWeightFP8

    w = torch.zeros(3, 48, device=DEV)
    w[0, 0], w[1, 0] = 1, -1
    x = torch.zeros(m, 48, dtype=torch.bfloat16, device=DEV)
    x[1, 0] = float("inf")
    y = ops.qlinear(x, QWeightFP8(w.to(FP8), torch.ones(1, 1, device=DEV)))
    assert y[1, 0] == float("inf") and y[1, 1] == -float("inf") and torch.isnan(y[1, 2]) and bool((y[0] == 0).all())


@KINDS
@pytest.mark.parametrize("k", [16, 80, 144, 272, 2064])
@pytest.mark.parametrize("m", [1, 3, 16, 40])
def test_infinite_scales_of_the_last_block(ops, m, k, x8):
    """An infinite scale makes its sums infinite, not NaN: zeros behind the row's end may not meet it."""
    from chadslab_amd import QExpertsFP8

    e = QExpertsFP8(torch.ones(2, 140, k, device=DEV).to(FP8), torch.ones(2, 2, blocks(k), device=DEV))
    e.scale[0, 1, -1] = e.scale[1, 0, -1] = float("inf")
    x = torch.ones(m, k, dtype=torch.bfloat16, device=DEV)
    x = ops.quantize_fp8(x) if x8 else x
    want = torch.full((2, m, 140), float(k), device=DEV)
    want[0, :, 128:] = want[1, :, :128] = float("inf")
    for i in range(2):
        assert torch.equal(ops.qlinear(x, e.expert(i)).float(), want[i])
    half = m // 2
    y = ops.qgemm_grouped(x, e, torch.tensor([0, half, m], dtype=torch.int32, device=DEV))
    assert torch.equal(y, torch.cat((want[0, :half], want[1, half:])).to(torch.bfloat16))


@KINDS
@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (16, 1, 4096), (17, 1, 80), (500, 1, 336), (3, 5, 20000), (33, 3, 20000), (20000, 2, 64), (1, 70000, 32), (40, 70000, 32)])
def test_thin_products(ops, m, n, k, x8):
    r = np.random.Generator(np.random.PCG64(m + n + k))
    qw, x = weights(r, n, k), activations(r, m, k, x8)
    check(ops.qlinear(x, qw), x64(x), w64(qw), x8)


def test_strides_outputs_and_refusals(ops):
    from chadslab_amd import QRowsFP8, QWeightFP8

    r = np.random.Generator(np.random.PCG64(17))
    n, k = 48, 128
    qw = weights(r, n, k)
    b = w64(qw)
    for m in (4, 80):
        x = activations(r, m, 2 * k, False)
        check(ops.qlinear(x[:, k:], qw), x64(x)[:, k:], b)
        check(ops.qlinear(x.view(2, m, k), qw).view(2 * m, n), x64(x).view(2 * m, k), b)
        wide = QWeightFP8(qw.w.repeat(1, 2)[:, :k], qw.scale)  # strided weights
        check(ops.qlinear(x[:, :k], wide), x64(x)[:, :k], b)
        xq = activations(r, m, 2 * k, True)
        part = QRowsFP8(xq.w[:, k:], xq.scale[:, 1:])
        check(ops.qlinear(part, qw), x64(part), b, True)
        out = torch.full((m, n), 7.0, dtype=torch.bfloat16, device=DEV)
        assert ops.qgemm(x[:, :k].contiguous(), qw, out=out) is out
        check(out, x64(x)[:, :k], b)
    assert ops.qlinear(x[:0, :k], qw).shape == (0, n) and ops.qgemm(x[:0, :k], qw).dtype == torch.bfloat16
    assert ops.qlinear(x[:, :k], QWeightFP8(qw.w[:0], qw.scale[:0])).shape == (80, 0)
    assert not ops.qlinear(x[:, :0], QWeightFP8(qw.w[:, :0], qw.scale[:, :0])).any()
    assert ops.qlinear(x[:5, :k], qw, out_dtype=torch.float16).dtype == torch.float16
    for call, match in ((lambda: ops.qlinear(x[:, :k].float(), qw), "bfloat16"), (lambda: ops.qgemm(x[:, :k].contiguous(), qw, out=torch.empty(80, n, device=DEV)), "out must"),
                        (lambda: ops.qlinear(torch.zeros(1 + k, dtype=torch.bfloat16, device=DEV)[1:].view(1, k), qw), "aligned"),
                        (lambda: ops.qgemm(x[:, :k].contiguous(), qw, out=out.cpu()), "must live on"), (lambda: ops.qlinear(x[:, :64], qw), r"\[M,128\]"),
                        (lambda: ops.qgemv(x[:, :k], qw), "at most 16"), (lambda: ops.qlinear(x[:, :k], qw.to("cpu")), "GPU tensor")):
        with pytest.raises(ValueError, match=match):
            call()
    qw.scale = qw.scale[:, :0]  # exchanged after construction
    with pytest.raises(ValueError, match="scale must"):
        ops.qlinear(x[:, :k], qw)


# ---- products by group ----------------------------------------------------------------------------------------------------
def grouped_case(seed, counts, n, k, x8):
    r = np.random.Generator(np.random.PCG64(seed))
    w = weights(r, n, k, len(counts))
    return activations(r, int(sum(counts)), k, x8), w, torch.tensor([0, *np.cumsum(counts)], dtype=torch.int32, device=DEV)


def check_groups(y, x, w, bounds, cut=True):
    cut = cut and not isinstance(x, torch.Tensor)
    a, b = x64(x), w64(w)
    for e in range(w.E):
        if bounds[e + 1] > bounds[e]:
            check(y[bounds[e]:bounds[e + 1]], a[bounds[e]:bounds[e + 1]], b[e], cut and len(a) > 8 * w.E)


@KINDS
@pytest.mark.parametrize("counts,n,k", [([1], 40, 64), ([0, 3, 0, 0, 17, 1, 0], 130, 144), ([16, 16, 16], 64, 256), ([5, 0, 70, 33, 128, 1, 0, 2], 257, 272),
                                        ([1] * 70, 33, 80), ([0] * 130 + [9] + [0] * 69, 64, 128), ([300, 2, 0, 513], 200, 528), ([0, 700, 0, 0], 96, 2064)])
def test_grouped(ops, counts, n, k, x8):
    x, w, offsets = grouped_case(len(counts) * 31 + n, counts, n, k, x8)
    y = ops.qgemm_grouped(x, w, offsets)
    assert y.dtype == torch.bfloat16 and y.shape == (sum(counts), n)
    check_groups(y, x, w, offsets.tolist())


@KINDS
@pytest.mark.parametrize("rows", [40, 700])
def test_grouped_rows_of_no_group(ops, rows, x8):
    """In front of the first group and behind the last: 0 in a fresh result, left alone in a given one.  Offsets are clamped into the rows, a descending one
    counts as the largest before it."""
    n, k = 136, 144
    x, w, _ = grouped_case(rows, [rows, 0, 0], n, k, x8)
    for given, meant in (([3, 3, 9, rows - 4], None), ([0, 0, 0, 0], None), ([rows] * 4, None), ([0, 1, 1, 1], None), ([rows - 1, rows - 1, rows, rows], None), ([0, 5, 5, rows], None),
                         ([-5, 4, 2, 2 ** 31 - 1], [0, 4, 4, rows]), ([rows + 7, 0, 0, 0], [rows] * 4), ([2, -2 ** 31, 20, 10], [2, 2, 20, 20])):
        bounds, offsets = meant or given, torch.tensor(given, dtype=torch.int32, device=DEV)
        y = ops.qgemm_grouped(x, w, offsets)
        check_groups(y, x, w, bounds)
        assert not y[:bounds[0]].any() and not y[bounds[-1]:].any()
        out = torch.full((rows, n), 5.0, dtype=torch.bfloat16, device=DEV)
        assert ops.qgemm_grouped(x, w, offsets, out=out) is out
        assert torch.equal(out[bounds[0]:bounds[-1]], y[bounds[0]:bounds[-1]])
        assert bool((out[:bounds[0]] == 5).all()) and bool((out[bounds[-1]:] == 5).all())


def test_grouped_refusals_and_empty(ops):
    x, w, offsets = grouped_case(1, [3, 2], 32, 64, False)
    assert ops.qgemm_grouped(x[:0], w, offsets).shape == (0, 32)
    for bad in (offsets[:2], offsets.to(torch.int64), offsets.view(1, 3)):
        with pytest.raises(ValueError, match="offsets must"):
            ops.qgemm_grouped(x, w, bad)
    for call, match in ((lambda: ops.qgemm_grouped(x, w, offsets.cpu()), "GPU tensor"), (lambda: ops.qgemm_grouped(x.float(), w, offsets), "bfloat16"),
                        (lambda: ops.qgemm_grouped(x, w, offsets, out=torch.empty(5, 31, dtype=torch.bfloat16, device=DEV)), "out must"),
                        (lambda: ops.qgemm_grouped(x[:, :48], w, offsets), r"\[R,64\]")):
        with pytest.raises(ValueError, match=match):
            call()


# ---- mixture of experts ---------------------------------------------------------------------------------------------------
def moe_oracle(ops, x, logits, triple, how):
    """In 64 bits, h to 8 bits where x is: by the oracle's own quantiser."""
    gate, up, down = (w64(w).cpu().numpy() for w in triple)
    idx, w = O.moe_route_experts(logits, **how)
    a = x64(x).cpu().numpy()
    y = np.zeros_like(a)
    for t in range(len(a)):
        for j in range(idx.shape[1]):
            g, u = gate[idx[t, j]] @ a[t], up[idx[t, j]] @ a[t]
            h = g / (1 + np.exp(-g)) * u
            if not isinstance(x, torch.Tensor):
                h = O.dequant_fp8(*O.quantize_fp8(h[None], 1), 1)[0]
            y[t] += float(w[t, j]) * (down[idx[t, j]] @ h)
    return y


GROUPED = dict(score="sigmoid", groups=4, top_groups=2, group_sum=2, scale=2.5)


@KINDS
@pytest.mark.parametrize("tokens,h,f,experts,how", [(1, 16, 64, 4, dict(top_k=2)), (4, 256, 512, 8, dict(top_k=2)), (7, 96, 176, 3, dict(top_k=3, renorm=False)),
                                                    (33, 272, 352, 16, dict(top_k=4, **GROUPED)), (100, 512, 1040, 8, dict(top_k=2, renorm=False)),
                                                    (300, 256, 224, 5, dict(top_k=1)), (64, 64, 16, 1, dict(top_k=1)), (50, 128, 80, 64, dict(top_k=6, **GROUPED)),
                                                    (9, 48, 144, 300, dict(top_k=8, score="sigmoid"))])
def test_moe(ops, tokens, h, f, experts, how, x8):
    """What is rounded is h to bf16 (2^-8; its errors are independent, so the norm of what they do is at most that) and the result (2^-8), and the fp32 sums
    and weights by 2^-18.  With 8-bit activations h is not rounded to bf16; it is quantised here as there, but from sums that differ: streamed by some 2^-20, so
    that a value in about 2^16 goes to the other neighbour, a 2^-3 of itself away (2^-3 * 2^-8 of the norm); on the tiles, whose sums are cut, by some 2^-15 of the norm, so
    that one in 2^11 does (2^-3 * 2^-5.5), and the down product's sums are cut as well (2^-15): less than the 2^-8 that h in bf16 would take."""
    r = np.random.Generator(np.random.PCG64(tokens + h + f))
    triple = tuple(weights(r, *s, experts) for s in ((f, h), (f, h), (h, f)))
    x = activations(r, tokens, h, x8)
    if x8:
        x.scale.mul_(8)
    logits = r.standard_normal((tokens, experts)).astype(np.float32)
    if experts > 8:
        logits[:, 1] = -np.inf
    bias = (r.standard_normal(experts) * 0.1).astype(np.float32) if "score" in how else None
    y = ops.moe_ffn(x, dev(logits), triple, bias=None if bias is None else dev(bias), **how)
    want = moe_oracle(ops, x, logits, triple, dict(how, bias=bias))
    assert y.dtype == torch.bfloat16 and O.rel_l2(y.double().cpu().numpy(), want) <= 2 * 2.0 ** -8 + 2.0 ** -18


@KINDS
@pytest.mark.parametrize("tokens", [6, 90, 700])
def test_moe_is_its_parts_and_replays(ops, x8, tokens):
    """The layer against its own operators in a row (route, sort, products by group, gate, down, weighted sum), eager and from a graph."""
    r = np.random.Generator(np.random.PCG64(77))
    h, f, experts, how = 256, 320, 32, dict(top_k=4, **GROUPED)
    gate, up, down = (weights(r, *s, experts) for s in ((f, h), (f, h), (h, f)))
    x = activations(r, tokens, h, False)
    logits, bias = dev(r.standard_normal((tokens, experts)).astype(np.float32)), dev((r.standard_normal(experts) * 0.1).astype(np.float32))

    def parts():
        idx, w = ops.moe_route(logits, bias=bias, **how)
        order = torch.sort(idx.flatten().long(), stable=True).indices
        offsets = torch.searchsorted(idx.flatten().long().sort().values, torch.arange(experts + 1, device=DEV)).to(torch.int32)
        xs = x[order // 4]
        xs = ops.quantize_fp8(xs) if x8 else xs
        g, u = ops.qgemm_grouped(xs, gate, offsets).float(), ops.qgemm_grouped(xs, up, offsets).float()
        hh = g * torch.sigmoid(g) * u
        d = ops.qgemm_grouped(ops.quantize_fp8(hh) if x8 else hh.to(torch.bfloat16), down, offsets).float()
        y = torch.empty_like(d)
        y[order] = d
        return (y.view(tokens, 4, h) * w[..., None]).sum(1)

    def layer():
        return ops.moe_ffn(ops.quantize_fp8(x) if x8 else x, logits, (gate, up, down), bias=bias, **how)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        layer()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y = layer()
    for turn in range(3):
        x.copy_(activations(r, tokens, h, False))
        logits.copy_(torch.randn_like(logits))
        eager, want = layer(), parts()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eager)
        # gate and up (half a step of bf16 each, silu's slope is at most 1.1) and the down product are rounded here, h and the result there (bf16); with 8-bit h a
        # rounding of 2^-8 before it moves a value in 2^4 / 2^1 * ... to its neighbour, 2^-3 away: at most sqrt(2^-8 / 2^-4 * 2) * 2^-4 on average over a step
        bound = (1.1 + 1 + 2 * 2) * 2.0 ** -8 + (2.0 ** -5 if x8 else 0)
        assert float((eager.double() - want.double()).norm() / want.double().norm()) <= bound


def test_moe_refusals(ops):
    r = np.random.Generator(np.random.PCG64(1))
    gate, up, down = (weights(r, *s, 4) for s in ((64, 32), (64, 32), (32, 64)))
    x, z = torch.zeros(3, 32, dtype=torch.bfloat16, device=DEV), torch.zeros(3, 4, device=DEV)
    assert not ops.moe_ffn(x, z, (gate, up, down)).any()
    assert not ops.moe_ffn(ops.quantize_fp8(x), z, [gate, up, down]).any()
    with pytest.raises(TypeError, match="triple"):
        ops.moe_ffn(x, z, (gate, up))
    for call, match in ((lambda: ops.moe_ffn(x, z, (gate, down, up)), "gate and up"), (lambda: ops.moe_ffn(x, z[:, :3], (gate, up, down)), "logits"),
                        (lambda: ops.moe_ffn(x, z, (gate, up, down), top_k=0), "unsupported"), (lambda: ops.moe_ffn(x, z, (gate, up, down), top_k=5), "unsupported"),
                        (lambda: ops.moe_ffn(x, z, (gate, up, down), groups=3), "groups"), (lambda: ops.moe_ffn(x, z, (gate, up, down), groups=4, top_groups=1), "groups"),
                        (lambda: ops.moe_ffn(x, z, (gate, up, down), bias=z[0, :3]), "bias must"), (lambda: ops.moe_ffn(x, z, (gate, up, down), score="tanh"), "score must"),
                        (lambda: ops.moe_ffn(x[:, :16], z, (gate, up, down)), r"\[T,32\]")):
        with pytest.raises(ValueError, match=match):
            call()
    mx = tuple(ops.quantize_mxfp4(ops.dequantize(w)) for w in (gate, up, down))
    with pytest.raises(ValueError, match="go with QExpertsFP8"):
        ops.moe_ffn(x, z, mx, score="sigmoid")
    with pytest.raises(TypeError, match="triple"):
        ops.moe_ffn(x, z, (mx[0], up, down))
    with pytest.raises(TypeError):
        ops.moe_ffn(ops.quantize_fp8(x), z, mx)


# ---- streams, graphs, threads of the interpreter --------------------------------------------------------------------------
@pytest.mark.parametrize("m", [3, 48, 300])
def test_captured_products_replay(ops, m):
    """Two graphs of different products and eager work in between: every replay is the eager result of the inputs it finds."""
    r = np.random.Generator(np.random.PCG64(m))
    n, k = 512, 4096
    cases, side = [], torch.cuda.Stream()
    for i in range(2):
        qw, x = weights(r, n, k), activations(r, m, k, False)
        with torch.cuda.stream(side):
            ops.qlinear(ops.quantize_fp8(x), qw)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            y = ops.qlinear(x, qw), ops.qlinear(ops.quantize_fp8(x), qw)
        cases.append((g, x, qw, y))
    for turn in range(3):
        for g, x, qw, y in cases:
            x.copy_(activations(r, m, k, False))
            want = ops.qlinear(x, qw), ops.qlinear(ops.quantize_fp8(x), qw)
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y[0], want[0]) and torch.equal(y[1], want[1])


@KINDS
@pytest.mark.parametrize("rows", [30, 400])
def test_captured_groups_follow_their_offsets(ops, rows, x8):
    """A captured product by group reads the offsets of the replay, not those of the capture."""
    x, w, offsets = grouped_case(rows, [rows // 4 + 1] * 4, 200, 272, x8)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.qgemm_grouped(x, w, offsets)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        y = ops.qgemm_grouped(x, w, offsets)
    rows = x64(x).shape[0]
    for bounds in ([0, 0, 0, 0, rows], [2, 9, 9, rows - 1, rows - 1], [0, 5, rows // 2, rows, rows]):
        offsets.copy_(torch.tensor(bounds, dtype=torch.int32))
        eager = ops.qgemm_grouped(x, w, offsets)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eager)
        check_groups(y, x, w, bounds)
        assert not y[:bounds[0]].any() and not y[bounds[-1]:].any()


@KINDS
def test_same_call_gives_the_same_bits_on_any_stream(ops, x8):
    r = np.random.Generator(np.random.PCG64(2))
    qw = weights(r, 600, 4096)
    for m in (1, 16, 60, 260):
        x = activations(r, m, 4096, x8)
        want = ops.qlinear(x, qw)
        torch.cuda.synchronize()
        streams, got = [torch.cuda.Stream() for _ in range(3)], []
        for st in streams:
            with torch.cuda.stream(st):
                got += [ops.qlinear(x, qw) for _ in range(4)]
        torch.cuda.synchronize()
        assert all(torch.equal(g, want) for g in got)


def test_without_the_host_module(ops, monkeypatch):
    """The Python road to the same kernels: the same bits."""
    from chadslab_amd import QExpertsFP8, QRowsFP8, QWeightFP8, _lib

    r = np.random.Generator(np.random.PCG64(5))
    qe, down = weights(r, 144, 256, 8), weights(r, 256, 144, 8)
    qw = qe.expert(1)
    x = activations(r, 40, 256, False)
    z, bias = dev(r.standard_normal((40, 8)).astype(np.float32)), dev(r.standard_normal(8).astype(np.float32) * 0.1)
    offsets = torch.tensor([0, 7, 7, 30, 31, 32, 33, 39, 40], dtype=torch.int32, device=DEV)

    def calls():
        q, e, w = ops.quantize_fp8(x), ops.quantize_fp8(x.float().view(2, 20, 256), rows=False), ops.quantize_fp8(x.half(), rows=False)
        assert type(q) is QRowsFP8 and type(e) is QExpertsFP8 and type(w) is QWeightFP8 and repr(q) and (q.M, q.K, e.E, w.N) == (40, 256, 2, 40)
        how = dict(top_k=3, score="sigmoid", bias=bias, groups=4, top_groups=3, group_sum=2, scale=1.5)
        return [q.w.view(torch.uint8), q.scale, e.w.view(torch.uint8), e.scale, w.scale, ops.dequantize(q), ops.dequantize(e), ops.dequantize(w), ops.qlinear(x, qw),
                ops.qlinear(x[:3], qw), ops.qlinear(q, qw), ops.qlinear(x[:3], qw, out_dtype=torch.bfloat16), ops.qgemm_grouped(x, qe, offsets),
                ops.qgemm_grouped(q, qe, offsets), ops.moe_ffn(x, z, (qe, qe, down)), ops.moe_ffn(q, z, (qe, qe, down), **how), *ops.moe_route(z, **how)]

    native = calls()
    monkeypatch.setattr(_lib, "_native", _lib._NoHostModule)
    for a, b in zip(native, calls()):
        assert a.dtype == b.dtype and torch.equal(a, b)


def test_weights_and_activations_quantised_and_multiplied(ops):
    """Load time and serving in a row: weights quantised on the GPU, activations quantised per call, both products."""
    r = np.random.Generator(np.random.PCG64(8))
    w, x = dev(r.standard_normal((300, 528)).astype(np.float32) * 0.05), dev(r.standard_normal((50, 528)).astype(np.float32)).to(torch.bfloat16)
    qw = ops.quantize_fp8(w, rows=False)
    check(ops.qlinear(x, qw), x.double(), w64(qw))
    q = ops.quantize_fp8(x)
    check(ops.qlinear(q, qw), x64(q), w64(qw), True)
    # a value is off by half a step of its own (2^-4) or of the smallest, independently: the product by no more than that of its norm
    assert O.rel_l2(ops.qlinear(q, qw).double().cpu().numpy(), (x.double() @ w.double().T).cpu().numpy()) <= 2 * 2.0 ** -4


def test_library_refuses(ops):
    """The C entry points' own checks: status and message, no launch."""
    from ctypes import byref

    from chadslab_amd import _lib

    lib = _lib.load()
    a = torch.zeros(4096, dtype=torch.uint8, device=DEV).data_ptr()
    for call, status in (((a, None, a, a, a, 0, 1, 1, 24, None, 0, None), -2), ((a, None, a, a, a, 0, -1, 1, 32, None, 0, None), -2), ((a, None, a, a, a, 0, 1, 1, 2 ** 26 + 16, None, 0, None), -2),
                         ((None, None, a, a, a, 0, 1, 1, 32, None, 0, None), -1), ((a, None, a, None, a, 0, 1, 1, 32, None, 0, None), -1), ((a + 8, None, a, a, a, 0, 1, 1, 32, None, 0, None), -3),
                         ((a, None, a + 4, a, a, 0, 1, 1, 32, None, 0, None), -3), ((a, a + 2, a, a, a, 0, 1, 1, 32, None, 0, None), -3), ((a, None, a, a, a, 0, 20, 1, 32, a + 4, 64, None), -3),
                         ((a, None, a, a, a, 0, 2 ** 31 - 1, 2 ** 31 - 1, 32, None, 0, None), -2)):
        assert lib.chadq_product_fp8(*call) == status, call
    assert lib.chadq_product_fp8(None, None, None, None, None, 0, 0, 5, 32, None, 0, None) == 0
    for call, status in (((a, None, a, a, a, a, 4, 0, 1, 32, 1, None), -2), ((a, None, a, a, None, a, 4, 1, 1, 32, 1, None), -1), ((a, None, a, a, a + 2, a, 4, 1, 1, 32, 1, None), -3),
                         ((a, None, a, a, a, a, 4, 1, 1, 33, 1, None), -2)):
        assert lib.chadq_product_fp8_grouped(*call) == status, call
    for call, status in (((a, 3, a, a, 1, 1, 32, 1, None), -2), ((a, 0, a, a, 1, 1, 24, 1, None), -2), ((a, 0, a, a, -1, 1, 32, 1, None), -2), ((a, 0, None, a, 1, 1, 32, 1, None), -1),
                         ((a + 4, 0, a, a, 1, 1, 32, 0, None), -3), ((a, 0, a + 8, a, 1, 1, 32, 0, None), -3), ((a, 0, a, a, 2 ** 62, 1, 32, 0, None), -2)):
        assert lib.chadq_quantize_fp8(*call) == status, call
    assert lib.chadq_dequant_fp8(a, a, a + 4, 1, 1, 32, 1, None) == -3 and lib.chadq_dequant_fp8(a, a, a, 1, 1, 31, 1, None) == -2
    sizes = lib.chadq_moe_ffn_fp8_workspace_bytes
    assert sizes(4, 64, 64, 513, 2, 0) == 0 and sizes(4, 64, 40, 4, 2, 0) == 0 and sizes(4, 64, 64, 4, 5, 1) == 0 and sizes(4, 64, 48, 4, 2, 1) > 0
    good = dict(bias=None, sigmoid=0, renorm=1, groups=4, top_groups=2, group_sum=1, top_k=2, scale=1.0)
    for change in (dict(groups=3), dict(groups=0), dict(groups=128), dict(top_groups=5), dict(top_groups=0), dict(group_sum=3), dict(group_sum=0), dict(top_k=33), dict(top_k=0),
                   dict(groups=64, group_sum=2), dict(top_groups=1, top_k=17)):
        assert lib.chadq_moe_route_experts(a, byref(_lib.Routing(**dict(good, **change))), a, a, 1, 64, None) == -2, change
    assert lib.chadq_moe_route_experts(None, byref(_lib.Routing(**good)), a, a, 1, 64, None) == -1 and lib.chadq_moe_route_experts(a, None, a, a, 1, 64, None) == -1
    assert lib.chadq_moe_route_experts(a + 2, byref(_lib.Routing(**good)), a, a, 1, 64, None) == -3 and lib.chadq_moe_route_experts(a, byref(_lib.Routing(**good)), a, a, 1, 513, None) == -2


def test_more_blocks_than_a_launch_has_threads_for(ops):
    """2^24 small matrices and more, a workgroup to each: all are done, and the ones at the borders are right."""
    e = 2 ** 24 + 3
    at = torch.tensor([0, 2 ** 22 - 1, 2 ** 22, 2 ** 24 - 1, 2 ** 24, e - 1], device=DEV)
    some = dev(np.random.Generator(np.random.PCG64(8)).standard_normal((6, 1, 16)).astype(np.float32)).to(torch.bfloat16)
    x = torch.full((e, 1, 16), 3.5, dtype=torch.bfloat16, device=DEV)
    x[at] = some
    q, want = ops.quantize_fp8(x, rows=False), ops.quantize_fp8(some, rows=False)
    values = q.w.view(torch.uint8)
    assert torch.equal(values[at], want.w.view(torch.uint8)) and torch.equal(q.scale[at], want.scale)
    values[at], q.scale[at] = 0x7E, 2.0 ** -7  # 448 and 3.5 / 448, as of all others
    assert bool((values == 0x7E).all()) and bool((q.scale == 2.0 ** -7).all())
    assert torch.equal(ops.dequantize(q)[at], torch.full((6, 1, 16), 3.5, device=DEV))
