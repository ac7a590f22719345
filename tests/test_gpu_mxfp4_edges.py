"""MXFP4 on the GPU: calls at the ends of what the operators document, and refusals of what lies beyond."""
import numpy as np
import pytest
import torch

from oracle import chadq_oracle as O
from tests.test_gpu_mxfp4 import DEV, activations, check, dev, ops, weights  # noqa: F401  (ops: the fixture)

pytestmark = pytest.mark.gpu


def test_exchanged_arrays_are_looked_at_again(ops):
    """Arrays put into a container after it was made: used where they fit each other, refused where they do not."""
    from chadslab_amd import QExpertsMXFP4, QWeightMXFP4

    r = np.random.Generator(np.random.PCG64(4))
    n, k = 64, 128
    (c, s), (c2, s2) = weights(r, n, k), weights(r, 2 * n, k)
    off = torch.tensor([0, 5], dtype=torch.int32, device=DEV)
    for m in (5, 40):
        x, x64 = activations(r, m, k, False)
        qw = QWeightMXFP4(dev(c), dev(s))
        qw.packed = dev(c2)
        for call in (lambda: ops.qlinear(x, qw), lambda: ops.qgemm(x, qw), lambda: ops.dequantize(qw), lambda: ops.qlinear(qw, QWeightMXFP4(dev(c), dev(s)))):
            with pytest.raises(ValueError, match="scale must be"):
                call()
        e = QExpertsMXFP4(dev(c)[None], dev(s)[None])
        e.scale = e.scale[:, :n // 2]
        for call in (lambda: ops.qgemm_grouped(x, e, off), lambda: ops.dequantize(e), lambda: ops.moe_ffn(x, torch.zeros(m, 1, device=DEV), (e, e, e), top_k=1)):
            with pytest.raises(ValueError, match="scale must be"):
                call()
        qw.scale = dev(s2)
        check(ops.qlinear(x, qw), x64, dev(O.dequant_mxfp4(c2, s2)))
        check(ops.qgemm(x, qw), x64, dev(O.dequant_mxfp4(c2, s2)))


def test_too_many_tiles_are_refused(ops):
    """Rows or columns up to the last 32-bit number, the other few: the status of a size that is refused, and no launch."""
    from chadslab_amd import _lib

    lib = _lib.load()
    a = torch.zeros(4096, dtype=torch.uint8, device=DEV).data_ptr()
    for most in (2 ** 31 - 1, 2 ** 31 - 32, 2 ** 31 - 300):
        for m, n in ((most, 1), (17, most), (40, most), (most, 17)):
            for k in (32, 4096):
                for xs in (None, a):
                    assert lib.chadq_product_mxfp4(a, xs, a, a, a, 1, m, n, k, None, 0, None) == -2 and b"too many tiles" in lib.chadq_last_error()
                    assert lib.chadq_product_mxfp4_grouped(a, xs, a, a, a, a, m, 1, n, k, 1, None) == -2 and b"too many tiles" in lib.chadq_last_error()
    assert lib.chadq_product_mxfp4_grouped(a, None, a, a, a, a, 2 ** 31 - 1, 2 ** 31 - 2, 1, 32, 1, None) == -2  # (rows and groups)


@pytest.mark.parametrize("x4", [False, True], ids=["bf16", "mxfp4"])
@pytest.mark.parametrize("n", [4194240, 4194241, 5000000])
def test_few_rows_of_millions_of_columns(ops, n, x4):
    """On both sides of what the streaming grid holds; one matrix and by group."""
    from chadslab_amd import QExpertsMXFP4, QWeightMXFP4

    k = 32
    g = torch.Generator(device=DEV).manual_seed(n)
    c = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device=DEV, generator=g)
    s = torch.randint(118, 124, (n, 1), dtype=torch.uint8, device=DEV, generator=g)
    w64 = ops.dequantize(QWeightMXFP4(c, s)).double()
    for m in (1, 16):
        x, x64 = activations(np.random.Generator(np.random.PCG64(m)), m, k, x4)
        check(ops.qlinear(x, QWeightMXFP4(c, s)), x64, w64)
        check(ops.qlinear(x, QWeightMXFP4(c, s), out_dtype=torch.bfloat16), x64, w64)
    off = torch.tensor([1, 14], dtype=torch.int32, device=DEV)
    y = ops.qgemm_grouped(x, QExpertsMXFP4(c[None], s[None]), off)
    check(y[1:14], x64[1:14], w64)
    assert not y[0].any() and not y[14:].any()


def test_moe_of_millions_of_hidden_columns(ops):
    """Gate and up beyond the streaming grid's columns; their product is then the down product's K, beyond what the tiles' offsets hold."""
    from chadslab_amd import QExpertsMXFP4

    h, f, t = 32, 4194240 + 96, 2
    g = torch.Generator(device=DEV).manual_seed(1)

    def experts(n, k):
        return QExpertsMXFP4(torch.randint(0, 256, (1, n, k // 2), dtype=torch.uint8, device=DEV, generator=g),
                             torch.randint(118, 124, (1, n, k // 32), dtype=torch.uint8, device=DEV, generator=g))

    gate, up, down = experts(f, h), experts(f, h), experts(h, f)
    x = torch.randn(t, h, device=DEV, generator=g).to(torch.bfloat16)
    y = ops.moe_ffn(x, torch.zeros(t, 1, device=DEV), (gate, up, down), top_k=1)
    a, b, d = (ops.dequantize(m)[0].double() for m in (gate, up, down))
    u = x.double() @ a.T
    want = (u * torch.sigmoid(u) * (x.double() @ b.T)) @ d.T
    # h and the result are rounded to bf16 (as in test_moe); down adds 131075 instructions' worth of products in fp32, each addition off by at most 2^-24 of a
    # sum that grows with the root of their number, independently: 2^-24 sqrt(131075 / 2) = 2^-16
    assert O.rel_l2(y.double().cpu().numpy(), want.cpu().numpy()) <= 2 * 2.0 ** -8 + 2.0 ** -16


# ---- K in parts, the last one shorter; (the rule, asked on the host, is held to the tile and the number of parts given here) ----
@pytest.mark.parametrize("x4,m,n,k,want", [(False, 93, 16, 7392, ("64x32", 8)), (False, 1392, 65, 6592, ("64x64", 5)), (False, 1409, 77, 7904, ("128x64", 8)),
                                           (False, 1869, 130, 24384, ("256x64", 8)), (False, 1488, 338, 10592, ("128x128", 7)), (False, 2044, 641, 12672, ("256x128", 5)),
                                           (False, 1901, 663, 11872, ("256x96", 4)), (False, 1812, 276, 12256, ("128x96", 4)), (True, 49, 16, 3712, ("64x32", 4)),
                                           (True, 1680, 65, 5792, ("64x64", 3)), (True, 1393, 202, 22112, ("128x64", 5)), (True, 1063, 1225, 16640, ("256x64", 3)),
                                           (True, 1871, 153, 22592, ("128x128", 8)), (True, 2021, 684, 25344, ("256x128", 5)), (True, 2039, 2091, 16800, ("256x256", 3)),
                                           (True, 670, 2161, 24416, ("256x96", 4)), (True, 1362, 195, 18880, ("128x96", 8))])
def test_every_tile_in_parts_of_k(ops, x4, m, n, k, want):
    """Through Python, and through the C entry point into fp32 and bf16 with a workspace full of NaN."""
    from chadslab_amd import QWeightMXFP4, _lib

    lib = _lib.load()
    need = lib.chadq_product_mxfp4_workspace_bytes(m, n, k, int(x4))
    assert need == want[1] * m * n * 4
    r = np.random.Generator(np.random.PCG64(m + n))
    c, s = weights(r, n, k)
    qw, w64 = QWeightMXFP4(dev(c), dev(s)), dev(O.dequant_mxfp4(c, s))
    x, x64 = activations(r, m, k, x4)
    y = ops.qlinear(x, qw)
    check(y, x64, w64)
    xt, xs = (x.packed, x.scale.data_ptr()) if x4 else (x, None)
    for dtype in (torch.float32, torch.bfloat16):
        ws = torch.full((need,), 255, dtype=torch.uint8, device=DEV)
        out = torch.full((m, n), float("nan"), dtype=dtype, device=DEV)
        assert lib.chadq_product_mxfp4(xt.data_ptr(), xs, qw.packed.data_ptr(), qw.scale.data_ptr(), out.data_ptr(), int(dtype == torch.bfloat16), m, n, k, ws.data_ptr(),
                                       need, torch.cuda.current_stream().cuda_stream) == 0
        check(out, x64, w64)
    assert torch.equal(out, y)


def moe_in_64_bits(x64, logits, mats, top_k, renorm):
    idx, w = O.moe_route(logits, top_k, renorm)
    idx, w = dev(idx.astype(np.int64)), dev(w.astype(np.float64))
    y = torch.zeros_like(x64)
    for e in range(len(mats[0][0])):
        gate, up, down = (dev(O.dequant_mxfp4(c[e], s[e])) for c, s in mats)
        g, u = x64 @ gate.T, x64 @ up.T
        y += (w * (idx == e)).sum(1, keepdim=True) * ((g * torch.sigmoid(g) * u) @ down.T)
    return y


@pytest.mark.parametrize("tokens,h,f,experts,top_k,want", [(57, 320, 5568, 4, 2, ("64x32", 4)), (60, 384, 11808, 8, 2, ("64x32", 4)), (824, 32, 6112, 4, 4, ("64x32", 2)),
                                                           (973, 32, 7232, 4, 4, ("64x64", 4)), (541, 224, 12096, 4, 4, ("128x64", 3)),
                                                           (1021, 608, 10656, 2, 2, ("128x128", 3)), (1015, 96, 16000, 4, 4, ("128x96", 4)),
                                                           (789, 416, 13760, 4, 4, ("256x128", 4)), (855, 1504, 6080, 1, 1, ("256x64", 3)), (664, 448, 11904, 4, 4, ("256x96", 4))])
def test_moe_down_in_parts_of_k(ops, tokens, h, f, experts, top_k, want):
    """The experts' down product summed in parts that the weighted sum joins: against 64 bits (bound: as in test_moe), the same bits twice and from a graph."""
    from chadslab_amd import QExpertsMXFP4, _lib

    pairs = tokens * top_k
    need = _lib.load().chadq_moe_ffn_mxfp4_workspace_bytes(tokens, h, f, experts, top_k)
    assert 0 <= need - pairs * (2 * f + 4 * want[1] * h) <= 16 * pairs + 4096  # h as bf16, every part as fp32, and the router's four words to a pair
    r = np.random.Generator(np.random.PCG64(tokens + f))
    mats = [weights(r, experts, *shape, spread=0.5) for shape in ((f, h), (f, h), (h, f))]
    x, x64 = activations(r, tokens, h, False)
    logits = r.standard_normal((tokens, experts)).astype(np.float32)
    if experts > top_k:
        logits[:, 1] = -50.0  # nobody's choice
    triple, z = tuple(QExpertsMXFP4(dev(c), dev(s)) for c, s in mats), dev(logits)
    y = ops.moe_ffn(x, z, triple, top_k=top_k)
    assert torch.isfinite(y).all()
    assert O.rel_l2(y.double().cpu().numpy(), moe_in_64_bits(x64, logits, mats, top_k, True).cpu().numpy()) <= 2 * 2.0 ** -8 + 2.0 ** -18
    assert torch.equal(ops.moe_ffn(x, z, triple, top_k=top_k), y)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        captured = ops.moe_ffn(x, z, triple, top_k=top_k)
    for turn in range(3):
        x.copy_(activations(r, tokens, h, False)[0])
        z.copy_(torch.randn_like(z))
        eager = ops.moe_ffn(x, z, triple, top_k=top_k)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, eager)


# ---- K, addresses and groups at their largest -----------------------------------------------------------------------------
def sparse_rows(m, k, g, x4):
    """Activations of -1, 0 and 1, some ten thousand of them not 0, the row's first and last blocks among them: sums of halves below 2^23, exact in any order."""
    from chadslab_amd import QWeightMXFP4

    at = torch.cat((torch.randint(0, k, (10000,), device=DEV, generator=g), torch.arange(40, device=DEV), torch.arange(k - 40, k, device=DEV))).unique()
    v = torch.randint(0, 2, (m, len(at)), device=DEV, generator=g, dtype=torch.int8) * 2 - 1
    if not x4:
        x = torch.zeros(m, k, dtype=torch.bfloat16, device=DEV)
        x[:, at] = v.to(torch.bfloat16)
        return x, at, v
    codes = torch.zeros(m, k, dtype=torch.uint8, device=DEV)
    codes[:, at] = torch.where(v > 0, 2, 10).to(torch.uint8)  # 1, -1
    return QWeightMXFP4(codes[:, 0::2] | codes[:, 1::2] << 4, torch.full((m, k // 32), 127, dtype=torch.uint8, device=DEV)), at, v


def columns(codes, at):
    """The values of codes [.., K/2] at some k, in 64 bits."""
    c = codes[..., at // 2]
    c = torch.where(at % 2 == 1, c >> 4, c & 15).long()
    return dev(np.concatenate((O.MX_VALUES, -O.MX_VALUES)))[c]


@pytest.mark.parametrize("x4,m,k", [(False, 1, 2 ** 26), (False, 16, 2 ** 26), (True, 3, 2 ** 26), (True, 16, 2 ** 26), (False, 20, 4194272), (False, 20, 4194304), (False, 70, 4194336),
                                    (True, 20, 16777184), (True, 20, 16777216), (True, 70, 16777248), (False, 40, 2 ** 20 + 32), (True, 40, 2 ** 20 + 32)])
def test_the_longest_k(ops, x4, m, k):
    """Up to 2^26, and on both sides of what the tiles' 32-bit offsets hold (rows of 2^23 bytes); one matrix and by group."""
    from chadslab_amd import QExpertsMXFP4, QWeightMXFP4

    g = torch.Generator(device=DEV).manual_seed(k + m)
    n = 5
    codes = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device=DEV, generator=g)
    scale = torch.full((n, k // 32), 127, dtype=torch.uint8, device=DEV)
    x, at, v = sparse_rows(m, k, g, x4)
    want = v.double() @ columns(codes, at).T
    assert bool((want.abs() < 2 ** 22).all())
    y = ops.qlinear(x, QWeightMXFP4(codes, scale))
    assert torch.equal(y.double(), want.to(y.dtype).double())
    off = torch.tensor([0, m - 1, m], dtype=torch.int32, device=DEV)
    if k <= 2 ** 24:
        y = ops.qgemm_grouped(x, QExpertsMXFP4(codes[:4].view(2, 2, -1), scale[:4].view(2, 2, -1)), off)
        assert torch.equal(y.double(), torch.cat((want[:m - 1, :2], want[m - 1:, 2:4])).to(torch.bfloat16).double())


@pytest.mark.parametrize("x4", [False, True], ids=["bf16", "mxfp4"])
def test_weights_beyond_four_gigabytes(ops, x4):
    """Codes of 4.6 GB, as one matrix and as experts'; the last rows' addresses do not fit 32 bits."""
    from chadslab_amd import QExpertsMXFP4, QWeightMXFP4

    g = torch.Generator(device=DEV).manual_seed(11)
    n, k = 70016, 131072
    codes = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device=DEV, generator=g)
    scale = torch.full((n, k // 32), 127, dtype=torch.uint8, device=DEV)
    some = torch.cat((torch.arange(40, device=DEV), torch.arange(n - 300, n, device=DEV)))
    e = 32
    experts = QExpertsMXFP4(codes.view(e, n // e, -1), scale.view(e, n // e, -1))
    for m in (1, 16, 40, 300):
        x, at, v = sparse_rows(m, k, g, x4)
        want = v.double() @ columns(codes[some], at).T
        y = ops.qlinear(x, QWeightMXFP4(codes, scale))[:, some]
        assert torch.equal(y.double(), want.to(y.dtype).double())
        off = torch.full((e + 1,), m, dtype=torch.int32, device=DEV)
        off[:e] = 0  # all rows are the last expert's
        y = ops.qgemm_grouped(x, experts, off)[:, -300:]
        assert torch.equal(y.double(), want[:, -300:].to(torch.bfloat16).double())


@pytest.mark.parametrize("x4", [False, True], ids=["bf16", "mxfp4"])
def test_results_beyond_four_gigabytes(ops, x4):
    """40000 x 60000: rows behind 2^31 elements, computed and cleared."""
    from chadslab_amd import QExpertsMXFP4, QWeightMXFP4

    m, n, k = 40000, 60000, 64
    r = np.random.Generator(np.random.PCG64(12))
    c, s = weights(r, n, k)
    x, x64 = activations(r, m, k, x4)
    qw, w64 = QWeightMXFP4(dev(c), dev(s)), dev(O.dequant_mxfp4(c, s))
    rows, cols = [0, 1, 35790, 35791, 35792, 35793, 39998, 39999], slice(0, n, 7)
    y = ops.qlinear(x, qw)
    check(y[rows][:, cols], x64[rows], w64[cols])
    off = torch.tensor([2, 39999], dtype=torch.int32, device=DEV)
    out = ops.qgemm_grouped(x, QExpertsMXFP4(qw.packed[None], qw.scale[None]), off)
    assert not out[:2].any() and not out[39999].any()
    check(out[rows[2:-1]][:, cols], x64[rows[2:-1]], w64[cols])


def test_quantising_beyond_four_gigabytes(ops):
    x = torch.randn(70000, 40960, device=DEV, generator=torch.Generator(device=DEV).manual_seed(13), dtype=torch.bfloat16)
    q = ops.quantize_mxfp4(x)
    for rows in (slice(0, 3), slice(52427, 52430), slice(69990, 70000)):  # (2^31 values are 52428.8 rows)
        part = ops.quantize_mxfp4(x[rows].contiguous())
        assert torch.equal(q.packed[rows], part.packed) and torch.equal(q.scale[rows], part.scale)
    codes, scale = O.quantize_mxfp4(x[-2:].double().cpu().numpy())
    assert np.array_equal(q.packed[-2:].cpu().numpy(), codes) and np.array_equal(q.scale[-2:].cpu().numpy(), scale)
    back = ops.dequantize(q)
    assert np.array_equal(back[-2:].double().cpu().numpy(), O.dequant_mxfp4(codes, scale))


@pytest.mark.parametrize("x4", [False, True], ids=["bf16", "mxfp4"])
@pytest.mark.parametrize("groups,rows,k", [(65, 700, 96), (100, 1500, 288), (257, 3000, 64), (1000, 9000, 32), (64, 512, 352), (300, 2000, 96)])
def test_many_groups(ops, groups, rows, k, x4):
    """More groups than a wave has lanes, streamed and in tiles: uneven ones, and all rows in one of them; rows of no group."""
    from chadslab_amd import QExpertsMXFP4

    n = 40
    r = np.random.Generator(np.random.PCG64(groups))
    c, s = weights(r, groups, n, k)
    x, x64 = activations(r, rows, k, x4)
    w, w64 = QExpertsMXFP4(dev(c), dev(s)), dev(O.dequant_mxfp4(c, s))
    first, last = 3, rows - 5
    spread = r.multinomial(last - first, r.dirichlet(np.full(groups, 0.3)))
    one = np.zeros(groups, dtype=np.int64)
    one[groups - 2] = last - first
    for counts in (spread, one):
        bounds = [first, *(first + np.cumsum(counts)).tolist()]
        y = ops.qgemm_grouped(x, w, torch.tensor(bounds, dtype=torch.int32, device=DEV))
        for e in np.flatnonzero(counts):
            check(y[bounds[e]:bounds[e + 1]], x64[bounds[e]:bounds[e + 1]], w64[e])
        assert not y[:first].any() and not y[last:].any()


# ---- alignment, threads, what is not finite ---------------------------------------------------------------------------------
@pytest.mark.parametrize("m,n,k", [(4, 64, 128), (40, 64, 128), (40, 66, 128), (48, 512, 8192), (300, 64, 96)])
def test_results_at_any_address(ops, m, n, k):
    """`out` may begin at any element; what lies around it stays."""
    from chadslab_amd import QExpertsMXFP4, QWeightMXFP4

    r = np.random.Generator(np.random.PCG64(m))
    c, s = weights(r, n, k)
    x, x64 = activations(r, m, k, False)
    qw, w64, off = QWeightMXFP4(dev(c), dev(s)), dev(O.dequant_mxfp4(c, s)), torch.tensor([0, m], dtype=torch.int32, device=DEV)
    calls = [(torch.bfloat16, lambda o: ops.qgemm(x, qw, out=o)), (torch.bfloat16, lambda o: ops.qgemm_grouped(x, QExpertsMXFP4(qw.packed[None], qw.scale[None]), off, out=o))]
    if m <= 16:
        calls.append((torch.float32, lambda o: ops.qgemv(x, qw, out=o)))
    for shift in (1, 2, 3, 5):
        for dtype, call in calls:
            buf = torch.full((m * n + 16,), 7.0, dtype=dtype, device=DEV)
            check(call(buf[shift:shift + m * n].view(m, n)), x64, w64)
            assert bool((buf[:shift] == 7).all()) and bool((buf[shift + m * n:] == 7).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_blocks_of_subnormal_values(ops, dtype):
    """Blocks whose largest value is subnormal, or hardly not: bytes from 0 on (fp16's subnormal values are ordinary ones)."""
    info = torch.finfo(dtype)
    step = info.smallest_normal * info.eps
    r = np.random.Generator(np.random.PCG64(21))
    top = np.exp2(r.uniform(0, 4 - np.log2(info.eps), (500, 1)))  # in steps of the smallest value, to 16 times the smallest normal one
    x = np.rint(r.uniform(-1, 1, (500, 32)) * top) * step
    xt = torch.from_numpy(x).to(dtype)
    q = ops.quantize_mxfp4(xt.to(DEV))
    codes, scale = O.quantize_mxfp4(xt.double().numpy())
    assert np.array_equal(q.packed.cpu().numpy(), codes) and np.array_equal(q.scale.cpu().numpy(), scale)
    assert np.array_equal(ops.dequantize(q).double().cpu().numpy(), O.dequant_mxfp4(codes, scale))


@pytest.mark.parametrize("tokens", [3, 40, 300])
def test_what_is_not_finite_stays_with_its_token(ops, tokens):
    """A token with a NaN, one with infinities, and an expert with a NaN block: only the tokens that they meet are not finite."""
    from chadslab_amd import QExpertsMXFP4

    h, f, experts, top_k = 96, 160, 6, 2
    r = np.random.Generator(np.random.PCG64(tokens))
    mats = [weights(r, experts, *shape, spread=0.5) for shape in ((f, h), (f, h), (h, f))]
    for c, s in mats[:2]:
        c[c & 7 == 0] |= 1  # (no zeros to meet the infinities)
        c[c & 0x70 == 0] |= 0x10
    mats[0][1][4, 7, 1] = 255
    x, _ = activations(r, tokens, h, False)
    logits = r.standard_normal((tokens, experts)).astype(np.float32)
    logits[:2, 4] = -50.0
    clean = [tuple(QExpertsMXFP4(dev(c), dev(np.where(s == 255, 120, s).astype(np.uint8))) for c, s in mats), tuple(QExpertsMXFP4(dev(c), dev(s)) for c, s in mats)]
    before = ops.moe_ffn(x, dev(logits), clean[0], top_k=top_k)
    bad = x.clone()
    bad[0, 5], bad[1, 6] = float("nan"), float("inf")
    y = ops.moe_ffn(bad, dev(logits), clean[1], top_k=top_k)
    idx, _ = O.moe_route(logits, top_k, True)
    hit = torch.from_numpy((idx == 4).any(1))
    hit[:2] = True
    assert torch.equal((~torch.isfinite(y)).any(1).cpu(), hit) and torch.equal(y[~hit.to(DEV)], before[~hit.to(DEV)])


@pytest.mark.parametrize("tokens,experts,top_k", [(1, 16, 8), (5, 16, 8), (70, 16, 8), (300, 9, 7), (64, 16, 1), (65, 8, 8)])
def test_moe_of_many_choices(ops, tokens, experts, top_k):
    from chadslab_amd import QExpertsMXFP4

    h, f = 160, 224
    r = np.random.Generator(np.random.PCG64(tokens))
    mats = [weights(r, experts, *shape, spread=0.5) for shape in ((f, h), (f, h), (h, f))]
    x, x64 = activations(r, tokens, h, False)
    logits = r.standard_normal((tokens, experts)).astype(np.float32)
    for renorm in (True, False):
        y = ops.moe_ffn(x, dev(logits), tuple(QExpertsMXFP4(dev(c), dev(s)) for c, s in mats), top_k=top_k, renorm=renorm)
        assert O.rel_l2(y.double().cpu().numpy(), moe_in_64_bits(x64, logits, mats, top_k, renorm).cpu().numpy()) <= 2 * 2.0 ** -8 + 2.0 ** -18


def test_calls_of_several_threads(ops):
    """Threads with streams of their own, products that need a workspace among them: each gets the bits of the call alone."""
    import threading

    from chadslab_amd import QWeightMXFP4

    r = np.random.Generator(np.random.PCG64(31))
    c, s = weights(r, 512, 8192)
    qw = QWeightMXFP4(dev(c), dev(s))
    xs = [activations(r, m, 8192, False)[0] for m in (1, 16, 48, 100)]
    want = [(ops.qlinear(x, qw), ops.qlinear(ops.quantize_mxfp4(x), qw)) for x in xs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                got = ops.qlinear(xs[i], qw), ops.qlinear(ops.quantize_mxfp4(xs[i]), qw)
            torch.cuda.current_stream().synchronize()
            if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("tokens", [262143, 262144])
def test_moe_of_activations_around_two_gigabytes(ops, tokens):
    """Rows that are read through the sorted token list, on both sides of what the tiles' 32-bit offsets reach."""
    from chadslab_amd import QExpertsMXFP4

    h, f, experts = 4096, 64, 2
    r = np.random.Generator(np.random.PCG64(3))
    mats = [weights(r, experts, *shape, spread=0.5) for shape in ((f, h), (f, h), (h, f))]
    g = torch.Generator(device=DEV).manual_seed(5)
    x = torch.randn(tokens, h, device=DEV, generator=g, dtype=torch.bfloat16)
    logits = torch.randn(tokens, experts, device=DEV, generator=g)
    y = ops.moe_ffn(x, logits, tuple(QExpertsMXFP4(dev(c), dev(s)) for c, s in mats), top_k=1)
    some = torch.cat((torch.arange(3, device=DEV), torch.arange(0, tokens, 1009, device=DEV), torch.arange(tokens - 3, tokens, device=DEV)))
    want = moe_in_64_bits(x[some].double(), logits[some].cpu().numpy(), mats, 1, True)
    assert O.rel_l2(y[some].double().cpu().numpy(), want.cpu().numpy()) <= 2 * 2.0 ** -8 + 2.0 ** -18
    assert torch.isfinite(y).all()
