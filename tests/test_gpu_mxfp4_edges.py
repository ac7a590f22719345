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
