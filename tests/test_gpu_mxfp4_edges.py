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
