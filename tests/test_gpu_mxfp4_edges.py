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
