"""MXFP4 on the CPU: the oracle's quantiser and values against their definitions one by one, the containers' and the operators'
refusals.  No GPU."""
import numpy as np
import pytest
import torch

from oracle import chadq_oracle as O


def test_values_of_all_codes_and_scales():
    codes = np.tile((np.arange(16, dtype=np.uint8)[0::2] | (np.arange(16, dtype=np.uint8)[1::2] << 4)), (256, 2))
    v = O.dequant_mxfp4(codes, np.arange(256, dtype=np.uint8)[:, None])
    for e in range(256):
        for c in range(16):
            m = c & 7
            want = (m & 1) / 2 if m < 2 else 2.0 ** (m // 2 - 1) * (1 + (m & 1) / 2)  # e2m1 read bit by bit
            want = (-want if c & 8 else want) * 2.0 ** (e - 127) if e < 255 else np.nan
            assert v[e, c] == want or (e == 255 and np.isnan(v[e, c]))


def test_oracle_takes_the_nearest_code_ties_to_even():
    r = np.random.Generator(np.random.PCG64(5))
    x = r.standard_normal((16, 64)) * np.exp(r.standard_normal((16, 1)) * 20)
    x[0, :16] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.99, -0.25, -0.75, -5.0, 4.0, 0.0, -0.0, 0.5]
    x[1, :32] = 0.0
    codes, scale = O.quantize_mxfp4(x.astype(np.float32))
    v = O.dequant_mxfp4(codes, scale)
    assert list(v[0, :13]) == [0, 1, 1, 2, 2, 4, 4, 6, 6, 0, -1, -4, 4] and scale[1, 0] == 0
    for row in range(16):
        for g in range(2):
            b = x[row, 32 * g:32 * g + 32].astype(np.float32).astype(np.float64)
            if not b.any():
                continue
            e = max(int(np.floor(np.log2(np.abs(b).max()))) - 2, -127)
            assert scale[row, g] == e + 127
            for i in range(32):
                q, t = abs(v[row, 32 * g + i]) / 2.0 ** e, min(abs(b[i]) / 2.0 ** e, 6.0)
                assert abs(q - t) == np.abs(O.MX_VALUES - t).min()


def test_containers_refuse_wrong_shapes_and_types():
    from chadslab_amd import QExpertsMXFP4, QWeightMXFP4

    p, s = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    q = QWeightMXFP4(p, s)
    assert (q.N, q.K) == (4, 64) and q.to("cpu").packed.shape == (4, 32)
    for bad in ((p.to(torch.int8), s), (p, s.to(torch.float16)), (p, s[:, :1]), (p[:, :8], s), (p[0], s), (p, s[:3])):
        with pytest.raises(ValueError):
            QWeightMXFP4(*bad)
    e = QExpertsMXFP4(p.view(2, 2, 32), s.view(2, 2, 2))
    assert (e.E, e.N, e.K) == (2, 2, 64) and e.expert(1).N == 2
    for bad in ((p, s), (p.view(2, 2, 32), s), (p.view(2, 2, 32), s.view(2, 2, 2).float())):
        with pytest.raises(ValueError):
            QExpertsMXFP4(*bad)


def test_operators_refuse_cpu_tensors_and_wrong_arguments():
    from chadslab_amd import QExpertsMXFP4, QWeightInt4G32, QWeightMXFP4, ops

    p, s = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    q, e = QWeightMXFP4(p, s), QExpertsMXFP4(p.view(2, 2, 32), s.view(2, 2, 2))
    x, off = torch.zeros(1, 64, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32)
    for call in (lambda: ops.quantize_mxfp4(x), lambda: ops.dequantize(q), lambda: ops.dequantize(e), lambda: ops.qgemv(x, q),
                 lambda: ops.qgemm(x, q), lambda: ops.qlinear(x, q), lambda: ops.qlinear(q, q), lambda: ops.qgemm_grouped(x, e, off)):
        with pytest.raises(ValueError, match="GPU tensor"):
            call()
    with pytest.raises(ValueError, match="multiple of 32"):
        ops.quantize_mxfp4(torch.zeros(2, 40))
    with pytest.raises(ValueError, match="multiple of 32"):
        ops.quantize_mxfp4(torch.zeros(64))
    with pytest.raises(ValueError, match="float32"):
        ops.quantize_mxfp4(torch.zeros(2, 64, dtype=torch.int32))
    with pytest.raises(ValueError, match=r"\[M,64\]"):
        ops.qgemm(torch.zeros(1, 32, dtype=torch.bfloat16), q)
    with pytest.raises(ValueError, match="fp32_elements"):
        ops.qgemv(x, q, fp32_elements=True)
    with pytest.raises(ValueError, match="at most 16 rows"):
        ops.qgemv(torch.zeros(17, 64, dtype=torch.bfloat16), q)
    with pytest.raises(TypeError, match="QExpertsMXFP4"):
        ops.qgemm_grouped(x, q, off)
    with pytest.raises(ValueError, match=r"\[R,64\]"):
        ops.qgemm_grouped(torch.zeros(1, 32, dtype=torch.bfloat16), e, off)
    i4 = QWeightInt4G32(p, torch.ones(4, 2, dtype=torch.float16))
    for call in (ops.qgemv, ops.qgemm, ops.qlinear):
        with pytest.raises(TypeError, match="MXFP4 activations"):
            call(q, i4)


def test_library_refuses_bad_sizes_without_a_launch():
    """The size rules that need no device: no workspace is ever asked for what the product refuses."""
    from chadslab_amd import _lib

    f = _lib.load().chadq_product_mxfp4_workspace_bytes
    for m, n, k in ((0, 64, 64), (4, 0, 64), (4, 64, 0), (4, 64, 48), (-1, 64, 64)):
        assert f(m, n, k, 0) == 0 and f(m, n, k, 1) == 0


def test_weight_file_holds_them(tmp_path):
    """One matrix and those of experts come back as they were; what a file cannot hold is refused instead of written as addresses."""
    from chadslab_amd import QExpertsMXFP4, QWeightMXFP4, wfile
    from chadslab_amd.formats import QWeightInt4G32Tiles

    r = np.random.Generator(np.random.PCG64(8))
    q, e = (c(*(torch.from_numpy(r.integers(0, 256, (*s, n), dtype=np.uint8)) for n in (48, 3))) for c, s in ((QWeightMXFP4, (5,)), (QExpertsMXFP4, (2, 5))))
    path = str(tmp_path / "w.chadq")
    wfile.save(path, {"one": q, "experts": e, "norm": torch.arange(4.0)})
    back = wfile.load(path)
    for name, want in (("one", q), ("experts", e)):
        assert type(back[name]) is type(want) and torch.equal(back[name].packed, want.packed) and torch.equal(back[name].scale, want.scale)
    assert torch.equal(back["norm"], torch.arange(4.0)) and wfile.read_header(path)["tensors"]["experts"]["shape"] == [2, 5, 96]
    for bad in (object(), QWeightInt4G32Tiles.__new__(QWeightInt4G32Tiles)):
        with pytest.raises(TypeError):
            wfile.save(path, {"w": bad})


def test_operators_look_at_a_containers_arrays_again():
    """Arrays exchanged since a container was made: those that no longer fit each other are refused, not read as far as the other's shape says."""
    from chadslab_amd import QExpertsMXFP4, QWeightMXFP4, ops

    p, s = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    x, off, z = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32), torch.zeros(4, 2)

    def weight(packed=p, scale=s):
        q = QWeightMXFP4(p, s)
        q.packed, q.scale = packed, scale
        return q

    def experts(packed=p.view(2, 2, 32), scale=s.view(2, 2, 2)):
        e = QExpertsMXFP4(p.view(2, 2, 32), s.view(2, 2, 2))
        e.packed, e.scale = packed, scale
        return e

    whole, group = weight(), experts()
    for bad, message in ((weight(scale=s[:, :1]), "scale must be uint8"), (weight(scale=s[:3]), "scale must be uint8"), (weight(scale=s.float()), "scale must be uint8"),
                         (weight(packed=p.view(2, 2, 32)), "packed must be uint8"), (weight(packed=p.flatten()), "packed must be uint8"), (weight(packed=p[:, :8]), "multiple of 32")):
        for call in (lambda: ops.dequantize(bad), lambda: ops.qgemv(x, bad), lambda: ops.qgemm(x, bad), lambda: ops.qlinear(x, bad), lambda: ops.qlinear(bad, whole),
                     lambda: ops.qgemm(bad, whole), lambda: ops.qgemm_grouped(bad, group, off)):
            with pytest.raises(ValueError, match=message):
                call()
    for bad, message in ((experts(scale=s.view(2, 2, 2)[:, :1]), "scale must be uint8"), (experts(scale=s.view(2, 2, 2)[:1]), "scale must be uint8"),
                         (experts(packed=p), "packed must be uint8"), (experts(packed=p.view(2, 2, 32)[..., :8]), "multiple of 32")):
        for call in (lambda: ops.dequantize(bad), lambda: ops.qgemm_grouped(x, bad, off), lambda: ops.moe_ffn(x, z, (bad, group, group), top_k=1), lambda: ops.moe_ffn(x, z, (group, group, bad), top_k=1)):
            with pytest.raises(ValueError, match=message):
                call()


def test_quantised_activations_of_more_than_two_dimensions_are_refused():
    """quantize_mxfp4 takes three dimensions for the matrices of experts; as activations these are refused by name."""
    from chadslab_amd import QExpertsMXFP4, QWeightInt4G32, QWeightInt8, QWeightMXFP4, ops

    p, s = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    q, e, off = QWeightMXFP4(p, s), QExpertsMXFP4(p.view(2, 2, 32), s.view(2, 2, 2)), torch.zeros(3, dtype=torch.int32)
    for call in (ops.qlinear, ops.qgemv, ops.qgemm, lambda x, _: ops.qgemm_grouped(x, e, off), lambda x, w: ops.qlinear(x, w, out_dtype=torch.bfloat16)):
        with pytest.raises(TypeError, match="quantize_mxfp4"):
            call(e, q)
        with pytest.raises(TypeError, match="x must be"):
            call(p.numpy(), q)
    for w in (QWeightInt4G32(p, torch.ones(4, 2, dtype=torch.float16)), QWeightInt8(p.to(torch.int8), torch.ones(4))):
        for call in (ops.qlinear, ops.qgemv, ops.qgemm):
            with pytest.raises(TypeError, match="MXFP4 activations"):
                call(e, w)


def test_int4_experts_are_not_looked_at_one_by_one_for_mxfp4(monkeypatch):
    """A call on int4 experts goes to the native function without a walk over them (1 us of host time at 16 experts)."""
    from chadslab_amd import QExpertsMXFP4, _lib, ops

    class Counted(list):
        walks = 0

        def __iter__(self):
            self.walks += 1
            return super().__iter__()

    class Native(_lib._NoHostModule):
        @staticmethod
        def moe_ffn(x, logits, experts, top_k, renorm):
            return "native"

    monkeypatch.setattr(_lib, "native", lambda: Native)
    experts = Counted([(None, None, None)] * 16)
    assert ops.moe_ffn(None, None, experts) == "native" and experts.walks == 0
    # MXFP4 in any other place than a triple's is still refused as what it is
    monkeypatch.setattr(_lib, "native", lambda: _lib._NoHostModule)
    e = QExpertsMXFP4(torch.zeros(2, 2, 32, dtype=torch.uint8), torch.zeros(2, 2, 2, dtype=torch.uint8))
    for bad in ([e], [e, e], (None, e, e), [e, e, e, e], (e, None, e)):
        with pytest.raises(TypeError, match="triple"):
            ops.moe_ffn(None, None, bad)


def test_tiles_of_the_largest_sizes_are_counted():
    """Rows or columns within a tile of 2^31: their tiles are too many, not fewer than none, so K in parts (gigabytes of workspace) is not what the rule wants."""
    from chadslab_amd import _lib

    f = _lib.load().chadq_product_mxfp4_workspace_bytes
    for most in (2 ** 31 - 1, 2 ** 31 - 32, 2 ** 31 - 300):
        for small in (1, 17, 100):
            for k in (1024, 4096, 14336):
                assert f(most, small, k, 0) == f(most, small, k, 1) == 0
                assert f(small, most, k, 0) == f(small, most, k, 1) == 0
