"""Products on FP8 weights on every tile that the rule by size takes, K in parts, and addresses beyond 32 bits, against torch in 64 bits on the GPU.  The bounds
are those of test_gpu_fp8: an element is off by (98 + G) 2^-24 S, and by 7 2^-13 S more where 8-bit activations meet the 8-bit matrix instruction, S = sum |x w|
of it, and a bf16 result by half a step, 2^-8, more.  K in parts adds at most 8 additions, which the 64 partial sums counted there hold."""
import threading

import numpy as np
import pytest
import torch

from test_fp8_rules import DENSE, DOWN, GROUPED, first_of_each, pick, sizes
from test_gpu_fp8 import DEV, FP8, KINDS, activations, blocks, check, check_groups, narrow, ops, rows_of, scales, values, w64, weights, x64  # noqa: F401

pytestmark = pytest.mark.gpu


@KINDS
def test_every_dense_tile(ops, x8):
    for (tile, parts), (m, n, k, _) in first_of_each(DENSE, x8).items():
        print(tile, parts, m, n, k, flush=True)
        r = np.random.Generator(np.random.PCG64(m + n + k))
        qw, x = weights(r, n, k), activations(r, m, k, x8)
        check(ops.qlinear(x, qw), x64(x), w64(qw), x8)
        qw, x = weights(r, n, k, values=narrow), activations(r, m, k, x8, values=narrow)
        check(ops.qlinear(x, qw), x64(x), w64(qw))


@KINDS
def test_every_tile_by_group(ops, x8):
    """Groups of the same rows, and one with most of them, empty ones beside it."""
    for (tile, _), (m, n, k, e) in first_of_each(GROUPED, x8).items():
        print(tile, m, n, k, e, flush=True)
        r = np.random.Generator(np.random.PCG64(m + n + k + e))
        w, x = weights(r, n, k, e, values=narrow), activations(r, m, k, x8, values=narrow)
        for bounds in ([m * i // e for i in range(e + 1)], [1] * (e // 2 + 1) + [m - 3] * (e - e // 2)):
            y = ops.qgemm_grouped(x, w, torch.tensor(bounds, dtype=torch.int32, device=DEV))
            check_groups(y, x, w, bounds, cut=False)
            assert not y[:bounds[0]].any() and not y[bounds[-1]:].any()


def layer_in_64(ops, x, triple, idx, weight):
    """-> the result and S: per token, sum over its experts of weight * (|h| |down|^T)"""
    a, y = x64(x), torch.zeros(x.shape[0] if isinstance(x, torch.Tensor) else x.M, triple[2].N, dtype=torch.float64, device=DEV)
    s = torch.zeros_like(y)
    for e in range(triple[0].E):
        at, j = (idx == e).nonzero(as_tuple=True)
        if not len(at):
            continue
        g, u, d = (w64(w.expert(e)) for w in triple)
        h = a[at] @ g.T
        h = h * torch.sigmoid(h) * (a[at] @ u.T)
        if not isinstance(x, torch.Tensor):
            h = x64(ops.quantize_fp8(h.float()))
        y.index_add_(0, at, weight[at, j, None].double() * (h @ d.T))
        s.index_add_(0, at, weight[at, j, None].double() * (h.abs() @ d.abs().T))
    return y, s


@KINDS
@pytest.mark.parametrize("which", ["gate and up", "down"])
def test_every_tile_of_the_layer(ops, x8, which):
    """Pairs by expert to their products' tiles, two experts to a token.  Of the norm: h in bf16 and the result (2^-8 each), the fp32 sums and weights 2^-18.
    With 8-bit x the values of gate and up are narrow, so h is the same as in 64 bits but for fp32 roundings, and an h goes to its other
    neighbour at a 2^-16th of places, 2^-3 of itself away (2^-3 2^-8 of the norm); the down product is cut: 7 2^-13 of the norm of S."""
    seen = set()
    for pairs, n, k, e in sizes(GROUPED, 1 << 33):
        h, f = (k, n) if which == "gate and up" else (n, k)
        if n % 16 or pairs % 2 or h * f > 1 << 24:
            continue
        gated, most = (True, 1) if which == "gate and up" else (False, 4)
        tile, part_k = pick(pairs, n, k, e, x8, gated, most)
        if (tile, part_k > 0) in seen:
            continue
        seen.add((tile, part_k > 0))
        print(tile, part_k, pairs, h, f, e, flush=True)
        r = np.random.Generator(np.random.PCG64(pairs + h + f))
        triple = (*(weights(r, f, h, e, values=narrow) for _ in range(2)), weights(r, h, f, e))
        x = activations(r, pairs // 2, h, x8, values=narrow)
        logits = torch.from_numpy(r.standard_normal((pairs // 2, e)).astype(np.float32)).to(DEV)
        want, s = layer_in_64(ops, x, triple, *ops.moe_route(logits, top_k=2))
        off = (ops.moe_ffn(x, logits, triple, top_k=2).double() - want).norm()
        bound = (2 * 2.0 ** -8 + 2.0 ** -18) * want.norm() + (7 * 2.0 ** -13 * s.norm() if x8 else 0)
        assert off <= bound, (tile, part_k, float(off / bound))
    assert len(seen) >= (2 if x8 and which != "down" else 5)


@KINDS
@pytest.mark.parametrize("tokens,experts,top_k,most", [(20000, 512, 8, 0), (13000, 7, 1, 3), (1537, 300, 8, 299)])
def test_layer_of_many_pairs(ops, tokens, experts, top_k, most, x8):
    """Sorted in one launch and, from some ten thousand pairs on, in two; an expert that most tokens take, and ones that nobody takes.  Bounds as above."""
    r = np.random.Generator(np.random.PCG64(tokens))
    h, f = 144, 80
    triple = (*(weights(r, f, h, experts, values=narrow) for _ in range(2)), weights(r, h, f, experts))
    x = activations(r, tokens, h, x8, values=narrow)
    logits = torch.from_numpy(r.standard_normal((tokens, experts)).astype(np.float32)).to(DEV)
    logits[:, most] += 3
    logits[:, experts // 2] = -float("inf")
    how = dict(top_k=top_k, score="sigmoid")
    idx, weight = ops.moe_route(logits, **how)
    want, s = layer_in_64(ops, x, triple, idx, weight)
    off = (ops.moe_ffn(x, logits, triple, **how).double() - want).norm()
    assert off <= (2 * 2.0 ** -8 + 2.0 ** -18) * want.norm() + (7 * 2.0 ** -13 * s.norm() if x8 else 0)


@KINDS
@pytest.mark.parametrize("k", [1024, 2048, 4096, 8192, 11264])
def test_rows_a_power_of_two_apart(ops, k, x8):
    """Where workgroups begin at a k of their own: groups and single matrices, streamed and in tiles, long rows in chunks; on every tile that the rule takes for such rows."""
    r = np.random.Generator(np.random.PCG64(k))
    for m in (1, 7, 16):
        w, x = weights(r, 1290, k, values=narrow), activations(r, m, k, x8, values=narrow)
        check(ops.qlinear(x, w), x64(x), w64(w))
    seen = {"streamed": (9, 40, 1290), "uneven": (9, 71, 130)}
    for e in (2, 9, 33):
        for m in (17, 64, 300, 700, 1501, 4100, 8200):
            for n in (64, 272, 1040, 2064, 8200):
                if m > 8 * e and e * n * k <= 1 << 28 and m * n * k <= 1 << 34:
                    seen.setdefault(pick(m, n, k, e, x8)[0], (e, m, n))
    assert len(seen) >= 7 or k > 4096
    for name, (e, m, n) in seen.items():
        print(name, e, m, n, flush=True)
        w, x = weights(r, n, k, e, values=narrow), activations(r, m, k, x8, values=narrow)
        bounds = [0, *np.sort(r.integers(0, m + 1, e - 1)).tolist(), m]
        check_groups(ops.qgemm_grouped(x, w, torch.tensor(bounds, dtype=torch.int32, device=DEV)), x, w, bounds, cut=False)


@KINDS
@pytest.mark.parametrize("pairs,h,f,e", [(60, 64, 8192, 2), (700, 272, 8192, 2), (2050, 512, 8192, 2), (300, 2048, 4096, 5), (700, 4096, 1024, 9), (66, 1024, 2048, 9)])
def test_layer_of_rows_a_power_of_two_apart(ops, pairs, h, f, e, x8):
    """Down products of that kind in parts of K among them.  Bounds as above."""
    r = np.random.Generator(np.random.PCG64(pairs + h))
    triple = (*(weights(r, f, h, e, values=narrow) for _ in range(2)), weights(r, h, f, e))
    x = activations(r, pairs // 2, h, x8, values=narrow)
    logits = torch.from_numpy(r.standard_normal((pairs // 2, e)).astype(np.float32)).to(DEV)
    want, s = layer_in_64(ops, x, triple, *ops.moe_route(logits, top_k=2))
    off = (ops.moe_ffn(x, logits, triple, top_k=2).double() - want).norm()
    assert off <= (2 * 2.0 ** -8 + 2.0 ** -18) * want.norm() + (7 * 2.0 ** -13 * s.norm() if x8 else 0)


@KINDS
@pytest.mark.parametrize("n", [136, 75])
def test_results_at_any_address(ops, n, x8):
    """Results that begin at any element, from either kernel; what lies around them stays."""
    r = np.random.Generator(np.random.PCG64(n))
    k = 272
    w = weights(r, n, k, 3, values=narrow)
    for m in (5, 40, 300):
        x = activations(r, m, k, x8, values=narrow)
        offsets = torch.tensor([0, m // 3, m - 2, m], dtype=torch.int32, device=DEV)
        for shift in (1, 2, 3, 4, 7):
            room = torch.full((m * n + 16,), 5.0, dtype=torch.bfloat16, device=DEV)
            y = room[shift:shift + m * n].view(m, n)
            assert ops.qgemm(x, w.expert(1), out=y) is y
            check(y, x64(x), w64(w.expert(1)))
            assert ops.qgemm_grouped(x, w, offsets, out=y) is y
            check_groups(y, x, w, offsets.tolist(), cut=False)
            assert bool((room[:shift] == 5).all()) and bool((room[shift + m * n:] == 5).all())


@KINDS
def test_workspace_is_a_choice(ops, x8):
    """The C entry with all the workspace it asks for, with less and with none; beyond its bytes nothing is written."""
    from chadslab_amd import _lib

    lib = _lib.load()
    asked = 0
    for m, n, k in ((17, 17, 4112), (40, 200, 8208), (100, 1040, 14352), (300, 130, 8208), (2050, 17, 4112)):
        r = np.random.Generator(np.random.PCG64(m))
        qw, x = weights(r, n, k, values=narrow), activations(r, m, k, x8, values=narrow)
        need = lib.chadq_product_fp8_workspace_bytes(m, n, k, x8)
        asked += need > 0
        for given in {need, max(0, need - 4), 0}:
            ws = torch.full((need + 256,), 77, dtype=torch.uint8, device=DEV)
            y = torch.full((m + 1, n), 5.0, dtype=torch.bfloat16, device=DEV)
            xs = x.scale.data_ptr() if x8 else None
            assert lib.chadq_product_fp8(x.w.data_ptr() if x8 else x.data_ptr(), xs, qw.w.data_ptr(), qw.scale.data_ptr(), y.data_ptr(), 1, m, n, k,
                                         ws.data_ptr() if given else None, given, torch.cuda.current_stream().cuda_stream) == 0
            check(y[:m], x64(x), w64(qw))
            assert bool((y[m] == 5).all()) and bool((ws[given:] == 77).all())
    assert asked >= 3


def bytes_of(*shape):
    """Values of both signs from 1 to 15 (exact in any sum here), made on the GPU."""
    b = torch.randint(0x38, 0x38 + 32, shape, dtype=torch.uint8, device=DEV)
    return b.bitwise_or_(torch.randint(0, 2, shape, dtype=torch.uint8, device=DEV) << 7).view(FP8)


def some(*shape):
    return torch.rand(shape, device=DEV) * 0.01 + 0.001


@KINDS
@pytest.mark.parametrize("m", [3, 40])
def test_weights_beyond_32_bits(ops, m, x8):
    from chadslab_amd import QRowsFP8, QWeightFP8

    torch.manual_seed(m)
    n, k = 70001, 65552
    qw = QWeightFP8(bytes_of(n, k), some(blocks(n), blocks(k)))
    x = QRowsFP8(bytes_of(m, k), some(m, blocks(k))) if x8 else torch.randn(m, k, device=DEV).bfloat16()
    y = ops.qlinear(x, qw)
    for n0 in (0, 65408, 65536, 69888):  # (whole blocks of rows: 65520 rows are 2^32 bytes)
        part = QWeightFP8(qw.w[n0:n0 + 128], qw.scale[n0 // 128:n0 // 128 + 1])
        check(y[:, n0:n0 + 128], x64(x), w64(part))


@KINDS
@pytest.mark.parametrize("rows", [130, 1500])
def test_experts_beyond_32_bits(ops, rows, x8):
    from chadslab_amd import QExpertsFP8, QRowsFP8

    torch.manual_seed(rows)
    e, n, k = 66, 8208, 8208
    w = QExpertsFP8(bytes_of(e, n, k), some(e, blocks(n), blocks(k)))
    x = QRowsFP8(bytes_of(rows, k), some(rows, blocks(k))) if x8 else torch.randn(rows, k, device=DEV).bfloat16()
    bounds = [rows * i // e for i in range(e + 1)]
    y = ops.qgemm_grouped(x, w, torch.tensor(bounds, dtype=torch.int32, device=DEV))
    for i in (0, 62, 64, 65):
        check(y[bounds[i]:bounds[i + 1]], x64(rows_of(x, slice(bounds[i], bounds[i + 1]))), w64(w.expert(i)))


@KINDS
def test_results_beyond_32_bits(ops, x8):
    """More than 2^31 elements: rows whose results begin behind 2^32 bytes; and activations as large."""
    from chadslab_amd import QRowsFP8, QWeightFP8

    torch.manual_seed(1)
    for m, n, k in ((70001, 32784, 32), (70001, 48, 65552)):
        qw = QWeightFP8(bytes_of(n, k), some(blocks(n), blocks(k)))
        x = QRowsFP8(bytes_of(m, k), some(m, blocks(k))) if x8 else torch.randint(-8, 9, (m, k), dtype=torch.int8, device=DEV).bfloat16()
        y = ops.qlinear(x, qw)
        for m0 in (0, 32760, 65500, 69900):
            rows = slice(m0, m0 + 101)
            check(y[rows], x64(rows_of(x, rows)), w64(qw))
        del x, y


@pytest.mark.parametrize("rows", [True, False])
def test_quantise_beyond_32_bits(ops, rows):
    torch.manual_seed(2)
    n, k = 70016, 65552
    x = torch.randint(-127, 128, (n, k), dtype=torch.int8, device=DEV).bfloat16()
    q = ops.quantize_fp8(x, rows=rows)
    for n0 in (0, 32640, 65408, 65536, 69888):
        part = ops.quantize_fp8(x[n0:n0 + 128].contiguous(), rows=rows)
        at = slice(n0, n0 + 128) if rows else slice(n0 // 128, n0 // 128 + 1)
        assert torch.equal(q.w.view(torch.uint8)[n0:n0 + 128], part.w.view(torch.uint8)) and torch.equal(q.scale[at], part.scale)
    del x
    y = ops.dequantize(q)
    for n0 in (0, 65408, 69888):
        s = q.scale[n0:n0 + 128] if rows else q.scale[n0 // 128:n0 // 128 + 1]
        assert torch.equal(y[n0:n0 + 128], q.w[n0:n0 + 128].float() * s.repeat_interleave(128, 1)[:, :k])


def test_two_threads(ops):
    """Two threads of the interpreter, each on a stream of its own, the same weights: what each gets is what it gets alone."""
    r = np.random.Generator(np.random.PCG64(4))
    triple = tuple(weights(r, *s, 16) for s in ((320, 256), (320, 256), (256, 320)))
    qw = weights(r, 300, 8208)
    xs = [activations(r, 60, 256, False) for _ in range(2)]
    longs = [activations(r, 40, 8208, False) for _ in range(2)]
    zs = [torch.from_numpy(r.standard_normal((60, 16)).astype(np.float32)).to(DEV) for _ in range(2)]

    def calls(i):
        return (ops.moe_ffn(xs[i], zs[i], triple, top_k=4, score="sigmoid", groups=4, top_groups=2), ops.moe_ffn(ops.quantize_fp8(xs[i]), zs[i], triple, top_k=2),
                ops.qlinear(longs[i], qw), ops.qlinear(ops.quantize_fp8(longs[i]), qw))

    want = [calls(i) for i in range(2)]
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got[i].append(calls(i))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert all(len(g) == 10 for g in got)
    assert all(torch.equal(a, b) for i in range(2) for turn in got[i] for a, b in zip(turn, want[i]))


@pytest.mark.parametrize("h", [16, 48, 240, 256, 272, 1008, 1024, 1040, 1104, 2064, 3088])
@pytest.mark.parametrize("tokens,top_k", [(1, 1), (3, 2), (301, 3)])
def test_weighted_sum_of_every_width(ops, tokens, top_k, h):
    """The layer's last step deals columns to threads by their number: widths at its borders.  Bounds as above."""
    r = np.random.Generator(np.random.PCG64(h + tokens))
    triple = (*(weights(r, 32, h, 4, values=narrow) for _ in range(2)), weights(r, h, 32, 4))
    x = activations(r, tokens, h, False, values=narrow)
    logits = torch.from_numpy(r.standard_normal((tokens, 4)).astype(np.float32)).to(DEV)
    want, _ = layer_in_64(ops, x, triple, *ops.moe_route(logits, top_k=top_k, score="sigmoid"))
    off = (ops.moe_ffn(x, logits, triple, top_k=top_k, score="sigmoid").double() - want).norm()
    assert off <= (2 * 2.0 ** -8 + 2.0 ** -18) * want.norm()


def test_weighted_sum_of_very_many_tokens(ops):
    """More tokens than a grid has workgroups for: they repeat, and so does the result."""
    r = np.random.Generator(np.random.PCG64(9))
    for h in (16, 256):
        triple = (*(weights(r, 16, h, 2) for _ in range(2)), weights(r, h, 16, 2))
        x = activations(r, 4096, h, False).repeat(257, 1)
        logits = torch.from_numpy(r.standard_normal((4096, 2)).astype(np.float32)).to(DEV).repeat(257, 1)
        y = ops.moe_ffn(x, logits, triple, top_k=1)
        assert bool(y.any()) and torch.equal(y, y[:4096].repeat(257, 1))


@KINDS
@pytest.mark.parametrize("more", ["bytes", "pairs"])
def test_layer_of_more_tokens_than_go_together(ops, more, x8):
    """Just past 2^31 bytes of activations, or 2^20 pairs: the layer is its two halves', bit for bit, and those are tested above."""
    r = np.random.Generator(np.random.PCG64(12))
    h, f, e, top_k, tokens = (4096, 32, 4, 1, 2 ** 31 // (4096 if x8 else 8192) + 5) if more == "bytes" else (64, 48, 12, 8, 2 ** 17 + 5)
    triple = (*(weights(r, f, h, e) for _ in range(2)), weights(r, h, f, e))
    some = activations(r, 4099, h, x8)
    x = rows_of(some, torch.arange(tokens, device=DEV) % 4099)
    logits = torch.from_numpy(r.standard_normal((tokens, e)).astype(np.float32)).to(DEV)
    half = (tokens + 1) // 2
    y = ops.moe_ffn(x, logits, triple, top_k=top_k, score="sigmoid")
    for part in (slice(0, half), slice(half, tokens)):
        assert torch.equal(y[part], ops.moe_ffn(rows_of(x, part), logits[part], triple, top_k=top_k, score="sigmoid"))
    assert bool(y.any(1).all())
