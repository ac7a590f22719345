"""Which tile a product on FP8 weights takes, and K in how many parts: the rule by size, asked directly on the host (a C++ function of libchadq.so).  No GPU."""
import ctypes

import pytest

from chadslab_amd import _lib

TILES = ["64x32", "64x64", "128x64", "128x64P", "256x64", "256x64P", "128x128", "128x128P", "256x128", "256x256"]
P, I, B = ctypes.c_void_p, ctypes.c_int, ctypes.c_bool


class Product(ctypes.Structure):
    _fields_ = [*((n, P) for n in ("x", "xs", "w", "ws", "y", "offsets")), *((n, I) for n in "MNKE"), ("y_bf16", B), ("clear_rest", B), ("rows", P), ("x_rows", I),
                ("w2", P), ("w2s", P), ("h8", P), ("h8s", P), ("part_k", I)]


class Pick(ctypes.Structure):
    _fields_ = [("tile", I), ("part_k", I)]


def pick(m, n, k, experts=1, x8=False, gated=False, most_parts=1):
    """-> (tile, k of a part or 0)"""
    fn = _lib.load()["_ZN5chadq13fp8_tile_pickERKNS_10Fp8ProductEi"]
    fn.restype, fn.argtypes = Pick, [ctypes.POINTER(Product), I]
    r = fn(ctypes.byref(Product(M=m, N=n, K=k, E=experts, xs=x8 or None, offsets=experts > 1 or None, w2=gated or None)), most_parts)
    return TILES[r.tile], r.part_k


MS = (17, 33, 64, 100, 129, 200, 300, 513, 700, 1000, 1501, 2050, 4100, 6000, 8200)
NS = (17, 64, 130, 272, 520, 1040, 2064, 4112, 8200, 14336)
KS = (16, 80, 144, 272, 528, 1040, 2064, 4112, 8208)
DENSE, GROUPED, DOWN = {1: 8}, {2: 1, 5: 1, 9: 1, 33: 1}, {2: 4, 5: 4, 9: 4, 33: 4}  # experts: parts of K at most


def sizes(forms, most=1 << 35):
    """Products of a form from the least work on: more rows than are streamed, weights of at most 2^29 bytes."""
    every = [(m, n, k, e) for e in forms for m in MS for n in NS for k in KS if m > 16 and (e == 1 or m > 8 * e) and e * n * k <= 1 << 29 and m * n * k <= most]
    return sorted(every, key=lambda s: s[0] * s[1] * s[2] + 100 * s[3] * s[1] * s[2] + 100 * s[0] * s[1])


def first_of_each(forms, x8, gated=False):
    """{(tile, in parts): the smallest (m, n, k, experts)}"""
    found = {}
    for m, n, k, e in sizes(forms):
        tile, part_k = pick(m, n, k, e, x8, gated, forms[e])
        found.setdefault((tile, part_k > 0), (m, n, k, e))
    return found


@pytest.mark.parametrize("x8", [False, True], ids=["bf16", "fp8"])
def test_every_tile_is_somebodys(x8):
    absent = {"256x64P"} if x8 else {"256x256"}
    assert {t for t, _ in first_of_each(DENSE, x8)} | {t for t, _ in first_of_each(GROUPED, x8)} == set(TILES) - absent
    gated = {"256x64", "256x128"} if x8 else {"128x64", "128x64P", "256x64", "256x64P", "128x128P", "256x128"}
    assert {t for t, _ in first_of_each(GROUPED, x8, True)} == gated


@pytest.mark.parametrize("x8", [False, True], ids=["bf16", "fp8"])
def test_parts_of_k(x8):
    """Whole 1024s, none of them empty, at most as many as asked for; none for few k."""
    seen = set()
    for forms in (DENSE, DOWN):
        for m, n, k, e in sizes(forms):
            tile, part_k = pick(m, n, k, e, x8, False, forms[e])
            if part_k:
                parts = -(-k // part_k)
                assert part_k % 1024 == 0 and 2 <= parts <= forms[e], (m, n, k, e)
                seen.add(parts)
            assert k > 1024 or not part_k
            assert pick(m, n, k, e, x8)[1] == 0
    assert len(seen) >= 2


def test_measured_choices():
    """Large products and long sums."""
    assert pick(4096, 14336, 4096, x8=True, most_parts=8) == ("256x256", 0)
    assert pick(17, 4096, 4096, x8=True, most_parts=8)[0] == "64x32"
    assert pick(8192, 8192, 8192, x8=True, most_parts=8) == ("256x256", 0)
    assert pick(1000, 4096, 14336, most_parts=8) == ("128x128", 0)


class CombineShape(ctypes.Structure):
    _fields_ = [("flat", I), ("threads", I), ("items", ctypes.c_int64)]


def test_weighted_sum_leaves_few_threads_idle():
    """The last step of a layer of experts: whatever the width, every column has a thread, and more than half of the threads have columns."""
    fn = _lib.load()["_ZN5chadq17moe_combine_shapeEii"]
    fn.restype, fn.argtypes = CombineShape, [I, I]
    for h in [*range(16, 4400, 16), 7168, 8192, 1 << 20]:
        s = fn(4000, h)
        quads = 4000 * (h // 4)
        assert s.threads % 64 == 0 and s.threads <= 256 and s.items * s.threads >= quads and (s.flat or s.threads * (s.items // 4000) >= h // 4), h
        assert quads > s.items * s.threads // 2, h


@pytest.mark.parametrize("x8", [0, 1])
def test_layers_of_very_many_tokens_go_in_ranges(x8):
    """Activations of 2 GB and more, and more than 2^20 pairs: equal ranges, whose workspace is the call's."""
    need = _lib.load().chadq_moe_ffn_fp8_workspace_bytes
    for h, f, e, top_k in ((4096, 64, 4, 1), (7168, 2048, 8, 2), (16, 16, 2, 1), (256, 128, 256, 8)):
        most = min((2 ** 31 - 2) // (h * (1 if x8 else 2)), 2 ** 20 // top_k)
        assert need(most, h, f, e, top_k, x8) >= most * top_k * h * 4
        for t in (most + 1, 2 * most, 2 * most + 1, 5 * most + 3):
            ranges = -(-t // most)
            assert need(t, h, f, e, top_k, x8) == need(-(-t // ranges), h, f, e, top_k, x8), (t, h)
