"""CPU-side checks of the int8 product, the sort and the products grouped by expert: the library exports what the header declares, its
host queries and refusals need no GPU, the Python calls refuse what they do not take, and the definition that the GPU tests compare with agrees with
a second one."""
import fractions
import os
import re

import numpy as np
import pytest
import torch

import ruquant_amd as rq
from ruquant_amd.lib import PROTOTYPES
from tests import i8_oracle as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PTR = 1 << 20   # an aligned address that nothing is read from: the calls are refused first
UNSUPPORTED, WORKSPACE, BAD = -1, -2, -3
F32, F16, BF16, I8 = 0, 1, 2, 3


def test_library_exports_every_declared_symbol():
    text = open(os.path.join(ROOT, "include", "rq_i8.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    names = sorted(set(re.findall(r"\b(rq_\w+)\s*\(", text)))
    assert len(names) == 10
    L = rq.load_library()
    for name in names:
        assert hasattr(L, name) and name in PROTOTYPES, name


def test_sizes():
    L = rq.load_library()
    size = L.rq_weight_prepared_bytes
    assert 5120 * 5120 <= size(I8, 1, 5120, 5120) <= 5120 * 5124 + 4096 and size(BF16, 1, 5120, 5120) == 2 * 5120 * 5120
    assert size(I8, 7, 100, 96) == 7 * size(I8, 1, 100, 96) and size(I8, 1, 1, 1) % 256 == 0
    for bad in ((F32, 1, 64, 64), (4, 1, 64, 64), (I8, 0, 64, 64), (I8, 1, 0, 64), (I8, 1, 64, 0), (I8, 1, 64, 131072), (I8, 1025, 64, 64),
                (I8, 1, -1, 64), (F16, 1, 64, -1), (I8, 1, 2 ** 24 + 1, 64)):
        assert size(*bad) == 0, bad
    ws = L.rq_i8_workspace_bytes
    assert ws(5120, 64, 1) == ws(5120, 17408, 2) == 256 and ws(5120, 64, 3) > 3 * 5120   # (256: not looked at)
    assert ws(5120, 64, 2048) >= 2048 * 5124 and ws(5120, 64, -1) == 0 and ws(0, 64, 1) == 0 and ws(64, 64, 2 ** 22 + 1) == 0
    sort = L.rq_sort_workspace_bytes
    assert sort(1, 8, 64) == 0 and sort(16384, 8, 256) > 0
    for bad in ((-1, 8, 64), (1, 0, 64), (1, 8, 0), (1, 8, 1025), (1, 1025, 8), (2 ** 22, 2, 8)):
        assert sort(*bad) == 0, bad
    group = L.rq_grouped_workspace_bytes
    assert group(I8, 64, 5120, 1280, 2048, 16384) >= 2048 * 5124 and group(I8, 64, 5120, 1280, 1, 8) == group(BF16, 64, 5120, 1280, 9, 72) == 256
    for bad in ((F32, 8, 64, 64, 1, 1), (I8, 1025, 64, 64, 1, 1), (I8, 8, 64, 64, 2 ** 22 + 1, 1), (I8, 8, 64, 64, 1, 2 ** 22 + 1),
                (I8, 8, 64, 64, -1, 1), (I8, 8, 64, 64, 1, -1)):
        assert group(*bad) == 0, bad


def test_workspaces_grow():
    """so that the most tokens' workspace serves every call"""
    L = rq.load_library()
    tokens = list(range(1, 300)) + list(range(300, 9000, 97))
    for K, N in ((1, 1), (33, 64), (4096, 100), (5120, 17408), (17408, 64), (17408, 5120), (131071, 700)):
        sizes = [L.rq_i8_workspace_bytes(K, N, M) for M in tokens]
        assert all(a <= b for a, b in zip(sizes, sizes[1:])) and sizes[0] > 0, (K, N)
        for kind in (I8, F16, BF16):
            for fixed in (1, 100, 5000):
                for sizes in ([L.rq_grouped_workspace_bytes(kind, 9, K, N, M, fixed) for M in tokens],
                              [L.rq_grouped_workspace_bytes(kind, 9, K, N, fixed, P) for P in tokens]):
                    assert all(a <= b for a, b in zip(sizes, sizes[1:])) and sizes[0] > 0, (K, N, kind)
    for E in (1, 60, 1024):
        sizes = [L.rq_sort_workspace_bytes(M, 8, E) for M in tokens + [20000, 100000, 2 ** 19]]
        assert all(a <= b for a, b in zip(sizes, sizes[1:]))


def test_refusals_without_a_gpu():
    L = rq.load_library()
    quantize = lambda dtype=F32, x=PTR, ldx=64, M=2, K=64, codes=PTR, scales=PTR: L.rq_i8_quantize(dtype, x, ldx, M, K, codes, scales, None)  # noqa: E731
    assert quantize(dtype=I8) == quantize(dtype=-1) == quantize(K=0) == quantize(M=-1) == quantize(K=2 ** 30 + 1) == UNSUPPORTED
    assert quantize(x=None) == quantize(x=PTR + 2) == quantize(ldx=63) == quantize(codes=None) == quantize(scales=None) == quantize(scales=PTR + 2) == BAD
    assert quantize(M=0, x=None) == 0
    back = lambda dtype=F32, codes=PTR, scales=PTR, M=2, K=64, out=PTR, ldo=64: L.rq_i8_dequantize(dtype, codes, scales, M, K, out, ldo, None)  # noqa: E731
    assert back(dtype=I8) == back(K=0) == back(M=-1) == UNSUPPORTED
    assert back(codes=None) == back(scales=None) == back(scales=PTR + 1) == back(out=PTR + 2) == back(ldo=63) == BAD
    prepare = lambda kind=I8, w=PTR, scales=PTR, E=1, N=64, K=64, to=PTR, n=1 << 20: L.rq_weight_prepare(kind, w, scales, E, N, K, to, n, None)  # noqa: E731
    assert prepare(kind=F32) == prepare(E=0) == prepare(K=131072) == UNSUPPORTED
    assert prepare(scales=None) == prepare(kind=F16) == prepare(w=None) == prepare(to=PTR + 16) == prepare(kind=F16, w=PTR + 1, scales=None) == BAD
    assert prepare(n=16) == WORKSPACE
    product = lambda w=PTR, K=64, N=64, dtype=F32, x=PTR, ldx=64, xs=None, M=2, out=F32, y=PTR, ldy=64, ws=PTR, n=1 << 20: L.rq_i8_mul_mat(  # noqa: E731
        w, K, N, dtype, x, ldx, xs, M, out, y, ldy, ws, n, None)
    assert product(dtype=4) == product(out=I8) == product(K=131072) == product(N=0) == product(M=-1) == product(M=2 ** 22 + 1) == UNSUPPORTED
    assert product(w=None) == product(w=PTR + 128) == product(x=None) == product(x=PTR + 2) == product(xs=PTR) == product(dtype=I8) == BAD
    assert product(dtype=I8, xs=PTR + 2) == product(ldx=63) == product(ldy=63) == product(y=None) == product(out=F16, y=PTR + 1) == BAD
    assert product(M=40, ws=None) == product(M=40, ws=PTR + 8) == product(M=40, n=16) == WORKSPACE
    assert product(M=0, x=None, ws=None) == 0
    sort = lambda ids=PTR, M=2, top=4, E=8, offsets=PTR, slots=PTR, tokens=PTR, ws=None, n=0: L.rq_sort_slots(  # noqa: E731
        ids, M, top, E, offsets, slots, tokens, ws, n, None)
    assert sort(M=-1) == sort(top=0) == sort(E=0) == sort(E=1025) == sort(M=2 ** 22) == UNSUPPORTED
    assert sort(ids=None) == sort(offsets=None) == sort(slots=None) == sort(tokens=PTR + 2) == sort(ids=PTR + 1) == BAD
    assert sort(M=16384, top=8) == sort(M=16384, top=8, ws=PTR + 8, n=1 << 20) == sort(M=16384, top=8, ws=PTR, n=8) == WORKSPACE
    group = lambda kind=I8, w=PTR, E=4, K=64, N=64, dtype=F32, x=PTR, ldx=64, xs=None, M=8, offsets=PTR, P=8, rows=None, places=None, out=F32, y=PTR, ldy=64, Y=8, ws=PTR, n=1 << 20: (  # noqa: E501,E731
        L.rq_grouped_mul_mat(kind, w, E, K, N, dtype, x, ldx, xs, M, offsets, P, rows, places, out, y, ldy, Y, ws, n, None))
    assert group(kind=F32) == group(dtype=4) == group(kind=F16) == group(kind=F16, dtype=BF16) == group(kind=F16, dtype=I8) == UNSUPPORTED
    assert group(E=1025) == group(P=2 ** 22 + 1) == group(M=-1) == group(out=I8) == group(Y=-1) == group(Y=2 ** 31) == UNSUPPORTED
    assert group(w=None) == group(x=None) == group(M=0) == group(offsets=None) == group(offsets=PTR + 2) == group(rows=PTR + 1) == BAD
    assert group(places=PTR + 2) == group(xs=PTR) == group(dtype=I8) == group(ldx=63) == group(ldy=63) == group(y=None) == group(w=PTR + 16) == BAD
    assert group(P=40, ws=None) == group(P=40, n=16) == group(P=40, ws=PTR + 64) == group(kind=F16, dtype=F16, P=40, ws=None) == WORKSPACE
    assert group(P=0, x=None) == group(Y=0, y=None) == 0


def test_python_refusals_without_a_gpu():
    x = torch.zeros((2, 64))
    for call in (lambda: rq.i8_quantize(x), lambda: rq.i8_dequantize(x.to(torch.int8), x[:, 0]), lambda: rq.I8Weight(x.to(torch.int8), x[:, 0]),
                 lambda: rq.HalfWeight(x.half()), lambda: rq.sort_slots(x.int(), 4)):
        with pytest.raises(rq.RqError):
            call()


@pytest.mark.parametrize("seed", range(4))
def test_oracle_agrees_with_exact_fractions(seed):
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((3, 20)) * 2.0 ** rng.integers(-30, 30)).astype(np.float32).astype(np.float64)
    codes, scales = ref.quantize(x)
    for m in range(3):
        largest = max(abs(fractions.Fraction(v)) for v in x[m])
        # (1 / 127 as an fp32 number is 2^-28 off, and its product rounded once)
        assert abs(fractions.Fraction(float(scales[m])) * 127 / largest - 1) <= fractions.Fraction(1, 2 ** 23)
        r = fractions.Fraction(float(np.float32(1) / scales[m]))
        for v, c in zip(x[m], codes[m]):
            assert c == round(fractions.Fraction(v) * r)   # (ties to even)
    ids = rng.integers(-1, 7, size=(5, 3)).astype(np.int32)
    offsets, slots, tokens = ref.sort(ids, 6)
    flat = ids.reshape(-1).tolist()
    assert slots.tolist() == [i for e in range(6) for i in range(15) if flat[i] == e] + [i for i in range(15) if not 0 <= flat[i] < 6]
    assert offsets.tolist() == [sum(0 <= v < e for v in flat) for e in range(7)] and tokens.tolist() == [i // 3 for i in slots]


def test_plans():
    """few rows stream the weight, many go in tiles; what is refused has no plan"""
    import ctypes
    L = rq.load_library()

    def plan(fn, *a):
        p = (ctypes.c_int64 * 8)()
        return fn(*a, p) or list(p)

    product, group = L.rq_i8_product_plan, L.rq_grouped_plan
    assert plan(product, 5120, 17408, BF16, 1)[0] == 1 and plan(product, 5120, 17408, I8, 1)[0] == 2 and plan(product, 5120, 17408, BF16, 16)[0] == 2
    main = plan(product, 5120, 17408, BF16, 2048)
    assert main[0] == 3 and main[1:4] == [256, 256, 64] and main[4] > 0
    assert plan(product, 17408, 512, I8, 64)[6] > 1   # (few tiles of long rows: shared)
    assert plan(group, I8, 64, 5120, 1280, BF16, 1, 8)[:2] == [1, 8]
    assert plan(group, BF16, 64, 5120, 1280, BF16, 2048, 16384)[:3] == [3, 256, 256]
    assert product(0, 64, F32, 1, None) == BAD and plan(product, 0, 64, F32, 1) == plan(product, 64, 64, 4, 1) == plan(product, 64, 64, F32, 0) == UNSUPPORTED
    assert plan(group, BF16, 8, 64, 64, F16, 1, 1) == plan(group, I8, 1025, 64, 64, F32, 1, 1) == plan(group, I8, 8, 64, 64, F32, 1, 0) == UNSUPPORTED
