"""CPU-side checks of the MXFP4 operators: the library exports what the header declares, its host queries and refusals need no GPU, and
the definition that the GPU tests compare with agrees with a second one."""
import os
import re

import numpy as np
import pytest

import ruquant_amd as rq
from ruquant_amd.lib import PROTOTYPES
from tests import mx_oracle as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PTR = 1 << 20   # an aligned address that nothing is read from: the calls are refused first


def test_library_exports_every_declared_symbol():
    text = open(os.path.join(ROOT, "include", "rq_mx4.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    names = sorted(set(re.findall(r"\b(rq_\w+)\s*\(", text)))
    assert len(names) == 9
    L = rq.load_library()
    for name in names:
        assert hasattr(L, name) and name in PROTOTYPES, name


def test_sizes():
    L = rq.load_library()
    size = L.rq_mx4_prepared_bytes
    assert size(1, 5120, 5120) >= 5120 * 5120 * 17 // 32 and size(1, 5120, 5120) % 256 == 0
    assert size(7, 100, 96) == 7 * size(1, 100, 96)
    for bad in ((0, 64, 64), (1, 0, 64), (1, 64, 0), (1, 64, 48), (1, 64, 2 ** 20 + 32), (1, -1, 64)):
        assert size(*bad) == 0, bad
    ws = L.rq_mx4_workspace_bytes
    assert ws(5120, 17408, 2048) > ws(5120, 17408, 32) > ws(5120, 17408, 1) == 256
    assert ws(5120, 17408, -1) == 0 and ws(40, 64, 3) == 0 and ws(64, 64, 2 ** 22 + 1) == 0
    ex = L.rq_mx4_experts_workspace_bytes
    assert ex(64, 5120, 1280, 5120, 2048, 8) > ex(64, 5120, 1280, 5120, 1, 8) > 0
    for bad in ((1025, 64, 64, 64, 1, 1), (8, 64, 48, 64, 1, 1), (8, 64, 64, 64, 1, 33), (8, 64, 64, 64, 1, 0), (8, 64, 64, 64, 2 ** 21, 4)):
        assert ex(*bad) == 0, bad


def test_workspaces_grow_with_the_tokens():
    """so that the most tokens' workspace serves every call"""
    L = rq.load_library()
    tokens = list(range(1, 300)) + list(range(300, 9000, 97))
    for K, N in ((32, 1), (256, 64), (4096, 100), (5120, 17408), (17408, 64), (17408, 5120), (65536, 700)):
        sizes = [L.rq_mx4_workspace_bytes(K, N, M) for M in tokens]
        assert all(a <= b for a, b in zip(sizes, sizes[1:])) and sizes[0] > 0, (K, N)
    for E, K, F, N, top in ((1, 32, 32, 1, 1), (8, 64, 32, 33, 2), (64, 5120, 1280, 5120, 8), (60, 512, 96, 100, 4), (1024, 64, 32, 16, 1)):
        sizes = [L.rq_mx4_experts_workspace_bytes(E, K, F, N, M, top) for M in tokens]
        assert all(a <= b for a, b in zip(sizes, sizes[1:])) and sizes[0] > 0, (E, K, F, N, top)


def test_refusals_without_a_gpu():
    L = rq.load_library()
    bad, unsupported, workspace = -3, -1, -2
    assert L.rq_mx4_quantize(3, PTR, 64, 1, 64, PTR, PTR, None) == unsupported
    assert L.rq_mx4_quantize(0, PTR, 64, 1, 40, PTR, PTR, None) == unsupported
    assert L.rq_mx4_quantize(0, None, 64, 1, 64, PTR, PTR, None) == bad
    assert L.rq_mx4_quantize(0, PTR, 63, 2, 64, PTR, PTR, None) == bad
    assert L.rq_mx4_quantize(0, None, 64, 0, 64, None, None, None) == 0
    assert L.rq_mx4_dequantize(0, PTR, None, 1, 64, PTR, 64, None) == bad
    assert L.rq_mx4_dequantize(-1, PTR, PTR, 1, 64, PTR, 64, None) == unsupported
    assert L.rq_mx4_prepare(PTR + 16, PTR, 1, 64, 64, PTR, 1 << 20, None) == bad
    assert L.rq_mx4_prepare(PTR, PTR, 1, 64, 64, PTR, 16, None) == workspace
    assert L.rq_mx4_mul_mat(PTR, 64, 64, 0, PTR, 64, 40, 0, PTR, 64, None, 0, None) == workspace
    assert L.rq_mx4_mul_mat(PTR, 64, 64, 0, PTR, 64, 40, 0, PTR, 63, PTR, 1 << 20, None) == bad
    assert L.rq_mx4_mul_mat(PTR, 64, 64, 0, PTR + 1, 64, 1, 0, PTR, 64, PTR, 1 << 20, None) == bad
    assert L.rq_mx4_mul_mat(PTR, 65, 64, 0, PTR, 64, 1, 0, PTR, 64, PTR, 1 << 20, None) == unsupported
    route = lambda E=64, scoring=0, groups=1, top_groups=1, top=8, logits=PTR, ids=PTR: L.rq_route(
        0, logits, E, 1, E, scoring, None, groups, top_groups, top, 1, 1.0, ids, PTR, None)
    assert route(E=1025) == route(scoring=2) == route(groups=3) == route(groups=2, top_groups=3) == route(top=65) == unsupported
    assert route(groups=16, top=5) == route(top=0) == route(top=33) == route(E=0) == unsupported
    assert route(logits=None) == route(ids=None) == route(ids=PTR + 2) == bad
    experts = lambda **k: L.rq_mx4_experts(
        k.get("gate", PTR), PTR, PTR, k.get("E", 8), 64, 64, 64, 0, PTR, k.get("ldx", 64), 2, k.get("ids", PTR), PTR, k.get("top", 2), 0, PTR,
        64, k.get("ws", PTR), k.get("n", 1 << 20), None)
    assert experts(gate=None) == experts(ldx=63) == experts(ids=None) == experts(gate=PTR + 64) == bad
    assert experts(E=0) == experts(top=33) == unsupported
    assert experts(ws=None) == experts(n=16) == experts(ws=PTR + 8) == workspace


@pytest.mark.parametrize("seed", range(4))
def test_oracle_agrees_with_an_enumeration(seed):
    """every element the nearest of all 15 values of its block's unit, the unit by repeated halving"""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((3, 64)) * 2.0 ** rng.integers(-30, 30)
    x[1, :4] = [0.0, -0.25, 5.0, 7.5]
    v = ref.values(*ref.quantize(x))
    for m in range(3):
        for b in range(2):
            block = x[m, 32 * b:32 * b + 32]
            unit = 1.0
            while np.abs(block).max() >= 8 * unit:
                unit *= 2
            while 0 < np.abs(block).max() < 4 * unit:
                unit /= 2
            for i, e in enumerate(block):
                away = np.abs(np.concatenate([ref.ELEMENTS, -ref.ELEMENTS]) * unit - e)
                assert abs(v[m, 32 * b + i] - e) == away.min()
