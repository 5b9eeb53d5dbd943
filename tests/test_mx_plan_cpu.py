"""Which form an MXFP4 call takes, without a GPU: the shapes that the GPU tests mean a form by reach it."""
import ctypes

import pytest

import ruquant_amd as rq
from tests import mx_plan_util as plans


@pytest.mark.parametrize("K,N,M,tiles,behind", plans.PRODUCTS)
def test_products_in_tiles(K, N, M, tiles, behind):
    kind, form, rest, first, splits = plans.product(K, N, M)
    assert (kind, form, rest, splits) == (plans.TILES, tiles, behind, 1)
    assert first < N if rest[0] else first >= N


def test_every_form_of_the_tiles_is_meant():
    """six forms as the first, and all sizes of tiles behind another"""
    assert len({p[3] for p in plans.PRODUCTS}) == 6
    assert {p[4] for p in plans.PRODUCTS} == {(0, 0), (64, 64), (128, 64), (128, 128), (128, 256), (256, 256)}
    assert {p[6] for p in plans.EXPERTS} == {(128, 64), (128, 128), (256, 128)}


@pytest.mark.parametrize("K,N,M", plans.SHARED)
def test_shared_tiles(K, N, M):
    kind, form, rest, _, splits = plans.product(K, N, M)
    assert kind == plans.TILES and form == (64, 64, 2) and rest == (0, 0) and splits > 1


@pytest.mark.parametrize("K,N,M,kind", [(5120, 5120, 1, plans.ALONE), (17408, 5120, 3, plans.ROWS), (1024, 17408, 16, plans.ROWS), (5120, 5120, 17, plans.TILES),
                                        (2 ** 17, 64, 1, plans.ROWS), (2 ** 20, 40, 1, plans.TILES)])
def test_few_tokens(K, N, M, kind):
    assert plans.product(K, N, M)[0] == kind


@pytest.mark.parametrize("E,K,F,N,M,top,tiles", plans.EXPERTS)
def test_experts_in_tiles(E, K, F, N, M, top, tiles):
    assert plans.experts(E, K, F, N, M, top) == (plans.TILES, tiles)


@pytest.mark.parametrize("E,K,F,N,top,slots,tiles", [
    (64, 5120, 1280, 5120, 8, (1, 4, 6), (12, 24)), (8, 5120, 1280, 5120, 8, (1, 2), (4, 8)), (64, 5120, 1280, 5120, 32, (1,), (3, 4)),
    (256, 2048, 512, 2048, 8, (1, 8, 24), (25,)), (8, 2048, 512, 2048, 8, (1, 8), (16, 24)), (8, 4096, 4096, 4096, 2, (1, 3), (8, 16)),
    (32, 1024, 256, 1024, 4, (1, 24), (25,)), (4, 5120, 17408, 5120, 2, (1,), (3, 8)), (24, 768, 192, 768, 12, (1, 16), (24,)),
    (16, 4096, 704, 1024, 1, (1, 24), ()), (2, 65568, 64, 64, 1, (), (1, 2))])
def test_experts_slot_by_slot_or_in_tiles(E, K, F, N, top, slots, tiles):
    """numbers of tokens for which one of the two was measured clearly the faster; from the first one in tiles on, every one is"""
    for M in slots:
        assert plans.experts(E, K, F, N, M, top)[0] == plans.ALONE, M
    for M in tiles:
        assert plans.experts(E, K, F, N, M, top)[0] == plans.TILES, M
    kinds = [plans.experts(E, K, F, N, M, top)[0] for M in range(1, 60)]
    assert kinds == sorted(kinds)


def test_experts_workspaces_grow_over_the_change_of_form():
    L = rq.load_library()
    for E, K, F, N, top in ((64, 5120, 1280, 5120, 8), (8, 5120, 1280, 5120, 8), (256, 2048, 512, 2048, 8), (1, 32, 65536, 1, 1), (1024, 64, 32, 16, 32), (2, 32, 32, 1, 32),
                            (4, 5120, 17408, 5120, 2), (1, 65536, 32, 1, 32)):
        sizes = [L.rq_mx4_experts_workspace_bytes(E, K, F, N, M, top) for M in range(1, 60)]
        assert all(a <= b for a, b in zip(sizes, sizes[1:])) and sizes[0] > 0, (E, K, F, N, top)


def test_refusals():
    L, p = rq.load_library(), (ctypes.c_int64 * 8)()
    assert L.rq_mx4_product_plan(40, 64, 1, p) == L.rq_mx4_product_plan(64, 64, 0, p) == L.rq_mx4_product_plan(64, 64, 2 ** 22 + 1, p) == -1
    assert L.rq_mx4_experts_plan(0, 64, 64, 64, 1, 1, p) == L.rq_mx4_experts_plan(8, 64, 64, 64, 0, 1, p) == -1
    assert L.rq_mx4_product_plan(64, 64, 1, None) == L.rq_mx4_experts_plan(8, 64, 64, 64, 1, 1, None) == -3
