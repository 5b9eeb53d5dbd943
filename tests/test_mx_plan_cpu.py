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


def test_refusals():
    L, p = rq.load_library(), (ctypes.c_int64 * 8)()
    assert L.rq_mx4_product_plan(40, 64, 1, p) == L.rq_mx4_product_plan(64, 64, 0, p) == L.rq_mx4_product_plan(64, 64, 2 ** 22 + 1, p) == -1
    assert L.rq_mx4_experts_plan(0, 64, 64, 64, 1, 1, p) == L.rq_mx4_experts_plan(8, 64, 64, 64, 0, 1, p) == -1
    assert L.rq_mx4_product_plan(64, 64, 1, None) == L.rq_mx4_experts_plan(8, 64, 64, 64, 1, 1, None) == -3
