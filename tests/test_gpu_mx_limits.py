"""The MXFP4 operators at the ends of the ranges that they take, on the GPU."""
import numpy as np
import pytest
import torch

import ruquant_amd as rq
from tests import mx_oracle as ref
from tests import mx_plan_util as plans

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_route_of_more_tokens_than_a_launch_has():
    """2^26 tokens and some, 64 threads each, are more than the 2^32 threads of a launch"""
    M = 2 ** 26 + 5
    logits = torch.randint(-3, 4, (M, 2), device=DEV, dtype=torch.int8).half()
    ids, w = rq.route(logits, 1, renormalize=False)
    first = logits[:, 0] >= logits[:, 1]   # (ties to the lowest index)
    assert torch.equal(ids[:, 0] == 0, first) and bool(((ids == 0) | (ids == 1)).all())
    few = 4096
    for at in (0, 2 ** 25 - few // 2, 2 ** 26 - few // 2, M - few):
        part = rq.route(logits[at:at + few], 1, renormalize=False)
        assert torch.equal(part[0], ids[at:at + few]) and torch.equal(part[1], w[at:at + few])


def _weight(E, N, K, g):
    return rq.MXWeight(torch.empty((E, N, K // 2), dtype=torch.uint8, device=DEV).random_(0, 256, generator=g),
                       torch.empty((E, N, K // 32), dtype=torch.uint8, device=DEV).random_(115, 119, generator=g))


@pytest.fixture
def room():
    """These calls' workspaces are some ten gigabytes."""
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 120e9:
        pytest.skip("120 GB of free memory")
    yield
    torch.cuda.empty_cache()


def test_experts_of_more_slots_and_inputs_than_a_grid_is_wide(room):
    """2^22 slots of 2^15 inputs are rounded by 2^32 threads; each token's row as with few others"""
    M, top, K, F, N = 2 ** 17, 32, 2 ** 15, 32, 4
    g = torch.Generator(device=DEV).manual_seed(1)
    gate, up, down = _weight(1, F, K, g), _weight(1, F, K, g), _weight(1, N, F, g)
    x = torch.randn((M, K), device=DEV, dtype=torch.float16, generator=g)
    ids, w = torch.zeros((M, top), dtype=torch.int32, device=DEV), torch.rand((M, top), device=DEV, generator=g)
    y = rq.expert_ffn(gate, up, down, x, ids, w)
    assert bool(torch.isfinite(y).all()) and bool(y.any())
    for at in (0, M // 2 - 50, M - 100):
        assert torch.equal(rq.expert_ffn(gate, up, down, x[at:at + 100], ids[at:at + 100], w[at:at + 100]), y[at:at + 100])


def test_experts_of_more_tiles_than_a_grid_is_wide(room):
    """1040 tiles of tokens x 2^14 of rows, 256 threads each, are more than 2^32; each token's row as in calls of a quarter"""
    E, M, top, K, F, N = 416, 1248, 32, 32, 2 ** 20, 4
    g = torch.Generator(device=DEV).manual_seed(2)
    gate, down = _weight(E, F, K, g), _weight(E, N, F, g)
    x = torch.randn((M, K), device=DEV, dtype=torch.float16, generator=g)
    ids = torch.randn((M, E), device=DEV, generator=g).topk(top, dim=1).indices.int()
    w = torch.rand((M, top), device=DEV, generator=g)
    y = rq.expert_ffn(gate, gate, down, x, ids, w, out=torch.empty((M, N), device=DEV))
    assert bool(torch.isfinite(y).all()) and bool(y.any())
    for at in range(0, M, 312):
        part = slice(at, at + 312)
        assert torch.equal(rq.expert_ffn(gate, gate, down, x[part], ids[part], w[part], out=torch.empty((312, N), device=DEV)), y[part])


def _host_weight(shape, K, seed):
    rng = np.random.default_rng(seed)
    middle = 127 - K.bit_length() // 2
    return (rng.integers(0, 256, size=(*shape, K // 2), dtype=np.uint8),
            rng.integers(middle - 3, middle + 3, size=(*shape, K // 32), dtype=np.uint8))


def _on_gpu(pair):
    return rq.MXWeight(*(torch.from_numpy(a).to(DEV) for a in pair))


def _check_experts(E, K, F, N, M, top, ids, seed):
    mats = [_host_weight((E, F), K, seed), _host_weight((E, F), K, seed + 1), _host_weight((E, N), F, seed + 2)]
    rng = np.random.default_rng(seed)
    x = torch.from_numpy(rng.standard_normal((M, K)).astype(np.float32)).bfloat16()
    w = rng.standard_normal((M, top)).astype(np.float32)
    y = rq.expert_ffn(*(_on_gpu(m) for m in mats), x.to(DEV), torch.from_numpy(ids).to(DEV), torch.from_numpy(w).to(DEV),
                      out=torch.empty((M, N), device=DEV)).double().cpu().numpy()
    want, bound = ref.experts(x.double().numpy(), mats, ids, w, False)
    off = np.abs(y - want)
    bound = bound + 1.01 * 2.0 ** -24 * np.abs(want)
    assert (off <= bound).all(), "off by %g times the bound" % (off[bound > 0] / bound[bound > 0]).max()


@pytest.mark.parametrize("E,top", [(65, 8), (256, 8), (300, 5), (1024, 32)])
@pytest.mark.parametrize("M", [1, 4, 50])
def test_many_experts(M, E, top):
    """up to the most; the last one among those that are chosen"""
    rng = np.random.default_rng(E)
    ids = np.stack([rng.permutation(E)[:top] for _ in range(M)]).astype(np.int32)
    ids[M - 1, top - 1] = E - 1
    _check_experts(E, 96, 64, 40, M, top, ids, M)


@pytest.mark.parametrize("top", [7, 8, 9, 16, 17, 31, 32])
@pytest.mark.parametrize("M", [1, 2, 4])
def test_few_tokens_with_many_slots(M, top):
    """more slots of a token than wavefronts that share them out, fewer, and as many; absent ones; the same expert again"""
    E = 40
    rng = np.random.default_rng(top)
    ids = rng.integers(-1, E, size=(M, top)).astype(np.int32)
    _check_experts(E, 288, 352, 100, M, top, ids, M + top)
    _check_experts(E, 288, 352, 100, M, top, np.full((M, top), E - 1, dtype=np.int32), M + top)


@pytest.mark.parametrize("M,K,F", [(1, 65536, 64), (1, 65568, 64), (3, 65568, 64), (1, 64, 65568), (4, 64, 65568), (20, 64, 65568)])
def test_experts_of_long_rows(M, K, F):
    ids = np.random.default_rng(M).integers(0, 3, size=(M, 2)).astype(np.int32)
    _check_experts(3, K, F, 33, M, 2, ids, M)


@pytest.mark.parametrize("M,K,N,kind", [(1, 65536, 33, plans.ALONE), (1, 65568, 33, plans.ROWS), (2, 40000, 100, plans.ROWS), (1, 2 ** 17, 64, plans.ROWS),
                                        (3, 2 ** 17, 64, plans.TILES), (1, 2 ** 20, 40, plans.TILES), (18, 2 ** 20, 40, plans.TILES), (3, 2 ** 20 - 32, 7, plans.TILES)])
def test_products_of_long_rows(M, K, N, kind):
    assert plans.product(K, N, M)[0] == kind
    codes, scales = _host_weight((N,), K, M)
    x = torch.from_numpy(np.random.default_rng(K).standard_normal((M, K)).astype(np.float32)).bfloat16()
    y = rq.mx_mul_mat(_on_gpu((codes, scales)), x.to(DEV), out=torch.empty((M, N), device=DEV)).double().cpu().numpy()
    w = ref.values(codes, scales)
    xq = np.concatenate([ref.values(*ref.quantize(row[None])) for row in x.double().numpy()])
    # (an fp32 sum of K exact products, as in the tests of the product)
    bound = 2 * (K / 32 + 16) * 2.0 ** -24 * (np.abs(xq) @ np.abs(w).T) + 1.01 * 2.0 ** -24 * np.abs(xq @ w.T)
    assert (np.abs(y - xq @ w.T) <= bound).all()


def test_rows_that_are_longer_than_a_products():
    """quantised and taken back: 2^22 + 32 elements"""
    K = 2 ** 22 + 32
    x = torch.from_numpy(np.random.default_rng(5).standard_normal((2, K)).astype(np.float32)).bfloat16()
    codes, scales = rq.mx_quantize(x.to(DEV))
    back = rq.mx_dequantize(codes, scales).cpu()
    for m in range(2):
        want = ref.quantize(x[m:m + 1].double().numpy())
        assert (scales[m].cpu().numpy() == want[1][0]).all() and (back[m].double().numpy() == ref.values(*want)[0]).all()


@pytest.mark.parametrize("E,K,F,N,top", [(40, 288, 352, 100, 3), (256, 544, 96, 65, 8), (3, 416, 160, 300, 1)])
@pytest.mark.parametrize("M", [5, 13, 24])
def test_experts_of_some_tokens_slot_by_slot(M, E, K, F, N, top):
    assert plans.experts(E, K, F, N, M, top)[0] == plans.ALONE
    ids = np.random.default_rng(M).integers(-1, E, size=(M, top)).astype(np.int32)
    _check_experts(E, K, F, N, M, top, ids, M)
