"""The MXFP4 operators at the ends of the ranges that they take, on the GPU."""
import numpy as np
import pytest
import torch

import ruquant_amd as rq

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
