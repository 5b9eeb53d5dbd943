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
