"""NaN logits in the routing: such an expert weighs nothing and is chosen behind every number."""
import math

import pytest
import torch

import ruquant_amd as rq

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NAN = float("nan")


def _route(rows, top, bias=None, **k):
    ids, w = rq.route(torch.tensor(rows, device=DEV), top, bias=None if bias is None else torch.tensor(bias, device=DEV), **k)
    return ids.cpu().tolist(), w.cpu()


def test_behind_a_number_with_less_bias():
    ids, w = _route([[NAN, -1.0]], 1, bias=[0.5, 0.0], scoring="sigmoid")
    assert ids == [[1]] and w.tolist() == [[1.0]]
    ids, _ = _route([[NAN, -1.0, 0.0]], 3, bias=[0.5, -2.0, -1.0], scoring="softmax")
    assert ids == [[2, 1, 0]]


def test_behind_a_score_of_zero():
    """softmax(-200) beside 0 is 0 in fp32, and so is the score of minus infinity"""
    ids, w = _route([[NAN, 0.0, -200.0, -math.inf]], 4)
    assert ids == [[1, 2, 3, 0]] and w.tolist() == [[1, 0, 0, 0]]


def test_groups():
    # a group of nothing but NaN is behind one that holds a number
    assert _route([[NAN, NAN, NAN, 0.9, NAN, NAN]], 1, groups=3, top_groups=1)[0] == [[3]]
    assert _route([[NAN, NAN, NAN, 0.9, NAN, NAN]], 1, groups=3, top_groups=1, bias=[1.0, 1.0, 0.0, 0.0, 1.0, 1.0], scoring="sigmoid")[0] == [[3]]
    # and so with biases of minus infinity
    assert _route([[0.0, 0.0, 0.0, 0.9]], 1, groups=2, top_groups=1, bias=[-math.inf, -math.inf, -math.inf, 0.0])[0] == [[3]]


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups,top_groups", [(24, 1, 1), (24, 4, 3), (65, 1, 1), (128, 8, 5), (200, 1, 1), (256, 8, 8), (300, 2, 2), (512, 1, 1),
                                                 (1000, 1, 1), (1024, 16, 13)])
def test_as_an_expert_that_must_not_be_chosen(E, groups, top_groups, scoring):
    """a row with NaN logits chooses as one where those are minus infinity under a bias of minus infinity"""
    g = torch.Generator(device=DEV).manual_seed(E)
    logits = torch.randn((9, E), device=DEV, generator=g)
    bias = torch.rand((E,), device=DEV, generator=g) - 0.3
    gone = torch.rand((9, E), device=DEV, generator=g) < 0.3
    ids, w = rq.route(logits.masked_fill(gone, NAN), 8, scoring=scoring, bias=bias, groups=groups, top_groups=top_groups)
    assert not gone.gather(1, ids.long()).any()
    for m in range(9):
        one = rq.route(logits[m:m + 1].masked_fill(gone[m], -math.inf), 8, scoring=scoring, bias=bias.masked_fill(gone[m], -math.inf), groups=groups,
                       top_groups=top_groups)
        assert torch.equal(one[0][0], ids[m]) and torch.equal(one[1][0], w[m])
