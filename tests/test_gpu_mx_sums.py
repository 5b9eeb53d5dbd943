"""What the experts' feed-forward and the routing hold in how many bits, on the GPU."""
import numpy as np
import pytest
import torch

import ruquant_amd as rq
from tests import mx_oracle as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _gpu(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def _weights(shape, K, seed):
    rng = np.random.default_rng(seed)
    return (rng.integers(0, 256, size=(*shape, K // 2), dtype=np.uint8),
            rng.integers(120, 124, size=(*shape, K // 32), dtype=np.uint8))


def _weight(pair):
    return rq.MXWeight(*(_gpu(a) for a in pair))


@pytest.mark.parametrize("M", [3, 5, 40, 300])
def test_slots_that_cancel(M):
    """Two experts whose outputs are nearly the same, one taken from the other: what is left is as near the definition as sums in 32 bits
    and one last rounding allow, however small it is beside the experts' own outputs."""
    K, F, N = 128, 64, 72
    gate, up, down = _weights((1, F), K, 1), _weights((1, F), K, 2), _weights((1, N), F, 3)
    twice = lambda pair: tuple(a.repeat(2, axis=0) for a in pair)   # noqa: E731
    gate, up, down = twice(gate), twice(up), twice(down)
    down[0][1, :, 5] ^= 1   # one element of every row
    rng = np.random.default_rng(M)
    x = _gpu(rng.standard_normal((M, K)).astype(np.float32)).bfloat16()
    ids, w = np.tile(np.array([0, 1], dtype=np.int32), (M, 1)), np.tile(np.array([1, -1], dtype=np.float32), (M, 1))
    y = rq.expert_ffn(_weight(gate), _weight(up), _weight(down), x, _gpu(ids), _gpu(w)).double().cpu().numpy()
    want, bound = ref.experts(x.double().cpu().numpy(), (gate, up, down), ids, w, False)
    off = np.abs(y - want)
    bound = bound + 1.01 * 2.0 ** -8 * np.abs(want)
    assert (off <= bound).all(), "off by %g times the bound" % (off / bound).max()


@pytest.mark.parametrize("M,E,top,K,F,N", [(2, 4, 2, 128, 64, 72), (5, 4, 4, 544, 160, 96), (40, 6, 2, 320, 288, 130), (300, 3, 2, 384, 192, 140),
                                           (1000, 8, 4, 256, 96, 1000)])
def test_output_is_rounded_once(M, E, top, K, F, N):
    """an output in 16 bits is the one in fp32, rounded"""
    gate, up, down = (_weight(_weights((E, r), k, i)) for i, (r, k) in enumerate(((F, K), (F, K), (N, F))))
    g = torch.Generator(device=DEV).manual_seed(M)
    x = torch.randn((M, K), device=DEV, generator=g)
    ids = torch.randint(-1, E, (M, top), device=DEV, dtype=torch.int32, generator=g)
    w = torch.rand((M, top), device=DEV, generator=g)
    y = rq.expert_ffn(gate, up, down, x, ids, w)
    for dtype in (torch.bfloat16, torch.float16):
        out = rq.expert_ffn(gate, up, down, x, ids, w, out=torch.empty((M, N), dtype=dtype, device=DEV))
        assert torch.equal(out, y.to(dtype))


@pytest.mark.parametrize("E", [40, 128, 256, 300, 1024])
def test_weights_are_shares_of_the_whole_sum(E):
    """One score of 1 and 31 of 2^-24.5, each of which an fp32 sum that holds the first would drop. The sum is exact to 2^-24, and so are
    the first score (1 exactly) and the quotient; exp's error is one of 2^-19 in 31 scores that are 2^-19.6 of the sum."""
    logits = torch.full((3, E), -30.0, device=DEV)
    at = torch.arange(0, 32, device=DEV) * (E // 32)
    logits[:, at] = -17.0
    logits[:, at[7]] = 40.0
    ids, w = rq.route(logits, 32, scoring="sigmoid")
    small = 1 / (1 + np.exp(17.0))
    assert (ids[:, 0] == at[7]).all()
    assert np.abs(w[:, 0].double().cpu().numpy() - 1 / (1 + 31 * small)).max() <= 4 * 2.0 ** -24
    assert np.allclose(w[:, 1:].double().cpu().numpy(), small, rtol=2.0 ** -18)
