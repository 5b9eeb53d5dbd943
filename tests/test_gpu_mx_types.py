"""The MXFP4 quantiser over the whole range of the 16-bit types."""
import numpy as np
import pytest
import torch

import ruquant_amd as rq
from tests import mx_oracle as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"fp16": (torch.float16, -24, 15), "bf16": (torch.bfloat16, -133, 127)}   # exponents of the smallest and the largest number


def _check(x):
    codes, scales = rq.mx_quantize(x.to(DEV))
    want_codes, want_scales = ref.quantize(x.double().numpy())
    assert (scales.cpu().numpy() == want_scales).all()
    assert (ref.values(codes.cpu().numpy(), scales.cpu().numpy()) == ref.values(want_codes, want_scales)).all()


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_every_number(dtype):
    """all finite bit patterns, in blocks of neighbours and in blocks that reach over the whole range"""
    bits = torch.arange(65536, dtype=torch.int32)
    x = torch.where(bits >= 32768, bits - 65536, bits).to(torch.int16).view(TYPES[dtype][0])
    finite = torch.isfinite(x.float())
    x = x[finite]
    x = x[:x.numel() // 32 * 32]
    _check(x.view(-1, 32))
    _check(x[torch.randperm(x.numel(), generator=torch.Generator().manual_seed(1))].view(-1, 128))
    _check(x.view(32, -1).t().contiguous())


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_ties_and_saturation_at_every_exponent(dtype):
    """every tie between two codes, both signs, and values between 6 and 8 units, for every unit that the type has"""
    t, least, most = TYPES[dtype]
    v = np.array([0, 0.25, 0.5, 0.75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7, 7.9])
    block = np.concatenate([v, -v[1:16]])
    rows = []
    for e in range(least, most - 1):   # (7.9 units are the largest)
        rows += [block * 2.0 ** e, np.where(np.arange(32) == 16, 0.0, block) * 2.0 ** e, np.where(np.abs(block) > 6, 0.0, block) * -2.0 ** e]
    x = torch.from_numpy(np.stack(rows)).to(t)
    assert torch.isfinite(x.float()).all()
    _check(x)


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_products_of_the_smallest_and_the_largest(dtype):
    """one token and some, whose blocks are of the type's smallest numbers, its largest, and both: the weight's scales bring outputs into range"""
    t, least, most = TYPES[dtype]
    K, N = 128, 40
    rng = np.random.default_rng(2)
    codes = rng.integers(0, 256, size=(N, K // 2), dtype=np.uint8)
    for e, scale in ((least, 127 - least // 2), (most - 3, 127 - most // 2)):
        v = rng.integers(1, 8, size=(20, K)) * 2.0 ** e * rng.choice((-1.0, 1.0), size=(20, K))
        x = torch.from_numpy(v).to(t)
        scales = np.full((N, K // 32), scale, dtype=np.uint8)
        W = rq.MXWeight(torch.from_numpy(codes).to(DEV), torch.from_numpy(scales).to(DEV))
        xq, w = ref.values(*ref.quantize(x.double().numpy())), ref.values(codes, scales)
        want, size = xq @ w.T, np.abs(xq) @ np.abs(w).T
        for M in (1, 3, 12, 20):
            y = rq.mx_mul_mat(W, x[:M].to(DEV), out=torch.empty((M, N), device=DEV)).double().cpu().numpy()
            # (an fp32 sum of K exact products, as in the tests of the product)
            assert (np.abs(y - want[:M]) <= (2 * (K / 32 + 16) + 1.01) * 2.0 ** -24 * size[:M]).all()
