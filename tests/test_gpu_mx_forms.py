"""Every form of the MXFP4 tiles against the definition in 64 bits. The shapes say which form they mean, and the plan is asked."""
import numpy as np
import pytest
import torch

import ruquant_amd as rq
from tests import mx_oracle as ref
from tests import mx_plan_util as plans

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}   # unit roundoff


def _rounded64(x):
    """x's values after quantisation, by the oracle, some rows at a time"""
    x = x.double().cpu().numpy()
    return torch.from_numpy(np.concatenate([ref.values(*ref.quantize(x[i:i + 500])) for i in range(0, len(x), 500)])).to(DEV)


def _values64(codes, scales):
    t = torch.from_numpy(np.concatenate([ref.ELEMENTS, -ref.ELEMENTS])).to(DEV)
    v = t[torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).int()]
    return v * torch.exp2(scales.double() - 127).repeat_interleave(32, dim=-1)


def _weight(shape, K, g):
    middle = 127 - K.bit_length() // 2
    return (torch.empty((*shape, K // 2), dtype=torch.uint8, device=DEV).random_(0, 256, generator=g),
            torch.empty((*shape, K // 32), dtype=torch.uint8, device=DEV).random_(middle - 3, middle + 3, generator=g))


@pytest.mark.parametrize("K,N,M,tiles,behind", plans.PRODUCTS + [(*s, (64, 64, 2), (0, 0)) for s in plans.SHARED])
def test_product(K, N, M, tiles, behind):
    """all outputs, in each type: the rows of the tiles, those behind them, the last row and token tiles"""
    kind, form, rest, _, splits = plans.product(K, N, M)
    assert (kind, form, rest) == (plans.TILES, tiles, behind) and (splits > 1) == ((K, N, M) in plans.SHARED)
    g = torch.Generator(device=DEV).manual_seed(K + N + M)
    codes, scales = _weight((N,), K, g)
    W = rq.MXWeight(codes, scales)
    x = torch.randn((M, K), device=DEV, generator=g) * torch.exp2(torch.randint(-6, 7, (M, K // 32), device=DEV, generator=g)).repeat_interleave(32, dim=1)
    x = x.bfloat16()   # (the same values in every type, but for what is so small that its code is 0)
    xq = _rounded64(x)
    ys = {t: rq.mx_mul_mat(W, x.to(t), out=torch.full((M, N + 3), 7.0, dtype=t, device=DEV)[:, 1:N + 1]) for t in DTYPES}
    for n in range(0, N, 8192):
        w = _values64(codes[n:n + 8192], scales[n:n + 8192]).t().contiguous()
        want, size = torch.matmul(xq, w), torch.matmul(xq.abs(), w.abs())
        for t, unit in DTYPES.items():
            # an fp32 sum of exact products in chains of K / 32 additions and some joins, which the matrix core may cut (twice 2^-24 each), and
            # the last rounding; fp16's smallest unit is 2^-24
            bound = 2 * (K / 32 + 16) * 2.0 ** -24 * size + 1.01 * unit * want.abs() + (2.0 ** -25 if t == torch.float16 else 0)
            off = (ys[t][:, n:n + 8192].double() - want).abs()
            assert bool((off <= bound).all()), "%s: off by %g times the bound in rows from %d on" % (t, (off / bound).max(), n)
    for y in ys.values():   # (nothing beside the outputs is written)
        whole = y.as_strided((M, N + 3), (N + 3, 1), 0)
        assert bool((whole[:, 0] == 7).all()) and bool((whole[:, N + 1:] == 7).all())


@pytest.mark.parametrize("E,K,F,N,M,top,tiles", plans.EXPERTS)
def test_experts(E, K, F, N, M, top, tiles):
    """Uneven loads, absent experts and one without a token: some tokens against the definition, all of them the same bits as in calls of few,
    which take tiles of 64 tokens; 16-bit outputs are the fp32 ones, rounded."""
    assert plans.experts(E, K, F, N, M, top) == (plans.TILES, tiles)
    g = torch.Generator(device=DEV).manual_seed(E + K + M)
    mats = [_weight((E, F), K, g), _weight((E, F), K, g), _weight((E, N), F, g)]
    gate, up, down = (rq.MXWeight(*m) for m in mats)
    x = torch.randn((M, K), device=DEV, generator=g).bfloat16()
    ids = (E * torch.rand((M, top), device=DEV, generator=g) ** 2.5).int() - 1   # (the last expert has none, -1 is absent)
    w = torch.randn((M, top), device=DEV, generator=g)
    y = rq.expert_ffn(gate, up, down, x, ids, w, out=torch.empty((M, N), device=DEV))
    for t in (torch.bfloat16, torch.float16):
        assert torch.equal(rq.expert_ffn(gate, up, down, x, ids, w, out=torch.empty((M, N), dtype=t, device=DEV)), y.to(t))
    few = min(M, 96 * E // top)
    assert plans.experts(E, K, F, N, few, top) == (plans.TILES, (128, 64))
    for at in range(0, M, few):
        at = min(at, M - few)
        part = slice(at, at + few)
        assert torch.equal(rq.expert_ffn(gate, up, down, x[part], ids[part], w[part], out=torch.empty((few, N), device=DEV)), y[part])
    some = torch.cat([torch.arange(60, device=DEV), torch.randint(0, M, (80,), device=DEV, generator=g), torch.arange(M - 60, M, device=DEV)])
    want, bound = ref.experts(x[some].double().cpu().numpy(), [tuple(a.cpu().numpy() for a in m) for m in mats], ids[some].cpu().numpy(),
                              w[some].cpu().numpy(), False)
    off = np.abs(y[some].double().cpu().numpy() - want)
    bound = bound + 1.01 * 2.0 ** -24 * np.abs(want)
    assert (off <= bound).all(), "off by %g times the bound" % (off[bound > 0] / bound[bound > 0]).max()
