"""The int8 and grouped products at the ends of what their calls allow: offsets, sizes and indices that no ordinary step has. Every case names the form
that it means and asks the library's plan for it, so that a rule that moves shows."""
import pytest
import torch

import ruquant_amd as rq
from tests import i8_plan_util as plan
from tests.i8_plan_util import BF16, F16, F32, I8, ROUNDS, STREAM, TILES

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FLOATS = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
LOW, HIGH = -2 ** 31, 2 ** 31 - 1


def _codes(shape, g):
    return torch.randint(-127, 128, shape, dtype=torch.int8, device=DEV, generator=g)


def _scales(shape, g):
    return 0.5 + torch.rand(shape, device=DEV, generator=g)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _scaled(a, w, s, t):
    """the fp32 numbers ((sum) t) s; the sums of whole numbers are exact in 64 bits"""
    return (a.double() @ w.double().t().contiguous()).float() * t * s[:, None]


def _small(shape, g):
    """whole numbers of 16 bits whose products' sums are exact in fp32 in any order"""
    return torch.randint(-8, 9, shape, device=DEV, generator=g).float()


def _case(kind, E, K, N, M, g):
    """(weight, x, keyword arguments, y of row m of x by expert e): bits, whatever the kernel"""
    if kind == I8:
        a, w, s, t = _codes((M, K), g), _codes((E, N, K), g), _scales((M,), g), _scales((E, N), g)
        return rq.I8Weight(w, t), a, {"scales": s}, lambda m, e: _scaled(a[m], w[e], s[m], t[e])
    x, w = (_small(shape, g).to(torch.float16 if kind == F16 else torch.bfloat16) for shape in ((M, K), (E, N, K)))
    return rq.HalfWeight(w), x, {}, lambda m, e: (x[m].double() @ w[e].double().t().contiguous()).float()


# ---- offsets ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", [I8, F16, BF16])
@pytest.mark.parametrize("P,form", [(10, STREAM), (40, TILES)])
def test_offsets_of_any_number(P, form, kind):
    """starts in front of the first position, ends behind the last, an end as far in front of its start as there are numbers"""
    E, K, N = 5, 64, 40
    assert plan.grouped(kind, E, K, N, P, P)[0] == form
    g = torch.Generator(device=DEV).manual_seed(P)
    weight, x, more, rows = _case(kind, E, K, N, P, g)
    p = torch.arange(P, device=DEV)
    for offsets in ([LOW, 4, HIGH, LOW, LOW, LOW], [-1, 3, LOW, LOW, LOW, LOW], [P, -1, 4, P, LOW + 3, LOW], [HIGH, LOW, LOW, HIGH, LOW, LOW]):
        out = torch.full((P, N), 7.0, device=DEV)
        want = out.clone()
        ends = [min(max(o, 0), P) for o in offsets]
        for e, (i, j) in enumerate(zip(ends, ends[1:])):
            if i < j:
                want[i:j] = rows(p[i:j], e)
        assert torch.equal(rq.grouped_mul_mat(weight, x, _ints(offsets), out=out, **more), want), offsets


# ---- rows rounded by every workgroup ------------------------------------------------------------------------------------

def _floats(M, K, dtype, g):
    """rows of different magnitudes"""
    return (torch.randn((M, K), device=DEV, generator=g) * torch.exp2(torch.arange(M, device=DEV) % 7 - 3.0)[:, None]).to(dtype)


@pytest.mark.parametrize("dtype", sorted(FLOATS, key=str))
@pytest.mark.parametrize("K,N,M,form,rows", [(65344, 40, 1, ROUNDS, 1), (65345, 40, 1, STREAM, 0), (65472, 40, 1, STREAM, 0), (32640, 40, 2, ROUNDS, 2),
                                             (32641, 40, 2, ROUNDS, 1), (32704, 40, 2, ROUNDS, 1)])
def test_longest_rounded_rows(K, N, M, form, rows, dtype):
    assert plan.product(K, N, M, FLOATS[dtype])[:2] == [form, rows]
    g = torch.Generator(device=DEV).manual_seed(K + M)
    w, t, x = _codes((N, K), g), _scales((N,), g), _floats(M, K, dtype, g)
    a, s = rq.i8_quantize(x)
    assert torch.equal(rq.i8_mul_mat(rq.I8Weight(w, t), x), _scaled(a, w, s, t).to(dtype))
