"""The MXFP4 quantiser, dequantiser and product, the routing to experts and the experts' feed-forward on the GPU, against plain
implementations in 64 bits (numpy, host)."""
import math

import numpy as np
import pytest
import torch

import ruquant_amd as rq
from tests import mx_oracle as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
# unit roundoff of an output's type (one rounding at the end)
ROUNDING = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _gpu(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).to(DEV)
    return t if dtype is None else t.to(dtype)


def _host(t):
    return t.detach().to(torch.float64).cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def _activations(M, K, seed, dtype):
    """wide-ranging blocks: every block of 32 has a magnitude of its own; returns the tensor and its values in 64 bits"""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((M, K)) * np.exp2(rng.integers(-6, 7, size=(M, K // 32)).repeat(32, axis=1))
    t = _gpu(x.astype(np.float32), dtype)
    return t, _host(t)


def _weights(shape, K, seed):
    rng = np.random.default_rng(seed)
    codes = rng.integers(0, 256, size=(*shape, K // 2), dtype=np.uint8)
    middle = 127 - round(0.5 * math.log2(K)) - 1
    scales = rng.integers(middle - 2, middle + 3, size=(*shape, K // 32), dtype=np.uint8)
    return codes, scales


# ---- quantiser and dequantiser -------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("M,K", [(1, 32), (3, 32), (1, 5120), (7, 96), (65, 544), (257, 4128)])
def test_quantize_matches_definition(M, K, dtype):
    x, x64 = _activations(M, K, 10 * M + K, DTYPES[dtype])
    codes, scales = rq.mx_quantize(x)
    want_codes, want_scales = ref.quantize(x64)
    assert codes.shape == (M, K // 2) and scales.shape == (M, K // 32)
    assert (scales.cpu().numpy() == want_scales).all()
    assert (ref.values(codes.cpu().numpy(), scales.cpu().numpy()) == ref.values(want_codes, want_scales)).all()


def test_quantize_ties_saturation_and_extremes():
    """Every tie between two codes, both signs, values between 6 and 8 units, denormals, the largest and smallest numbers, zeros."""
    rows = []
    for unit in (2.0 ** -149, 2.0 ** -130, 2.0 ** -127, 2.0 ** -126, 2.0 ** -20, 1.0, 2.0 ** 60, 2.0 ** 124):
        v = np.array([0, 0.25, 0.5, 0.75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7, 7.9]) * unit
        block = np.concatenate([v, -v[1:16]])
        rows += [block, np.where(np.arange(32) == 16, 0.0, block), np.roll(block, 5) * np.nextafter(1, 2)]
    rows += [np.zeros(32), np.full(32, np.finfo(np.float32).max), np.full(32, -2.0 ** -149)]
    x = np.stack(rows).astype(np.float32)
    codes, scales = rq.mx_quantize(_gpu(x))
    want_codes, want_scales = ref.quantize(x.astype(np.float64))
    assert (scales.cpu().numpy() == want_scales).all()
    assert (ref.values(codes.cpu().numpy(), scales.cpu().numpy()) == ref.values(want_codes, want_scales)).all()


@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_blocks_with_infinities_or_nan_become_nan(dtype):
    x = torch.ones((2, 128), dtype=DTYPES[dtype], device=DEV)
    x[0, 5], x[0, 40], x[1, 127] = float("nan"), float("inf"), float("-inf")
    codes, scales = rq.mx_quantize(x)
    assert scales.cpu().tolist() == [[255, 255, 125, 125], [125, 125, 125, 255]]
    y = rq.mx_dequantize(codes, scales).cpu()
    assert torch.isnan(y[0, :64]).all() and torch.isnan(y[1, 96:]).all()
    assert (y[0, 64:] == 1).all() and (y[1, :96] == 1).all()


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("offset,ld", [(0, 192), (1, 192), (0, 193), (3, 197)])
def test_quantize_reads_any_rows(offset, ld, dtype):
    """row strides and starts that are not multiples of 16 bytes"""
    x, _ = _activations(9, 192, 3, DTYPES[dtype])
    room = torch.full((9 * 200,), float("nan"), dtype=DTYPES[dtype], device=DEV)
    view = room[offset:].as_strided((9, 192), (ld, 1), offset)
    view.copy_(x)
    for a, b in zip(rq.mx_quantize(view), rq.mx_quantize(x)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_dequantize_every_code_under_every_scale(dtype):
    codes = np.tile(np.arange(256, dtype=np.uint8), (256, 1))
    scales = np.repeat(np.arange(256, dtype=np.uint8)[:, None], 16, axis=1)
    got = rq.mx_dequantize(_gpu(codes), _gpu(scales), dtype=DTYPES[dtype])
    want = torch.from_numpy(ref.values(codes, scales).astype(np.float32)).to(DTYPES[dtype])
    assert got.dtype == DTYPES[dtype]
    got = got.cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(0.0, 1e30, -1e30), want.nan_to_num(0.0, 1e30, -1e30))


def test_dequantize_takes_more_dimensions_and_slices():
    codes, scales = (_gpu(a) for a in _weights((3, 5), 96, 1))
    want = ref.values(codes.cpu().numpy(), scales.cpu().numpy())
    assert (_host(rq.mx_dequantize(codes, scales)) == want).all()
    assert (_host(rq.mx_dequantize(codes[1:, 1:3], scales[1:, 1:3])) == want[1:, 1:3]).all()


def test_empty_tensors():
    codes, scales = rq.mx_quantize(torch.empty((0, 64), device=DEV))
    assert codes.shape == (0, 32) and scales.shape == (0, 2)
    assert rq.mx_dequantize(codes, scales).shape == (0, 64)


# ---- product ---------------------------------------------------------------------------------------------------------

def _sum_bound(absolute, K):
    """An fp32 sum of K exact products, in whatever order: every addition is within 2^-24 of what it adds up, and no chain is
    longer than K / 32 additions of a block's exact sum and some joins. The matrix core's own additions may cut instead of
    rounding: twice that."""
    return 2 * (K / 32 + 16) * 2.0 ** -24 * absolute


def _check_product(y, x64, codes, scales, dtype):
    xq = ref.values(*ref.quantize(x64))
    w = ref.values(codes, scales)
    want = xq @ w.T
    bound = _sum_bound(np.abs(xq) @ np.abs(w).T, xq.shape[1]) + ROUNDING[dtype] * 1.01 * np.abs(want)
    if dtype == torch.float16:
        bound = bound + 2.0 ** -25
    assert y.dtype == dtype
    off = np.abs(_host(y) - want)
    assert (off <= bound).all(), "off by %g times the bound at %s" % ((off / bound).max(), np.unravel_index((off / bound).argmax(), off.shape))


PRODUCTS = [(1, 32, 1), (1, 5120, 64), (1, 256, 4097), (2, 160, 65), (3, 17408, 48), (4, 1376, 1000), (5, 4128, 33), (15, 1024, 128),
            (16, 512, 200), (17, 640, 63), (31, 2048, 129), (33, 96, 257), (45, 5120, 401), (63, 128, 64), (64, 1280, 192), (65, 128, 64),
            (66, 32, 5), (100, 4128, 130), (127, 512, 127), (128, 384, 128), (129, 640, 300), (200, 1376, 513), (257, 5120, 520),
            (300, 2080, 1025)]


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("M,K,N", PRODUCTS)
def test_product_matches_definition(M, K, N, dtype):
    x, x64 = _activations(M, K, M + K + N, DTYPES[dtype])
    codes, scales = _weights((N,), K, M + N)
    y = rq.mx_mul_mat(rq.MXWeight(_gpu(codes), _gpu(scales)), x)
    _check_product(y, x64, codes, scales, DTYPES[dtype])


@pytest.mark.parametrize("M", [1, 3, 40, 150])
def test_product_into_wider_rows_of_another_type(M):
    """x and out are views with row strides of their own; nothing outside of them is written"""
    K, N = 416, 77
    x, x64 = _activations(M, K, 7, torch.bfloat16)
    room = torch.full((M, K + 9), float("nan"), dtype=torch.bfloat16, device=DEV)
    room[:, 3:3 + K] = x
    codes, scales = _weights((N,), K, 5)
    W = rq.MXWeight(_gpu(codes), _gpu(scales))
    for dtype in DTYPES.values():
        to = torch.full((M, N + 5), 7.0, dtype=dtype, device=DEV)
        ws = W.workspace(M)
        y = rq.mx_mul_mat(W, room[:, 3:3 + K], out=to[:, 2:2 + N], workspace=ws)
        _check_product(y, x64, codes, scales, dtype)
        assert (to[:, :2] == 7).all() and (to[:, 2 + N:] == 7).all()


@pytest.mark.parametrize("M", [1, 5, 20, 60, 140])
def test_product_rows_do_not_depend_on_the_others(M):
    """a token's result is the same bits with other tokens beside it, and again when called again"""
    K, N = 1056, 260
    codes, scales = _weights((N,), K, 9)
    W = rq.MXWeight(_gpu(codes), _gpu(scales))
    x, _ = _activations(M, K, 4, torch.float32)
    y = rq.mx_mul_mat(W, x)
    assert torch.equal(y, rq.mx_mul_mat(W, x))
    other = x.clone()
    other[:-1] = 100.0
    assert torch.equal(rq.mx_mul_mat(W, other)[-1], y[-1])


@pytest.mark.parametrize("M,K,N", [(300, 1024, 70000), (520, 2080, 70000), (1000, 640, 40000), (200, 1376, 90000), (65, 8192, 70000),
                                   (2000, 384, 20000), (300, 17408, 9000)])
def test_product_of_many_tiles_is_that_of_few(M, K, N):
    """Every tile adds up the inputs in the same order, so a product whose tiles go over the chip in several rounds has the same bits as that
    of its tokens some at a time, and as itself again: nothing of a tile's neighbours, or of a wavefront that is behind, shows."""
    g = torch.Generator(device=DEV).manual_seed(M + K)
    codes = torch.empty((N, K // 2), dtype=torch.uint8, device=DEV).random_(0, 256, generator=g)
    scales = torch.empty((N, K // 32), dtype=torch.uint8, device=DEV).random_(116, 124, generator=g)
    W = rq.MXWeight(codes, scales)
    x = torch.randn((M, K), device=DEV, generator=g)
    y = rq.mx_mul_mat(W, x)
    for _ in range(3):
        assert torch.equal(rq.mx_mul_mat(W, x), y)
    for i in range(0, M, 100):   # (at least 17 tokens: fewer add up in another order)
        part = x[min(i, M - 60):i + 100]
        assert torch.equal(rq.mx_mul_mat(W, part), y[min(i, M - 60):i + 100])


SHARED = [(4, 17408, 5000), (17, 17408, 1), (33, 8992, 70), (64, 16384, 512), (65, 17376, 257), (130, 9056, 600)]


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("M,K,N", SHARED)
def test_product_whose_tiles_are_shared(M, K, N, dtype):
    """Few outputs of many inputs, each of which several workgroups sum up: as defined, and the same bits again and again, whoever is last
    and whatever the workspace held."""
    x, x64 = _activations(M, K, M + K + N, DTYPES[dtype])
    codes, scales = _weights((N,), K, M + N)
    W = rq.MXWeight(_gpu(codes), _gpu(scales))
    ws = W.workspace(M)
    y = rq.mx_mul_mat(W, x, workspace=ws).clone()
    _check_product(y, x64, codes, scales, DTYPES[dtype])
    for i in range(12):
        ws.fill_(i % 2 * 255)
        assert torch.equal(rq.mx_mul_mat(W, x, workspace=ws), y)


def test_shared_tiles_of_calls_behind_one_another():
    """calls on one workspace with nothing between them: no sum of the one in front shows"""
    K, N = 16384, 512
    codes, scales = _weights((N,), K, 3)
    W = rq.MXWeight(_gpu(codes), _gpu(scales))
    xs = [_activations(M, K, M, torch.float32)[0] for M in (40, 64, 40, 17, 33, 64)]
    want = [rq.mx_mul_mat(W, x) for x in xs]
    torch.cuda.synchronize()
    ws = W.workspace(64)
    for _ in range(10):
        got = [rq.mx_mul_mat(W, x, workspace=ws) for x in xs]
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_one_workspace_serves_every_number_of_tokens():
    K, N, most = 8992, 300, 700
    codes, scales = _weights((N,), K, 3)
    W = rq.MXWeight(_gpu(codes), _gpu(scales))
    x, _ = _activations(most, K, 8, torch.bfloat16)
    room = torch.full((W.workspace(most).numel() + 4096,), 7, dtype=torch.uint8, device=DEV)
    ws = room[:-4096]
    for M in (700, 400, 260, 128, 64, 33, 17, 16, 12, 5, 2, 1):
        assert torch.equal(rq.mx_mul_mat(W, x[:M], workspace=ws), rq.mx_mul_mat(W, x[:M]))
    assert (room[-4096:] == 7).all()


def test_product_whose_tiles_are_shared_in_a_graph():
    M, K, N = 40, 16384, 512
    codes, scales = _weights((N,), K, 3)
    W = rq.MXWeight(_gpu(codes), _gpu(scales))
    x, _ = _activations(M, K, 8, torch.bfloat16)
    want = rq.mx_mul_mat(W, x).clone()
    y, ws = torch.empty_like(want), W.workspace(M)
    rq.mx_mul_mat(W, x, out=y, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(3):
            rq.mx_mul_mat(W, x, out=y, workspace=ws)
    for i in range(5):
        y.zero_()
        ws.fill_(i)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


@pytest.mark.parametrize("M", [1, 18, 130])
def test_product_with_nan_and_infinity(M):
    """a NaN in a token makes its row NaN and no other; a NaN scale of a weight makes its row's outputs NaN and no other"""
    K, N = 288, 70
    x, x64 = _activations(M, K, 4, torch.float32)
    codes, scales = _weights((N,), K, 9)
    W = rq.MXWeight(_gpu(codes), _gpu(scales))
    want = rq.mx_mul_mat(W, x)
    bad = x.clone()
    bad[M - 1, K - 1] = float("inf")
    y = rq.mx_mul_mat(W, bad)
    assert torch.isnan(y[M - 1]).all() and torch.equal(y[:M - 1], want[:M - 1])
    scales[N - 1, K // 32 - 1] = 255
    y = rq.mx_mul_mat(rq.MXWeight(_gpu(codes), _gpu(scales)), x)
    assert torch.isnan(y[:, N - 1]).all() and torch.equal(y[:, :N - 1], want[:, :N - 1])


# ---- routing -----------------------------------------------------------------------------------------------------------

ROUTES = [  # M, E, top, groups, top_groups
    (1, 1, 1, 1, 1), (1, 64, 8, 1, 1), (5, 7, 7, 1, 1), (130, 64, 1, 1, 1), (33, 65, 6, 1, 1), (64, 128, 32, 1, 1), (17, 256, 8, 8, 4),
    (100, 160, 6, 8, 3), (50, 24, 3, 4, 2), (9, 10, 2, 5, 2), (40, 8, 4, 8, 4), (3, 1024, 16, 1, 1), (20, 1024, 8, 64, 7), (31, 63, 5, 3, 1),
    (2, 300, 9, 1, 1), (12, 512, 10, 4, 4), (19, 256, 8, 2, 1), (40, 128, 6, 16, 5), (21, 128, 9, 4, 2), (12, 192, 5, 6, 2), (70, 256, 32, 32, 9),
    (6, 512, 3, 2, 2), (300, 256, 12, 1, 1)]


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("M,E,top,groups,top_groups", ROUTES)
def test_route_matches_definition(M, E, top, groups, top_groups, biased, scoring):
    rng = np.random.default_rng(M + E)
    logits = (2 * rng.standard_normal((M, E))).astype(np.float32)
    bias = (0.1 * rng.standard_normal(E)).astype(np.float32) if biased else None
    for renormalize, scale in ((True, 1.0), (False, 2.5)):
        ids, w = rq.route(_gpu(logits), top, scoring=scoring, bias=None if bias is None else _gpu(bias), groups=groups,
                          top_groups=top_groups, renormalize=renormalize, scale=scale)
        want_ids, want_w, gap, size = ref.route(logits.astype(np.float64), top, scoring, bias, groups, top_groups, renormalize, scale)
        ids, w = ids.cpu().numpy(), _host(w)
        # a token whose choice hangs on less than what fp32 scores can be off by (exp, a sum, a division, the bias, a group's
        # sum: under 16 units of 2^-24 of the largest number that its choice compares) may choose otherwise
        sure = gap > 16 * 2.0 ** -24 * size
        assert sure.mean() > 0.9 or M < 20
        assert (ids[sure] == want_ids[sure]).all()
        # exp's argument is off by at most 2^-24 of itself (below 32: 2^-19 of the score), and so are numerator and sum
        assert (np.abs(w - want_w)[sure] <= 2.0 ** -18 * np.abs(want_w[sure]) + 1e-30).all()


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("groups,top_groups", [(1, 1), (4, 2)])
def test_route_ties_go_to_the_lowest_index(groups, top_groups, dtype):
    """logits of few distinct values, rows of one value"""
    rng = np.random.default_rng(3)
    logits = rng.integers(-1, 2, size=(64, 96)).astype(np.float32)
    logits[::7] = 0.5
    for scoring in ("softmax", "sigmoid"):
        ids, _ = rq.route(_gpu(logits, DTYPES[dtype]), 12, scoring=scoring, groups=groups, top_groups=top_groups)
        want, _, _, _ = ref.route(logits.astype(np.float64), 12, scoring, None, groups, top_groups, True, 1.0)
        assert (ids.cpu().numpy() == want).all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_with_masked_experts(scoring):
    """experts at minus infinity, or at the type's lowest value, come last and weigh nothing; a row with none left weighs 0"""
    x = np.zeros((5, 12), dtype=np.float32)
    x[0, :9] = -np.inf
    x[1, 3:] = np.finfo(np.float32).min
    x[2, :] = -np.inf
    x[3, 4] = np.nan
    x[4, 7] = np.inf
    ids, w = rq.route(_gpu(x), 4, scoring=scoring)
    ids, w = ids.cpu().numpy(), w.cpu().numpy()
    assert ids[0].tolist() == [9, 10, 11, 0] and ids[1].tolist() == [0, 1, 2, 3] and ids[2].tolist() == [0, 1, 2, 3]
    assert ids[3].tolist() == [0, 1, 2, 3] and ids[4].tolist() == [7, 0, 1, 2]
    third = np.float32(1) / np.float32(3)
    assert np.allclose(w[0], [third, third, third, 0], rtol=2e-7) and np.allclose(w[1], [third, third, third, 0], rtol=2e-7)
    assert (w[2] == 0).all() and np.allclose(w[3], 0.25, rtol=2e-7)
    assert np.allclose(w[4], [1, 0, 0, 0] if scoring == "softmax" else np.array([1, 0.5, 0.5, 0.5]) / 2.5, rtol=2e-7)


def test_route_with_a_bias_of_infinities_and_nan():
    x = np.zeros((1, 8), dtype=np.float32)
    bias = np.array([0, -np.inf, np.nan, np.inf, 1, 0, -1, 0], dtype=np.float32)
    for groups, top_groups, top, want in ((1, 1, 8, [3, 4, 0, 5, 7, 6, 1, 2]), (4, 2, 4, [3, 4, 5, 2])):
        ids, w = rq.route(_gpu(x), top, scoring="sigmoid", bias=_gpu(bias), groups=groups, top_groups=top_groups)
        assert ids.cpu().tolist() == [want]
        assert np.allclose(w.cpu().numpy(), 1 / top, rtol=2e-7)


@pytest.mark.parametrize("E,groups", [(64, 1), (128, 4), (256, 8), (512, 2), (1000, 1)])
def test_route_reads_a_bias_at_any_address(E, groups):
    x, room = torch.randn((33, E), device=DEV), torch.randn(E + 3, device=DEV)
    for at in range(4):
        bias = room[at:at + E]
        for scoring in ("softmax", "sigmoid"):
            for a, b in zip(rq.route(x, 5, scoring, bias, groups, groups), rq.route(x, 5, scoring, bias.clone(), groups, groups)):
                assert torch.equal(a, b)


def test_route_reads_rows_of_a_wider_matrix():
    x = torch.randn((37, 90), device=DEV)
    for dtype in DTYPES.values():
        wide = x.to(dtype)
        for a, b in zip(rq.route(wide[:, 5:70], 6), rq.route(wide[:, 5:70].contiguous(), 6)):
            assert torch.equal(a, b)


# ---- the experts' feed-forward -------------------------------------------------------------------------------------------

def _experts(E, F, K, N, seed):
    mats = [_weights((E, F), K, seed), _weights((E, F), K, seed + 1), _weights((E, N), F, seed + 2)]
    return mats, [rq.MXWeight(_gpu(c), _gpu(s)) for c, s in mats]


def _check_experts(y, x64, mats, ids, w, dtype):
    want, bound = ref.experts(x64, mats, ids, w, dtype == torch.bfloat16)
    bound = bound + ROUNDING[dtype] * 1.01 * np.abs(want) + (2.0 ** -25 if dtype == torch.float16 else 0)
    off = np.abs(_host(y) - want)
    assert (off <= bound).all(), "off by %g times the bound" % (off / bound).max()


EXPERTS = [  # M, E, top, K, F, N
    (1, 8, 2, 256, 96, 256), (1, 1, 1, 32, 32, 1), (1, 64, 8, 1280, 352, 300), (2, 5, 3, 416, 64, 65), (7, 4, 4, 544, 160, 96),
    (20, 6, 2, 320, 288, 130), (37, 3, 2, 512, 224, 200), (90, 4, 3, 256, 128, 64), (150, 3, 2, 384, 192, 140), (400, 2, 2, 160, 96, 129),
    (260, 60, 4, 288, 32, 70)]


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("M,E,top,K,F,N", EXPERTS)
def test_experts_match_definition(M, E, top, K, F, N, dtype):
    mats, (gate, up, down) = _experts(E, F, K, N, M + E)
    x, x64 = _activations(M, K, 8, DTYPES[dtype])
    x, x64 = x / 16, x64 / 16   # (exact)
    rng = np.random.default_rng(M)
    ids = np.stack([rng.permutation(E)[:top] for _ in range(M)]).astype(np.int32)
    w = rng.random((M, top)).astype(np.float32)
    y = rq.expert_ffn(gate, up, down, x, _gpu(ids), _gpu(w))
    assert y.dtype == DTYPES[dtype]
    _check_experts(y, x64, mats, ids, w, DTYPES[dtype])


@pytest.mark.parametrize("M", [1, 6, 64, 300])
def test_experts_skip_ids_that_are_none(M):
    """ids outside 0 .. E - 1 add nothing, whatever their weight; tokens without any expert give zeros; all tokens at one expert"""
    E, K, F, N, top = 5, 192, 96, 100, 3
    mats, (gate, up, down) = _experts(E, F, K, N, 40)
    x, x64 = _activations(M, K, 8, torch.float32)
    x, x64 = x / 16, x64 / 16
    rng = np.random.default_rng(M)
    ids = rng.integers(0, E, size=(M, top)).astype(np.int32)
    w = rng.random((M, top)).astype(np.float32)
    ids[rng.random((M, top)) < 0.4] = -1
    ids[::3, 1], w[ids < 0] = E, np.nan
    ids[M // 2], w[M // 2] = -1, np.inf
    w[ids == E] = np.nan
    y = rq.expert_ffn(gate, up, down, x, _gpu(ids), _gpu(w))
    assert (y[M // 2] == 0).all()
    _check_experts(y, x64, mats, ids, w, torch.float32)
    one = np.full((M, top), 2, dtype=np.int32)   # the same expert in every slot
    w = rng.random((M, top)).astype(np.float32)
    _check_experts(rq.expert_ffn(gate, up, down, x, _gpu(one), _gpu(w)), x64, mats, one, w, torch.float32)
    none = torch.full((M, top), -1, dtype=torch.int32, device=DEV)
    assert (rq.expert_ffn(gate, up, down, x, none, _gpu(w)) == 0).all()


@pytest.mark.parametrize("M", [1, 3, 30])
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_experts_read_any_rows(M, dtype):
    """x with a row stride and a start that are not multiples of 16 bytes"""
    E, K, F, N, top = 4, 96, 64, 40, 2
    _, (gate, up, down) = _experts(E, F, K, N, 7)
    x, _ = _activations(M, K, 2, DTYPES[dtype])
    room = torch.zeros((M, K + 3), dtype=DTYPES[dtype], device=DEV)
    room[:, 1:1 + K] = x
    ids = torch.arange(2 * M, device=DEV, dtype=torch.int32).view(M, 2) % E
    w = torch.rand((M, top), device=DEV)
    assert torch.equal(rq.expert_ffn(gate, up, down, room[:, 1:1 + K], ids, w), rq.expert_ffn(gate, up, down, x, ids, w))
    dense = rq.MXWeight(*(_gpu(a) for a in _weights((50,), K, 3)))
    assert torch.equal(rq.mx_mul_mat(dense, room[:, 1:1 + K]), rq.mx_mul_mat(dense, x))


def test_experts_with_many_slots():
    """more places than are sorted on the chip at once; every token's row as with its experts one at a time"""
    M, E, top, K, F, N = 3000, 5, 12, 64, 32, 33
    mats, (gate, up, down) = _experts(E, F, K, N, 5)
    x, x64 = _activations(M, K, 8, torch.float32)
    x, x64 = x / 16, x64 / 16
    rng = np.random.default_rng(1)
    ids = rng.integers(-1, E, size=(M, top)).astype(np.int32)
    w = rng.random((M, top)).astype(np.float32)
    _check_experts(rq.expert_ffn(gate, up, down, x, _gpu(ids), _gpu(w)), x64, mats, ids, w, torch.float32)


@pytest.mark.parametrize("M", [2, 40])
def test_experts_with_nan_and_infinity(M):
    """a token that holds one is NaN, the others keep their bits"""
    E, K, F, N, top = 4, 128, 64, 72, 2
    _, (gate, up, down) = _experts(E, F, K, N, 7)
    ids = torch.arange(2 * M, device=DEV, dtype=torch.int32).view(M, 2) % E
    w = torch.rand((M, top), device=DEV)
    for dtype in DTYPES.values():
        x, _ = _activations(M, K, 2, dtype)
        want = rq.expert_ffn(gate, up, down, x / 16, ids, w)
        bad = x / 16
        bad[M - 1, 5] = float("inf")
        y = rq.expert_ffn(gate, up, down, bad, ids, w)
        assert torch.isnan(y[M - 1]).all() and torch.equal(y[:M - 1], want[:M - 1])


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("M", [2, 40, 300])
def test_experts_outputs_stand_for_themselves(M, dtype):
    """an output whose weights hold a NaN is NaN, one 2^20 times its neighbours is itself, and neither shows in the outputs beside it"""
    E, K, F, N = 4, 128, 64, 72
    mats, (gate, up, down) = _experts(E, F, K, N, 7)
    ids = torch.arange(M, device=DEV, dtype=torch.int32).view(M, 1) % E
    w = torch.rand((M, 1), device=DEV) + 0.5
    x, _ = _activations(M, K, 2, DTYPES[dtype])
    want = rq.expert_ffn(gate, up, down, x / 16, ids, w)
    codes, scales = mats[2][0].copy(), mats[2][1].copy()
    scales[:, 3, 1] = 255
    codes[:, 70], scales[:, 70] = codes[:, 69], scales[:, 69] + 20
    y = rq.expert_ffn(gate, up, rq.MXWeight(_gpu(codes), _gpu(scales)), x / 16, ids, w)
    assert torch.isnan(y[:, 3]).all()
    if dtype != "fp16":   # (whose range ends in front of it)
        assert torch.equal(y[:, 70], want[:, 69] * 2.0 ** 20)
    # A neighbour may be held to 2^-40 of the large one, which can turn its last rounding, one unit in the last place (2^-7 at most).
    y, want = y.double(), want.double()
    off, large = (y - want).abs(), (want[:, 69] * 2.0 ** 20).abs()
    apart = torch.arange(N, device=DEV)
    assert (off[:, (apart < 64) & (apart != 3)] == 0).all()
    beside = (apart >= 64) & (apart != 70)
    assert (off[:, beside] <= 2.0 ** -7 * want[:, beside].abs() + 2.0 ** -39 * large[:, None]).all()


@pytest.mark.parametrize("E,top,M,K,F,N", [(32, 6, 2000, 1024, 640, 2048), (8, 2, 3000, 2048, 256, 1024), (60, 4, 600, 1376, 352, 1000)])
def test_experts_of_many_tiles_are_repeatable(E, top, M, K, F, N):
    """The same bits again and again, and for a part of the tokens (whose tiles are others)."""
    g = torch.Generator(device=DEV).manual_seed(M)
    weight = lambda *shape: rq.MXWeight(  # noqa: E731
        torch.empty((*shape[:-1], shape[-1] // 2), dtype=torch.uint8, device=DEV).random_(0, 256, generator=g),
        torch.empty((*shape[:-1], shape[-1] // 32), dtype=torch.uint8, device=DEV).random_(117, 121, generator=g))
    gate, up, down = weight(E, F, K), weight(E, F, K), weight(E, N, F)
    x = torch.randn((M, K), device=DEV, generator=g).bfloat16()
    ids = torch.randn((M, E), device=DEV, generator=g).topk(top, dim=1).indices.int()
    w = torch.rand((M, top), device=DEV, generator=g)
    y = rq.expert_ffn(gate, up, down, x, ids, w)
    for _ in range(4):
        assert torch.equal(rq.expert_ffn(gate, up, down, x, ids, w), y)
    for i in range(0, M, 500):
        assert torch.equal(rq.expert_ffn(gate, up, down, x[i:i + 500], ids[i:i + 500], w[i:i + 500]), y[i:i + 500])


@pytest.mark.parametrize("M", [1, 9, 70, 300])
def test_experts_are_repeatable_and_tokens_independent(M):
    E, K, F, N, top = 6, 512, 160, 192, 2
    _, (gate, up, down) = _experts(E, F, K, N, 3)
    x, _ = _activations(M, K, 8, torch.bfloat16)
    rng = np.random.default_rng(M)
    ids = _gpu(np.stack([rng.permutation(E)[:top] for _ in range(M)]).astype(np.int32))
    w = _gpu(rng.random((M, top)).astype(np.float32))
    out = torch.full((M, N + 3), 5.0, dtype=torch.bfloat16, device=DEV)
    ws = torch.empty(rq.expert_workspace_bytes(gate, down, M, top), dtype=torch.uint8, device=DEV)
    ws.fill_(255)   # (nothing of what a workspace held before shows)
    y = rq.expert_ffn(gate, up, down, x, ids, w, out=out[:, 1:1 + N], workspace=ws).clone()
    assert (out[:, 0] == 5).all() and (out[:, 1 + N:] == 5).all()
    for _ in range(3):
        assert torch.equal(rq.expert_ffn(gate, up, down, x, ids, w, workspace=ws), y)


# ---- graphs, streams, the whole layer -------------------------------------------------------------------------------------

def _layer(gate, up, down, router, x, bias, dense):
    """a mixture layer as a server runs it: router logits, choice, experts, and a plain product beside them"""
    logits = rq.mx_mul_mat(router, x, out=torch.empty((x.shape[0], router.N), dtype=torch.float32, device=DEV))
    ids, w = rq.route(logits, 3, scoring="sigmoid", bias=bias, groups=2, top_groups=1, scale=2.0)
    y = rq.expert_ffn(gate, up, down, x, ids, w)
    return y, rq.mx_mul_mat(dense, y), ids, w


@pytest.mark.parametrize("M", [1, 12, 80, 300])
def test_layer_in_a_graph_and_on_another_stream(M):
    """the operators together, replayed from a graph with eager work between the replays, and on a stream of their own"""
    E, K, F = 8, 320, 160
    _, (gate, up, down) = _experts(E, F, K, K, 3)
    router, dense = (rq.MXWeight(*(_gpu(a) for a in _weights((n,), K, 50 + n))) for n in (E, 200))
    bias = 0.1 * torch.randn((E,), device=DEV)
    xs = [_activations(M, K, 60 + i, torch.bfloat16)[0] / 16 for i in range(3)]
    want = [_layer(gate, up, down, router, x, bias, dense) for x in xs]
    x = xs[0].clone()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = _layer(gate, up, down, router, x, bias, dense)
    for i in (0, 1, 2, 1):
        x.copy_(xs[i])
        for t in got:
            t.fill_(3)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want[i]):
            assert torch.equal(a, b)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = [_layer(gate, up, down, router, x, bias, dense) for x in xs]
    torch.cuda.current_stream().wait_stream(stream)
    for a, b in zip(other, want):
        for s, t in zip(a, b):
            assert torch.equal(s, t)


# ---- refusals ---------------------------------------------------------------------------------------------------------------

def test_refusals():
    x = torch.zeros((2, 64), device=DEV)
    codes, scales = (_gpu(a) for a in _weights((4,), 64, 1))
    W = rq.MXWeight(codes, scales)
    three = rq.MXWeight(codes[None].expand(3, -1, -1), scales[None].expand(3, -1, -1))
    down = rq.MXWeight(*(_gpu(a) for a in _weights((3, 64), 64, 1)))
    gate = rq.MXWeight(*(_gpu(a) for a in _weights((3, 64), 64, 2)))
    ids, w = torch.zeros((2, 1), dtype=torch.int32, device=DEV), torch.zeros((2, 1), device=DEV)
    calls = [
        lambda: rq.mx_quantize(x[:, :40]), lambda: rq.mx_quantize(x.double()), lambda: rq.mx_quantize(x.cpu()), lambda: rq.mx_quantize(x.t()),
        lambda: rq.mx_quantize(x[0]), lambda: rq.mx_dequantize(codes, scales[:, :1]), lambda: rq.mx_dequantize(codes.int(), scales),
        lambda: rq.mx_dequantize(codes, scales, dtype=torch.float64), lambda: rq.MXWeight(codes[0], scales[0]),
        lambda: rq.MXWeight(codes.cpu(), scales.cpu()), lambda: rq.MXWeight(codes[:0], scales[:0]),
        lambda: rq.mx_mul_mat(W, x[:, :32]), lambda: rq.mx_mul_mat(three, x), lambda: rq.mx_mul_mat(W, x.cpu()),
        lambda: rq.mx_mul_mat(W, x, out=torch.zeros((2, 5), device=DEV)), lambda: rq.mx_mul_mat(W, x, out=torch.zeros((2, 4), device="cpu")),
        lambda: rq.mx_mul_mat(W, x, out=torch.zeros((2, 4), dtype=torch.int32, device=DEV)),
        lambda: rq.mx_mul_mat(W, x, out=torch.zeros((1, 4), device=DEV).expand(2, 4)),
        lambda: rq.mx_mul_mat(W, x.repeat(20, 1), workspace=torch.empty(256, dtype=torch.uint8, device=DEV)[:16]),
        lambda: rq.mx_mul_mat(W, x.repeat(20, 1), workspace=torch.empty(1 << 20, dtype=torch.uint8, device=DEV)[1:]),
        lambda: rq.route(x, 0), lambda: rq.route(x, 65), lambda: rq.route(x, 33), lambda: rq.route(x, 2, scoring="relu"),
        lambda: rq.route(x, 2, groups=5), lambda: rq.route(x, 2, groups=4, top_groups=5), lambda: rq.route(x, 17, groups=4),
        lambda: rq.route(x, 2, bias=torch.zeros(63, device=DEV)), lambda: rq.route(x, 2, bias=torch.zeros(64, device=DEV).half()),
        lambda: rq.route(x, 2, bias=torch.zeros(64)), lambda: rq.route(torch.zeros((1, 1025), device=DEV), 2), lambda: rq.route(x.long(), 2),
        lambda: rq.expert_ffn(gate, gate, W, x, ids, w), lambda: rq.expert_ffn(gate, gate, down, x[:, :32], ids, w),
        lambda: rq.expert_ffn(gate, three, down, x, ids, w), lambda: rq.expert_ffn(gate, gate, down, x, ids.long(), w),
        lambda: rq.expert_ffn(gate, gate, down, x, ids, w.half()), lambda: rq.expert_ffn(gate, gate, down, x, ids[:1], w),
        lambda: rq.expert_ffn(gate, gate, down, x, ids.cpu(), w), lambda: rq.expert_ffn(gate, gate, down, x, ids, w[:, :0]),
        lambda: rq.expert_ffn(gate, gate, down, x, ids, w, workspace=torch.empty(256, dtype=torch.uint8, device=DEV)),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(rq.RqError):
            call()
            pytest.fail("call %d was not refused" % i)
    assert rq.mx_mul_mat(W, x[:0]).shape == (0, 4) and rq.expert_ffn(gate, gate, down, x[:0], ids[:0], w[:0]).shape == (0, 64)
    assert rq.route(x[:0], 3)[0].shape == (0, 3)


def test_example_runs():
    """The mixture layer of examples/: rounding weights and activations to four bits (a unit in 8 to 16 of a block's largest) leaves its output
    within a third of the fp32 one, and not nearer than a thirtieth."""
    from examples.mixture_layer import main
    off = main(["--tokens", "1,5,70,200", "--hidden", "512", "--expert", "160", "--experts", "8", "--top", "3"])
    assert len(off) == 4 and all(1 / 30 < v < 1 / 3 for v in off), off
