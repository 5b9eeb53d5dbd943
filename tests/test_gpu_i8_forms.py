"""Every kernel that the plans of the int8 product and of the products grouped by expert choose, each at sizes that reach it, against sums in 64 bits."""
import pytest
import torch

import ruquant_amd as rq
from tests import i8_plan_util as plan
from tests.i8_plan_util import BF16, I8, ROUNDS, STREAM, TILES

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _codes(shape, g):
    return torch.randint(-127, 128, shape, dtype=torch.int8, device=DEV, generator=g)


def _scales(shape, g):
    return 0.5 + torch.rand(shape, device=DEV, generator=g)


def _scaled(a, w, s, t):
    """the fp32 numbers ((sum) t) s; the sums of whole numbers are exact in 64 bits"""
    return (a.double() @ w.double().t().contiguous()).float() * t * s[:, None]


# K, N, M, then of the plan: kind, rows and positions of a tile, rows and positions of the rest's tiles, whether tiles are shared, tiles a compute unit holds
DENSE = [(64, 33, 1, STREAM, 0, 0, 0, 0, False, 0), (200, 1000, 16, STREAM, 0, 0, 0, 0, False, 0),
         (64, 33, 17, TILES, 64, 64, 0, 0, False, 2), (700, 100, 130, TILES, 64, 64, 0, 0, False, 2), (5000, 33, 17, TILES, 64, 64, 0, 0, True, 2),
         (64, 16500, 65, TILES, 128, 64, 0, 0, False, 2), (9000, 8200, 17, TILES, 128, 64, 0, 0, True, 2),
         (64, 16500, 200, TILES, 128, 128, 0, 0, False, 2), (640, 16500, 65, TILES, 128, 128, 0, 0, False, 1),
         (9000, 8200, 65, TILES, 128, 128, 0, 0, True, 1), (64, 16500, 400, TILES, 256, 256, 0, 0, False, 1),
         (130, 16500, 2100, TILES, 256, 256, 128, 128, False, 1), (5000, 16500, 200, TILES, 128, 128, 64, 64, False, 1)]


@pytest.mark.parametrize("K,N,M,kind,rows,tokens,rest_rows,rest_tokens,shared,resident", DENSE)
def test_product_of_every_form(K, N, M, kind, rows, tokens, rest_rows, rest_tokens, shared, resident):
    p = plan.product(K, N, M)
    assert p[0] == kind and p[1:3] == [rows, tokens] and p[4:6] == [rest_rows, rest_tokens] and (p[6] > 1) == shared and p[7] == resident, p
    g = torch.Generator(device=DEV).manual_seed(K + N + M)
    a, w, s, t = _codes((M, K), g), _codes((N, K), g), _scales((M,), g), _scales((N,), g)
    W = rq.I8Weight(w, t)
    ws = W.workspace(M)
    want = _scaled(a, w, s, t)
    for fill in (0, 255):
        ws.fill_(fill)
        assert torch.equal(rq.i8_mul_mat(W, a, scales=s, workspace=ws), want)
    assert torch.equal(rq.i8_mul_mat(W, a, scales=s, dtype=torch.bfloat16, workspace=ws), want.bfloat16())


@pytest.mark.parametrize("K,N,M", [(64, 33, 1), (300, 1000, 1), (301, 1000, 2), (5120, 300, 1), (17408, 64, 2), (40000, 40, 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_rows_rounded_inside(K, N, M, dtype):
    """the same bits as of rows rounded by i8_quantize"""
    assert plan.product(K, N, M, BF16)[0] == ROUNDS
    g = torch.Generator(device=DEV).manual_seed(K)
    W = rq.I8Weight(_codes((N, K), g), _scales((N,), g))
    x = (torch.randn((M, K), device=DEV, generator=g) * 3).to(dtype)
    a, s = rq.i8_quantize(x)
    assert torch.equal(rq.i8_mul_mat(W, x), rq.i8_mul_mat(W, a, scales=s, dtype=dtype))


GROUPED = [(BF16, 2, 64, 33, 4, STREAM, 0, 0, False), (BF16, 1, 64, 33, 17, TILES, 64, 64, False), (BF16, 1, 2000, 33, 17, TILES, 64, 64, True),
           (BF16, 8, 64, 4100, 40, TILES, 128, 64, False), (BF16, 8, 5000, 1000, 40, TILES, 128, 64, True), (BF16, 40, 64, 1000, 3000, TILES, 128, 128, False),
           (BF16, 40, 640, 520, 3000, TILES, 128, 128, False), (BF16, 1, 5000, 1000, 1000, TILES, 128, 128, True),
           (BF16, 1, 64, 1000, 9000, TILES, 256, 256, False), (I8, 2, 64, 33, 4, STREAM, 0, 0, False), (I8, 1, 64, 33, 17, TILES, 64, 64, False),
           (I8, 1, 5000, 33, 17, TILES, 64, 64, True), (I8, 8, 64, 4100, 40, TILES, 128, 64, False), (I8, 4, 640, 4100, 400, TILES, 128, 128, False),
           (I8, 40, 64, 1000, 3000, TILES, 128, 128, False), (I8, 1, 64, 1000, 9000, TILES, 256, 256, False)]


@pytest.mark.parametrize("kind,E,K,N,P,what,rows,tokens,shared", GROUPED)
def test_grouped_of_every_form(kind, E, K, N, P, what, rows, tokens, shared):
    p = plan.grouped(kind, E, K, N, P, P)
    assert (p[0], p[1], p[2], p[6] > 1) == (what, rows, tokens, shared), p
    g = torch.Generator(device=DEV).manual_seed(E + K + N + P)
    cuts = sorted(torch.randint(0, P + 1, (E - 1,), generator=torch.Generator().manual_seed(P)).tolist())
    offsets = torch.tensor([0] + cuts + [P], dtype=torch.int32, device=DEV)
    ends = offsets.tolist()
    order = torch.randperm(P, device=DEV, generator=g).to(torch.int32)
    if kind == I8:
        a, w, s, t = _codes((P, K), g), _codes((E, N, K), g), _scales((P,), g), _scales((E, N), g)
        W = rq.I8Weight(w, t)
        want = torch.zeros((P, N), device=DEV)
        for e, (i, j) in enumerate(zip(ends, ends[1:])):
            q = order[i:j].long()
            want[i:j] = _scaled(a[q], w[e], s[q], t[e])
        y = rq.grouped_mul_mat(W, a, offsets, rows=order, scales=s)
        assert torch.equal(y, want)
        assert torch.equal(rq.grouped_mul_mat(W, a, offsets, rows=order, scales=s), want)
        return
    x, w = torch.randn((P, K), device=DEV, generator=g).bfloat16(), (torch.randn((E, N, K), device=DEV, generator=g) * K ** -0.5).bfloat16()
    want, size = torch.zeros((P, N), dtype=torch.float64, device=DEV), torch.zeros((P, N), dtype=torch.float64, device=DEV)
    for e, (i, j) in enumerate(zip(ends, ends[1:])):
        q = order[i:j].long()
        want[i:j] = x[q].double() @ w[e].double().t().contiguous()
        size[i:j] = x[q].double().abs() @ w[e].double().abs().t().contiguous()
    W = rq.HalfWeight(w)
    y = rq.grouped_mul_mat(W, x, offsets, rows=order, dtype=torch.float32)
    # (the products are exact; a sum passes K / 16 instructions of at most 32 products and the join of at most 8 parts, each addition within
    # 2^-24 of what it adds up, twice that if it cuts; then one rounding)
    bound = 2 * (K / 16 + 48) * 2.0 ** -24 * size + 2.0 ** -24 * want.abs()
    assert ((y.double() - want).abs() <= bound).all()
    assert torch.equal(rq.grouped_mul_mat(W, x, offsets, rows=order, dtype=torch.float32), y)


@pytest.mark.parametrize("K", [1, 15, 16, 17, 31, 33, 63, 65, 127, 129, 191, 193, 257])
@pytest.mark.parametrize("M", [5, 40, 300])
def test_rows_that_end_anywhere(K, M):
    """... inside 16 bytes, a step, a pair of steps, with other bytes behind them"""
    g = torch.Generator(device=DEV).manual_seed(K)
    w, t, s = _codes((70, K), g), _scales((70,), g), _scales((M,), g)
    room = torch.full((M, K + 37), 99, dtype=torch.int8, device=DEV)
    room[:, 3:3 + K] = _codes((M, K), g)
    a = room[:, 3:3 + K]
    assert torch.equal(rq.i8_mul_mat(rq.I8Weight(w, t), a, scales=s), _scaled(a, w, s, t))


@pytest.mark.parametrize("M", [2, 17, 300])
def test_graphs_that_share_a_workspace(M):
    """two captured calls, replayed in turn many times with other work between: the counters of shared tiles are cleared each time"""
    g = torch.Generator(device=DEV).manual_seed(M)
    K, N = 5000, 40
    a, s = [_codes((M, K), g) for _ in range(2)], _scales((M,), g)
    Ws = [rq.I8Weight(_codes((N, K), g), _scales((N,), g)) for _ in range(2)]
    ws = Ws[0].workspace(M)
    want = [rq.i8_mul_mat(W, x, scales=s) for W, x in zip(Ws, a)]
    outs, graphs = [], []
    for W, x in zip(Ws, a):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(rq.i8_mul_mat(W, x, scales=s, workspace=ws))
        graphs.append(graph)
    for turn in range(6):
        ws.fill_(turn * 51)
        for graph in graphs:
            graph.replay()
        rq.i8_mul_mat(Ws[0], a[1], scales=s, workspace=ws)
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)
            o.zero_()


def test_calls_at_once_on_two_streams():
    g = torch.Generator(device=DEV).manual_seed(3)
    K, N, M = 5000, 40, 40
    a, s, W = _codes((M, K), g), _scales((M,), g), rq.I8Weight(_codes((N, K), g), _scales((N,), g))
    want = rq.i8_mul_mat(W, a, scales=s)
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    torch.cuda.synchronize()
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(rq.i8_mul_mat(W, a, scales=s))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for side in got for y in side)


def test_a_workspace_that_is_too_small_or_has_gaps_is_refused():
    g = torch.Generator(device=DEV).manual_seed(3)
    W, x = rq.I8Weight(_codes((40, 640), g), _scales((40,), g)), torch.randn((40, 640), device=DEV)
    room = torch.full((1 << 24,), 7, dtype=torch.uint8, device=DEV)
    offsets = torch.tensor([0, 40], dtype=torch.int32, device=DEV)
    n = rq.grouped_workspace_bytes(W, 40, 40)
    for bad in (room[::2], room[8:], room[:256], room.cpu()):
        with pytest.raises(rq.RqError):
            rq.i8_mul_mat(W, x, workspace=bad)
        with pytest.raises(rq.RqError):
            rq.grouped_mul_mat(W, x, offsets, workspace=bad)
    with pytest.raises(rq.RqError):
        rq.grouped_mul_mat(W, x, offsets, workspace=room[:n - 1])
    torch.cuda.synchronize()
    assert bool((room == 7).all())
    assert torch.equal(rq.grouped_mul_mat(W, x, offsets, workspace=room[:n]), rq.i8_mul_mat(W, x, workspace=room))


def test_calls_that_look_at_no_workspace():
    """every type and alignment of x in calls whose workspace may be null"""
    g = torch.Generator(device=DEV).manual_seed(3)
    L = rq.load_library()
    w, t = _codes((3, 40, 333), g), _scales((3, 40), g)
    dense, W, H = rq.I8Weight(w[0], t[0]), rq.I8Weight(w, t), rq.HalfWeight(w.half())
    offsets = torch.tensor([0, 2, 2, 5], dtype=torch.int32, device=DEV)
    assert L.rq_i8_workspace_bytes(333, 40, 2) == rq.grouped_workspace_bytes(W, 5, 5) == rq.grouped_workspace_bytes(H, 5, 5) == 256
    none = torch.empty(0, dtype=torch.uint8, device=DEV)
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        x = torch.randn((5, 339), device=DEV, generator=g).to(dtype)[:, 3:336]
        a, s = rq.i8_quantize(x)
        want = torch.stack([_scaled(a[p:p + 1], w[e], s[p:p + 1], t[e])[0] for p, e in enumerate((0, 0, 2, 2, 2))])
        for rows, scales in ((x, None), (a, s)):
            assert torch.equal(rq.i8_mul_mat(dense, rows[:2], scales=None if scales is None else scales[:2], dtype=dtype, workspace=none), want[:2].to(dtype))
            assert torch.equal(rq.grouped_mul_mat(W, rows, offsets, scales=scales, dtype=dtype, workspace=none), want.to(dtype))
    x = torch.randn((5, 339), device=DEV, generator=g).half()[:, 3:336]
    want = torch.stack([x[p].double() @ w[e].double().t().contiguous() for p, e in enumerate((0, 0, 2, 2, 2))])
    y = rq.grouped_mul_mat(H, x, offsets, dtype=torch.float32, workspace=none)
    # (333 products of 11 by 7 bits, exact in fp32: as in the other test, 2 (K / 16 + 48) 2^-24 of their magnitudes' sum, and a rounding)
    size = torch.stack([x[p].double().abs() @ w[e].double().abs().t().contiguous() for p, e in enumerate((0, 0, 2, 2, 2))])
    assert ((y.double() - want).abs() <= 2 * (333 / 16 + 49) * 2.0 ** -24 * size).all()


def test_refused_tensors():
    g = torch.Generator(device=DEV).manual_seed(3)
    W, H = rq.I8Weight(_codes((2, 40, 64), g), _scales((2, 40), g)), rq.HalfWeight(torch.ones((2, 40, 64), dtype=torch.float16, device=DEV))
    x, a, s = torch.randn((6, 64), device=DEV), _codes((6, 64), g), _scales((6,), g)
    mx = rq.MXWeight(torch.zeros((2, 40, 32), dtype=torch.uint8, device=DEV), torch.zeros((2, 40, 2), dtype=torch.uint8, device=DEV))
    offsets, rows = torch.tensor([0, 3, 6], dtype=torch.int32, device=DEV), torch.arange(6, dtype=torch.int32, device=DEV)
    call = lambda weight=W, x=x, offsets=offsets, **k: rq.grouped_mul_mat(weight, x, offsets, **k)  # noqa: E731
    call(), call(x=a, scales=s), call(H, x.half()), call(rows=rows, out_rows=rows)
    for bad in (lambda: call(x=a), lambda: call(scales=s), lambda: call(x=a, scales=s[:5]), lambda: call(x=a, scales=s.double()), lambda: call(H), lambda: call(H, x.bfloat16()),
                lambda: call(weight=mx, x=x), lambda: rq.i8_mul_mat(mx, x), lambda: call(weight=x), lambda: call(x=x[:, :63]), lambda: call(x=x.double()), lambda: call(offsets=offsets[:2]), lambda: call(offsets=offsets.long()), lambda: call(offsets=offsets.cpu()),
                lambda: call(rows=rows.long()), lambda: call(rows=rows.view(2, 3)), lambda: call(out_rows=rows[:5]), lambda: call(rows=rows.cpu()),
                lambda: call(out=torch.empty((6, 41), device=DEV)), lambda: call(out=torch.empty((5, 40), device=DEV)), lambda: call(out=torch.empty((40, 6), device=DEV).t()),
                lambda: call(out=torch.empty((6, 40), dtype=torch.float64, device=DEV)), lambda: call(dtype=torch.int8), lambda: rq.i8_mul_mat(W, x), lambda: rq.i8_mul_mat(H, x.half()),
                lambda: rq.sort_slots(rows, 4), lambda: rq.sort_slots(rows.view(2, 3).long(), 4), lambda: rq.sort_slots(rows.view(2, 3).t(), 4),
                lambda: rq.sort_slots(rows.view(2, 3), 0), lambda: rq.sort_slots(rows.view(2, 3), 1025), lambda: rq.I8Weight(a, s.half()), lambda: rq.I8Weight(a[0], s[0]),
                lambda: rq.I8Weight(a, s[:5]), lambda: rq.HalfWeight(x), lambda: rq.HalfWeight(x.half()[0]), lambda: rq.i8_quantize(x.double()), lambda: rq.i8_quantize(x.t()),
                lambda: rq.i8_quantize(x[:, :0]), lambda: rq.i8_dequantize(a, s, dtype=torch.int8)):
        with pytest.raises(rq.RqError):
            bad()


@pytest.mark.parametrize("kind", [I8, BF16])
@pytest.mark.parametrize("E,K,N,P", [(4, 64, 40, 300), (8, 5000, 1000, 40), (2, 64, 40, 4)])
def test_offsets_that_overlap_stay_inside(kind, E, K, N, P):
    """every group claims all positions: more tiles than there can be. What y holds is one group's row or another's, and nothing beside it is touched"""
    g = torch.Generator(device=DEV).manual_seed(P)
    offsets = torch.tensor([0, P] * ((E + 2) // 2), dtype=torch.int32, device=DEV)[:E + 1]
    room = torch.full((P + 20, N), 7.0, device=DEV)
    ws = torch.full((rq.load_library().rq_grouped_workspace_bytes(kind, E, K, N, P, P) + 4096,), 7, dtype=torch.uint8, device=DEV)
    n = ws.numel() - 4096
    if kind == I8:
        a, s = _codes((P, K), g), _scales((P,), g)
        rq.grouped_mul_mat(rq.I8Weight(_codes((E, N, K), g), _scales((E, N), g)), a, offsets, scales=s, out=room[10:P + 10], workspace=ws[:n])
    else:
        rq.grouped_mul_mat(rq.HalfWeight(torch.ones((E, N, K), dtype=torch.bfloat16, device=DEV)), torch.ones((P, K), dtype=torch.bfloat16, device=DEV), offsets,
                           out=room[10:P + 10], workspace=ws[:n])
    assert (ws[n:] == 7).all() and (room[:10] == 7).all() and (room[P + 10:] == 7).all()


def test_sizes_behind_32_bits():
    """rows of x, of y and codes whose offsets pass 2^32"""
    if torch.cuda.mem_get_info()[0] < 64 << 30:
        pytest.skip("needs 64 GB")
    g = torch.Generator(device=DEV).manual_seed(3)
    M, K = 70001, 65544   # 4.6e9 elements
    x = torch.zeros((M, K), dtype=torch.bfloat16, device=DEV)
    some = torch.tensor([0, 1, 32768, 65535, 65536, M - 1], device=DEV)
    x[some] = torch.randn((6, K), device=DEV, generator=g).bfloat16()
    codes, scales = rq.i8_quantize(x)
    a, s = rq.i8_quantize(x[some])
    assert torch.equal(codes[some], a) and torch.equal(scales[some], s) and not codes[2:32768].any()
    w = _codes((1, 24, K), g)
    W = rq.I8Weight(w, torch.ones((1, 24), device=DEV))
    rows = torch.cat([some, some.flip(0)]).to(torch.int32)
    offsets = torch.tensor([0, 12], dtype=torch.int32, device=DEV)
    want = _scaled(a, w[0], s, torch.ones(24, device=DEV))
    assert torch.equal(rq.grouped_mul_mat(W, codes, offsets, rows=rows, scales=scales)[:6], want)
    many = rows.repeat(20)
    y = rq.grouped_mul_mat(W, codes, torch.tensor([0, 240], dtype=torch.int32, device=DEV), rows=many, scales=scales)
    assert torch.equal(y.view(20, 12, 24)[7, :6], want)
    del x, codes
    M, N = 130000, 17408   # 2.26e9 outputs
    a, w, s, t = _codes((M, 64), g), _codes((N, 64), g), _scales((M,), g), _scales((N,), g)
    y = rq.i8_mul_mat(rq.I8Weight(w, t), a, scales=s, dtype=torch.bfloat16)
    some = torch.tensor([0, 77, 61680, 123361, M - 1], device=DEV)
    assert torch.equal(y[some], _scaled(a[some], w, s[some], t).bfloat16())
