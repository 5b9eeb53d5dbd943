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
    w, t, x = _codes((N, K), g), _scales((N,), g) * K ** -0.5 / 64, _floats(M, K, dtype, g)
    a, s = rq.i8_quantize(x)
    assert torch.equal(rq.i8_mul_mat(rq.I8Weight(w, t), x), _scaled(a, w, s, t).to(dtype))


@pytest.mark.parametrize("dtype", sorted(FLOATS, key=str))
@pytest.mark.parametrize("E,K,N,sizes,rows", [(0, 40000, 64, [2], 1), (8, 9280, 64, [0, 0, 8], 7), (8, 9280, 1280, [0, 0, 8], 7), (8, 9344, 64, [7, 1], 6), (8, 17408, 64, [0, 8], 3),
                                              (8, 17408, 600, [1, 0, 6, 1], 3), (64, 40000, 40, [3, 2, 0, 3], 1), (3, 30000, 40, [3, 0, 2], 2)])
def test_rounding_in_passes(E, K, N, sizes, rows, dtype):
    """more rows in a group than are rounded at a time: each pass fills the place that the sums of the one before had"""
    P = sum(sizes)
    p = plan.grouped(I8, E, K, N, P, P, FLOATS[dtype]) if E else plan.product(K, N, P, FLOATS[dtype])
    assert p[:2] == [ROUNDS, rows] and max(sizes) > rows
    g = torch.Generator(device=DEV).manual_seed(K + N + P)
    w, t, x = _codes((len(sizes), N, K), g), _scales((len(sizes), N), g) * K ** -0.5 / 64, _floats(P, K, dtype, g)
    x[P - 1, K - 1] = float("nan")
    a, s = rq.i8_quantize(x)
    ends = [sum(sizes[:e]) for e in range(len(sizes) + 1)]
    want = torch.cat([_scaled(a[i:j], w[e], s[i:j], t[e]) for e, (i, j) in enumerate(zip(ends, ends[1:]))]).to(dtype)
    if not E:
        y = rq.i8_mul_mat(rq.I8Weight(w[0], t[0]), x)
    else:   # (the experts behind are asked for by nobody)
        w, t = torch.cat([w, w[:1].expand(E - len(sizes), -1, -1)]), torch.cat([t, t[:1].expand(E - len(sizes), -1)])
        y = rq.grouped_mul_mat(rq.I8Weight(w, t), x, _ints(ends + [P] * (E - len(sizes))))
    assert torch.isnan(y[P - 1]).all() and torch.isfinite(y[:P - 1]).all()
    assert torch.equal(y.nan_to_num(nan=-1.0), want.nan_to_num(nan=-1.0))


@pytest.mark.parametrize("dtype", sorted(FLOATS, key=str))
@pytest.mark.parametrize("K,N,chunk", [(200, 70, 8), (201, 40, 8), (9344, 40, 6), (17408, 600, 3)])
def test_rounded_rows_that_are_not_there(K, N, chunk, dtype):
    """... give zeros, also where the row that is read in their place is NaN, and places that are not there are not written"""
    E, M, P = 4, 5, 8
    assert plan.grouped(I8, E, K, N, M, P, FLOATS[dtype])[:2] == [ROUNDS, chunk]
    g = torch.Generator(device=DEV).manual_seed(K)
    w, t, x = _codes((E, N, K), g), _scales((E, N), g) * K ** -0.5 / 64, _floats(M, K, dtype, g)
    x[0, 3] = float("nan")
    rows, places, offsets = [-1, 4, M, 0, HIGH, 1, LOW, 1], [9, 0, 3, 10, 8, -1, LOW, 2], [0, 1, 1, 7, 8]
    a, s = rq.i8_quantize(x)
    weight, out = rq.I8Weight(w, t), torch.full((10, N), 7.0, dtype=dtype, device=DEV)
    want = out.clone()
    for p, (r, q) in enumerate(zip(rows, places)):
        e = next(e for e in range(E) if offsets[e] <= p < offsets[e + 1])
        if 0 <= q < 10:
            want[q] = _scaled(a[r:r + 1], w[e], s[r:r + 1], t[e])[0].to(dtype) if 0 <= r < M else 0
    given = torch.full_like(out, 7.0)
    rq.grouped_mul_mat(weight, x, _ints(offsets), rows=_ints(rows), out_rows=_ints(places), out=out)
    rq.grouped_mul_mat(weight, a, _ints(offsets), rows=_ints(rows), out_rows=_ints(places), scales=s, out=given)
    assert not torch.isnan(want).any() and torch.equal(out, want) and torch.equal(given, want)
    places[3] = 1   # (row 0 itself)
    rq.grouped_mul_mat(weight, x, _ints(offsets), rows=_ints(rows), out_rows=_ints(places), out=out)
    assert torch.isnan(out[1]).all() and torch.equal(out[2:], want[2:]) and torch.equal(out[0], want[0])


# ---- the streamed form ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind,dtype", [(I8, None), (I8, torch.float32), (I8, torch.bfloat16), (F16, None), (BF16, None)])
@pytest.mark.parametrize("sizes,behind,form", [([3, 0, 2, 1], 8, STREAM), ([2, 0, 0, 1], 4, ROUNDS), ([1, 0, 2, 0] * 5, 30, STREAM), ([17, 0, 3] + 17 * [0], 20, STREAM)])
def test_rows_of_no_group_beside_streamed_ones(sizes, behind, form, kind, dtype):
    E, P, K, N = len(sizes), sum(sizes) + behind, 128, 72
    used = P - behind
    assert plan.grouped(kind, E, K, N, P, P, kind if dtype is None else FLOATS[dtype])[0] == (form if dtype is not None else STREAM)
    g = torch.Generator(device=DEV).manual_seed(P)
    weight, x, more, rows = _case(kind, E, K, N, P, g)
    if dtype is not None:
        x, codes = _floats(P, K, dtype, g), _codes((E, N, K), g)
        scales, more, (a, s) = _scales((E, N), g), {}, rq.i8_quantize(x)
        weight, rows = rq.I8Weight(codes, scales), lambda m, e: _scaled(a[m], codes[e], s[m], scales[e])
        x[used:] = float("nan")
    elif kind != I8:
        x[used:] = float("nan")
    out = torch.full((P, N), 7.0, device=DEV)
    want, at = out.clone(), 0
    for e, n in enumerate(sizes):
        if n:
            want[at:at + n] = rows(torch.arange(at, at + n, device=DEV), e)
        at += n
    offsets = _ints([sum(sizes[:e]) for e in range(E + 1)])
    assert torch.equal(rq.grouped_mul_mat(weight, x, offsets, out=out, **more), want)


@pytest.mark.parametrize("kind", [I8, F16, BF16])
@pytest.mark.parametrize("E,N,sizes", [(128, 40, {77: 512}), (128, 40, {0: 17, 5: 16, 64: 33, 65: 1, 127: 445}), (128, 700, {3: 100, 126: 412})])
def test_few_rows_of_which_one_group_has_most(E, N, sizes, kind):
    """16 rows of a group at a time"""
    K, P = 200, sum(sizes.values())
    assert plan.grouped(kind, E, K, N, P, P)[0] == STREAM
    g = torch.Generator(device=DEV).manual_seed(N)
    weight, x, more, rows = _case(kind, E, K, N, P, g)
    ends, want = [0], []
    for e in range(E):
        n = sizes.get(e, 0)
        if n:
            want.append(rows(torch.arange(ends[-1], ends[-1] + n, device=DEV), e))
        ends.append(ends[-1] + n)
    assert torch.equal(rq.grouped_mul_mat(weight, x, _ints(ends), dtype=torch.float32, **more), torch.cat(want))


# ---- the tiles --------------------------------------------------------------------------------------------------------------

# of the plan: rows and positions of a tile, whether tiles are shared, tiles a compute unit holds; then kind, E, K, N, P that reach it
FORMS = [((64, 64, False, 2), F16, 3, 72, 70, 130), ((64, 64, True, 2), F16, 1, 1806, 16, 18), ((128, 64, False, 2), F16, 4, 33, 8804, 25),
         ((128, 64, True, 2), F16, 64, 3602, 70, 267), ((128, 128, False, 1), F16, 1, 301, 2389, 847), ((128, 128, False, 2), F16, 64, 32, 1003, 2339),
         ((128, 128, True, 1), F16, 1, 4487, 449, 2084), ((256, 256, False, 1), F16, 8, 32, 5616, 1009), ((64, 64, True, 2), BF16, 1, 1806, 16, 18),
         ((128, 64, False, 2), BF16, 4, 33, 8804, 25), ((128, 64, True, 2), BF16, 64, 3602, 70, 267), ((128, 128, False, 1), BF16, 1, 301, 2389, 847),
         ((128, 128, False, 2), BF16, 64, 32, 1003, 2339), ((128, 128, True, 1), BF16, 1, 4487, 449, 2084), ((256, 256, False, 1), BF16, 8, 32, 5616, 1009),
         ((64, 64, False, 2), I8, 3, 72, 70, 130), ((64, 64, True, 2), I8, 1, 3499, 17, 17), ((128, 64, False, 2), I8, 40, 42, 816, 166), ((128, 64, True, 2), I8, 64, 7879, 66, 261),
         ((128, 128, False, 1), I8, 1, 588, 7186, 263), ((128, 128, False, 2), I8, 64, 32, 1003, 2339), ((128, 128, True, 1), I8, 1, 8744, 226, 4168),
         ((256, 256, False, 1), I8, 4, 34, 11065, 499)]


@pytest.mark.parametrize("form,kind,E,K,N,P", FORMS)
def test_grouped_of_every_form_to_the_bit(form, kind, E, K, N, P):
    """rows that are gathered, one of them not there, ragged groups, outputs in an order of their own, what the workspace held"""
    M = P // 2 + 1
    p = plan.grouped(kind, E, K, N, M, P)
    assert (p[1], p[2], p[6] > 1, p[7]) == form, p
    g = torch.Generator(device=DEV).manual_seed(K + N + P)
    weight, x, more, rows = _case(kind, E, K, N, M, g)
    cuts = sorted(torch.randint(0, P - 1, (E - 1,), generator=torch.Generator().manual_seed(P)).tolist())
    ends = [0] + cuts + [P - 1]   # (the last position is no group's)
    read = torch.randint(0, M, (P,), device=DEV, generator=g)
    places = torch.randperm(P, device=DEV, generator=g)
    want = torch.zeros((P, N), device=DEV)
    for e, (i, j) in enumerate(zip(ends, ends[1:])):
        if i < j:
            want[places[i:j]] = rows(read[i:j], e)
    want[places[3]], want[places[P - 1]] = 0, 7
    read[3] = M
    ws = torch.empty((rq.grouped_workspace_bytes(weight, M, P),), dtype=torch.uint8, device=DEV)
    out = torch.empty((P, N), device=DEV)
    for fill in (0, 255):
        ws.fill_(fill), out.fill_(7)
        rq.grouped_mul_mat(weight, x, _ints(ends), rows=read.int(), out_rows=places.int(), out=out, workspace=ws, **more)
        assert torch.equal(out, want)
    half = torch.full((P, N), 7.0, dtype=torch.bfloat16, device=DEV)
    rq.grouped_mul_mat(weight, x, _ints(ends), rows=read.int(), out_rows=places.int(), out=half, **more)
    assert torch.equal(half, want.bfloat16())


# (rows and positions of a tile, tiles a compute unit holds), N, M, the steps of 64 bytes from which on that is the plan
STEPS = [((64, 64, 2), 33, 17, 1), ((128, 64, 2), 16500, 65, 1), ((128, 64, 2), 16500, 17, 8), ((128, 128, 2), 16500, 200, 1), ((128, 128, 1), 16500, 65, 10), ((256, 256, 1), 16500, 400, 1)]


@pytest.mark.parametrize("form,N,M,first", STEPS)
def test_every_number_of_steps(form, N, M, first):
    """rows whose last step, pair of steps and turn of the rings end anywhere; the weight and x as they lie, by one more row of x than is looked at"""
    last = 7 if (form, M) == ((128, 64, 2), 65) else 24
    g = torch.Generator(device=DEV).manual_seed(M)
    for steps in range(first, last + 1):
        K = 64 * steps
        p = plan.product(K, N, M)
        assert (p[1], p[2], p[7]) == form and p[6] == 1, p
        room, w, t, s = _codes((M + 1, K), g), _codes((N, K), g), _scales((N,), g), _scales((M,), g)
        assert torch.equal(rq.i8_mul_mat(rq.I8Weight(w, t), room[:M], scales=s), _scaled(room[:M], w, s, t)), steps


@pytest.mark.parametrize("form,N,M,steps", [((64, 64, 2), 33, 17, range(60, 86)), ((128, 64, 2), 8200, 17, range(136, 152)), ((128, 128, 1), 8200, 65, range(136, 152))])
def test_every_number_of_steps_of_shared_tiles(form, N, M, steps):
    """parts of equal length but the last"""
    g = torch.Generator(device=DEV).manual_seed(M)
    for n in steps:
        K = 64 * n - 5
        p = plan.product(K, N, M)
        assert (p[1], p[2], p[7]) == form and p[6] > 1, p
        a, w, t, s = _codes((M, K), g), _codes((N, K), g), _scales((N,), g), _scales((M,), g)
        assert torch.equal(rq.i8_mul_mat(rq.I8Weight(w, t), a, scales=s), _scaled(a, w, s, t)), n


# ---- both -------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", [I8, F16, BF16])
@pytest.mark.parametrize("P,form", [(9, STREAM), (300, TILES)])
def test_one_row_read_by_all_and_one_written(P, form, kind):
    E, K, N = 2, 65, 33
    assert plan.grouped(kind, E, K, N, 1, P)[0] == form
    g = torch.Generator(device=DEV).manual_seed(P)
    weight, x, more, rows = _case(kind, E, K, N, 1, g)
    want = torch.cat([rows(torch.zeros(n, dtype=torch.long, device=DEV), e) for e, n in enumerate((P // 3, P - P // 3))])
    offsets, read = _ints([0, P // 3, P]), torch.zeros(P, dtype=torch.int32, device=DEV)
    assert torch.equal(rq.grouped_mul_mat(weight, x, offsets, rows=read, dtype=torch.float32, **more), want)
    places = torch.full((P,), -1, dtype=torch.int32, device=DEV)
    places[P - 2], places[1] = 0, 1
    out = torch.full((1, N), 7.0, device=DEV)
    assert torch.equal(rq.grouped_mul_mat(weight, x, offsets, rows=read, out_rows=places, out=out, **more), want[P - 2:P - 1])


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("P,form", [(9, STREAM), (200, TILES)])
def test_an_infinity_or_nan_in_16_bits_stays_its_rows_own(P, form, kind):
    E, K, N = 1, 72, 40
    assert plan.grouped(kind, E, K, N, P, P)[0] == form
    g = torch.Generator(device=DEV).manual_seed(P)
    weight, x, _, rows = _case(kind, E, K, N, P, g)
    want = rows(torch.arange(P, device=DEV), 0)
    x[2, 71], x[P - 1, 0] = float("nan"), float("inf")
    y = rq.grouped_mul_mat(weight, x, _ints([0, P]), dtype=torch.float32)
    assert torch.isnan(y[2]).all() and not torch.isfinite(y[P - 1]).any()
    y[2], y[P - 1] = want[2], want[P - 1]
    assert torch.equal(y, want)


@pytest.mark.parametrize("kind,least", [(F16, -24), (BF16, -133)])
@pytest.mark.parametrize("P,form", [(9, STREAM), (200, TILES)])
def test_the_smallest_numbers_of_16_bits_count(P, form, kind, least):
    """numbers below the type's normal ones, in either operand, against whole numbers (powers of two: every product and sum is exact in fp32)"""
    E, K, N = 1, 72, 40
    assert plan.grouped(kind, E, K, N, P, P)[0] == form
    g = torch.Generator(device=DEV).manual_seed(P)
    dtype = torch.float16 if kind == F16 else torch.bfloat16
    x, w = _small((P, K), g), _small((E, N, K), g)
    want = x.double() @ w[0].double().t().contiguous()
    tiny = lambda v: (v.double() * 2.0 ** least).to(dtype)  # noqa: E731
    for big, a, b in ((2.0 ** 10, tiny(x), (w * 2.0 ** 10).to(dtype)), (2.0 ** 10, (x * 2.0 ** 10).to(dtype), tiny(w))):
        y = rq.grouped_mul_mat(rq.HalfWeight(b), a, _ints([0, P]), dtype=torch.float32)
        assert torch.equal(y.double(), want * 2.0 ** least * big)


# ---- a layer's products, each to the bit ----------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,absent", [(1, False), (2, True), (5, False), (50, True), (400, False)])
def test_products_of_a_layer_are_the_definition(M, absent, dtype):
    """route, sort, up where the tokens lie, an activation, down to the slots' places; slots whose expert is not here give zeros in a buffer of zeros"""
    E, K, F, top = 12, 256, 96, 3
    g = torch.Generator(device=DEV).manual_seed(M)
    up, down = ((_codes((E, n, k), g), _scales((E, n), g) * k ** -0.5 / 64) for n, k in ((F, K), (K, F)))
    x = _floats(M, K, dtype, g)
    ids, shares = rq.route(torch.randn((M, E), device=DEV, generator=g), top)
    if absent:
        ids = torch.where(torch.arange(M * top, device=DEV).view(M, top) % 4 == 1, -1, ids).contiguous()
    offsets, slots, tokens = rq.sort_slots(ids, E)
    experts, here = ids.flatten().long(), ids.flatten() >= 0
    h = rq.grouped_mul_mat(rq.I8Weight(*up), x, offsets, rows=tokens, out=torch.zeros((M * top, F), dtype=dtype, device=DEV))
    a, s = rq.i8_quantize(x)
    want = torch.zeros((M * top, F), dtype=dtype, device=DEV)   # (by slot)
    for i in here.nonzero().flatten().tolist():
        m, e = i // top, experts[i]
        want[i] = _scaled(a[m:m + 1], up[0][e], s[m:m + 1], up[1][e])[0].to(dtype)
    assert torch.equal(h, want[slots.long()])
    h = torch.relu(h)
    y = rq.grouped_mul_mat(rq.I8Weight(*down), h, offsets, out_rows=slots, out=torch.zeros((M * top, K), device=DEV))
    a, s = rq.i8_quantize(torch.relu(want))
    want = torch.zeros((M * top, K), device=DEV)
    for i in here.nonzero().flatten().tolist():
        want[i] = _scaled(a[i:i + 1], down[0][experts[i]], s[i:i + 1], down[1][experts[i]])[0]
    assert torch.equal(y, want)
    assert torch.isfinite((y.view(M, top, K) * shares[:, :, None]).sum(dim=1)).all()


# ---- sort, and sizes that take several launches --------------------------------------------------------------------------------

@pytest.mark.parametrize("E", [1, 63, 64, 65, 1023, 1024])
@pytest.mark.parametrize("M,top", [(2048, 1), (2049, 1), (1, 1024), (131072, 1), (131073, 1), (2 ** 22, 1), (2 ** 21, 2)])
def test_sort_on_both_sides_of_its_runs(M, top, E):
    """one run and two, the last of the short runs and the first long ones, the most slots of a call"""
    g = torch.Generator(device=DEV).manual_seed(E + M)
    ids = torch.randint(-1, E + 1, (M, top), dtype=torch.int32, device=DEV, generator=g)
    expert = torch.where(ids.flatten() < 0, E, ids.flatten())
    order = expert.sort(stable=True)
    ends = torch.searchsorted(order.values, torch.arange(E + 1, device=DEV, dtype=torch.int32))
    n = rq.load_library().rq_sort_workspace_bytes(M, top, E)
    assert (n == 0) == (M * top <= 2048)
    ws = torch.full((max(n, 1),), 255, dtype=torch.uint8, device=DEV)
    for workspace in (None, ws[:n]):
        offsets, slots, tokens = rq.sort_slots(ids, E, workspace=workspace)
        assert torch.equal(offsets, ends.int()) and torch.equal(slots, order.indices.int()) and torch.equal(tokens, slots // top)


def test_quantiser_of_more_rows_than_a_launch_has():
    """2^24 rows of up to 2048 inputs are one launch"""
    M, K = 2 ** 24 + 5, 3
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn((M, K), device=DEV, generator=g)
    codes, scales = rq.i8_quantize(x)
    some = torch.tensor([0, 1, 2 ** 24 - 1, 2 ** 24, 2 ** 24 + 1, M - 1], device=DEV)
    a, s = rq.i8_quantize(x[some])
    assert torch.equal(codes[some], a) and torch.equal(scales[some], s)
    assert torch.equal(scales, torch.maximum(x.abs().amax(dim=1) * torch.tensor(1 / 127, device=DEV), torch.tensor(2.0 ** -126, device=DEV)))
    assert ((rq.i8_dequantize(codes, scales) - x).abs() <= scales[:, None] * 0.5001).all()


def test_dequantiser_of_more_elements_than_a_launch_has():
    """2^31 runs of eight elements are one launch"""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    M = 2 ** 31 + 7
    codes = torch.full((M, 1), 3, dtype=torch.int8, device=DEV)
    codes[2 ** 31:] = -5
    out = rq.i8_dequantize(codes, torch.full((M,), 0.5, device=DEV), dtype=torch.float16)
    assert bool((out[:2 ** 31] == 1.5).all()) and bool((out[2 ** 31:] == -2.5).all())


def test_rows_brought_to_16_bytes_in_several_launches():
    """rows at odd addresses, more of them than one launch moves, read by few positions in tiles"""
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    M, K, N, P = 140001, 131071, 24, 40
    assert plan.grouped(I8, 1, K, N, M, P)[0] == TILES
    g = torch.Generator(device=DEV).manual_seed(3)
    a = torch.zeros((M, K), dtype=torch.int8, device=DEV)
    some = torch.tensor([0, 1, 65536, 130000, 131007, 131008, 131071, 131072, M - 2, M - 1], device=DEV)
    a[some] = _codes((10, K), g)
    w, t, s = _codes((N, K), g), _scales((N,), g), _scales((M,), g)
    read = some.repeat(4)
    y = rq.grouped_mul_mat(rq.I8Weight(w[None], t[None]), a, _ints([0, P]), rows=read.int(), scales=s)
    assert torch.equal(y, _scaled(a[read], w, s[read], t))


# ---- the smallest sizes, strides of given codes, graphs ------------------------------------------------------------------------

@pytest.mark.parametrize("kind", [I8, F16, BF16])
@pytest.mark.parametrize("K", [1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33])
def test_smallest_sizes(K, kind):
    g = torch.Generator(device=DEV).manual_seed(K)
    for P, form in ((1, STREAM), (5, STREAM), (40, TILES)):
        for N in (1, 2, 33):
            assert plan.grouped(kind, 2, K, N, P, P)[0] == form
            weight, x, more, rows = _case(kind, 2, K, N, P, g)
            want = torch.cat([rows(torch.arange(0, P // 2, device=DEV), 0), rows(torch.arange(P // 2, P, device=DEV), 1)])
            assert torch.equal(rq.grouped_mul_mat(weight, x, _ints([0, P // 2, P]), dtype=torch.float32, **more), want)


@pytest.mark.parametrize("P,form", [(12, STREAM), (90, TILES)])
@pytest.mark.parametrize("K,offset,ld", [(192, 0, 208), (192, 1, 208), (192, 16, 193), (187, 3, 197), (5, 1, 5)])
def test_groups_of_given_codes_at_any_address(K, offset, ld, P, form):
    E, N, M = 3, 50, P + 3
    assert plan.grouped(I8, E, K, N, M, P)[0] == form
    g = torch.Generator(device=DEV).manual_seed(K + ld)
    room = _codes((M * ld + 64,), g)
    a, w, s, t = room.as_strided((M, K), (ld, 1), offset), _codes((E, N, K), g), _scales((M,), g), _scales((E, N), g)
    read = torch.randint(0, M, (P,), device=DEV, generator=g)
    ends = [0, P // 4, P // 4, P]
    want = torch.cat([_scaled(a[read[i:j]], w[e], s[read[i:j]], t[e]) for e, (i, j) in enumerate(zip(ends, ends[1:]))])
    assert torch.equal(rq.grouped_mul_mat(rq.I8Weight(w, t), a, _ints(ends), rows=read.int(), scales=s), want)


@pytest.mark.parametrize("kind,E,K,N,P", [(F16, 64, 3602, 70, 267), (I8, 64, 7879, 66, 261), (I8, 8, 200, 70, 8)])
def test_captured_groups_whose_sizes_change(kind, E, K, N, P):
    """shared tiles, and rows few: one graph, other offsets at every replay, another call on the same workspace between"""
    p = plan.grouped(kind, E, K, N, P, P)
    assert p[6] > 1 or p[0] == STREAM
    g = torch.Generator(device=DEV).manual_seed(P)
    weight, x, more, rows = _case(kind, E, K, N, P, g)
    offsets, out = _ints([0] * (E + 1)), torch.zeros((P, N), device=DEV)
    ws = torch.empty((rq.grouped_workspace_bytes(weight, P, P),), dtype=torch.uint8, device=DEV)
    rq.grouped_mul_mat(weight, x, offsets, out=out, workspace=ws, **more)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rq.grouped_mul_mat(weight, x, offsets, out=out, workspace=ws, **more)
    for turn in range(6):
        pick = torch.Generator().manual_seed(turn)
        cuts = [0] * (E - 1) if turn == 0 else [P] * (E - 1) if turn == 1 else sorted(torch.randint(0, P + 1, (E - 1,), generator=pick).tolist())
        ends = [0] + cuts + [P]
        want = torch.full((P, N), 7.0, device=DEV)
        for e, (i, j) in enumerate(zip(ends, ends[1:])):
            if i < j:
                want[i:j] = rows(torch.arange(i, j, device=DEV), e)
        offsets.copy_(_ints(ends)), out.fill_(7), ws.fill_(255 * (turn & 1))
        graph.replay()
        assert torch.equal(out, want), turn
        out.fill_(7)
        rq.grouped_mul_mat(weight, x, offsets, out=out, workspace=ws, **more)
        assert torch.equal(out, want), turn
