"""The int8 quantiser, dequantiser and product, the sort of slots and the products grouped by expert on the GPU, against their definitions
in 64 bits (numpy, host)."""
import numpy as np
import pytest
import torch

import ruquant_amd as rq
from tests import i8_oracle as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
HALF = {"fp16": torch.float16, "bf16": torch.bfloat16}
ROUNDING = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _gpu(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).to(DEV)
    return t if dtype is None else t.to(dtype)


def _host(t):
    return t.detach().to(torch.float64).cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def _values(M, K, seed, dtype=torch.float32):
    """rows of different magnitudes with some large elements; the tensor and its values in 64 bits"""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((M, K)) * np.exp2(rng.integers(-6, 7, size=(M, 1)))
    x[rng.random((M, K)) < 0.01] *= 8
    t = _gpu(x.astype(np.float32), dtype)
    return t, _host(t)


def _weights(shape, K, seed):
    rng = np.random.default_rng(seed)
    codes = rng.integers(-127, 128, size=(*shape, K), dtype=np.int8)
    return codes, (rng.uniform(0.5, 1.5, size=shape) * K ** -0.5 / 64).astype(np.float32)


def _same(got, want32):
    """got: a tensor whose values are the fp32 numbers want32 rounded once to its type"""
    want = torch.from_numpy(np.ascontiguousarray(want32)).to(got.dtype)
    got = got.cpu()
    assert got.shape == want.shape
    bad = ~((got == want) | (torch.isnan(got) & torch.isnan(want)))
    assert not bad.any(), "%d of %d differ, the first at %s: %r, not %r" % (
        bad.sum(), bad.numel(), bad.nonzero()[0].tolist(), got[bad][0].item(), want[bad][0].item())


# ---- quantiser and dequantiser -------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("M,K", [(1, 1), (3, 7), (1, 5120), (9, 64), (65, 2047), (5, 2049), (7, 4128), (2, 8193), (3, 17408), (2, 40001)])
def test_quantize_matches_definition(M, K, dtype):
    x, x64 = _values(M, K, 10 * M + K, DTYPES[dtype])
    codes, scales = rq.i8_quantize(x)
    want_codes, want_scales = ref.quantize(x64)
    assert codes.dtype == torch.int8 and scales.dtype == torch.float32
    assert (scales.cpu().numpy() == want_scales).all()
    assert (codes.cpu().numpy() == want_codes).all()


def test_quantize_ties_and_extremes():
    """Every tie between two codes, next to every tie, denormals, the largest numbers, zeros."""
    halves = np.arange(-126.5, 127, 1.0)
    rows = []
    for unit in (2.0 ** -149, 2.0 ** -140, 2.0 ** -126, 2.0 ** -30, 1.0, 2.0 ** 100):
        for step in (0, 1, -1):
            v = (halves * unit).astype(np.float32)
            v = v if step == 0 else np.nextafter(v, np.float32(np.inf * step))
            rows.append(np.concatenate([v, np.float32([127 * unit, 0.0])]))
    rows += [np.zeros(256), np.full(256, np.finfo(np.float32).max), np.full(256, -2.0 ** -149)]
    rows += [np.where(np.arange(256) == 3, 3e38, 1e-38)]
    x = np.stack(rows).astype(np.float32)
    codes, scales = rq.i8_quantize(_gpu(x))
    want_codes, want_scales = ref.quantize(x.astype(np.float64))
    assert (scales.cpu().numpy() == want_scales).all()
    assert (codes.cpu().numpy() == want_codes).all()


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("K", [96, 97, 5000])
def test_rows_with_infinities_or_nan_become_nan(K, dtype):
    x = torch.ones((4, K), dtype=DTYPES[dtype], device=DEV)
    x[0, 5], x[1, K - 1], x[2, 0] = float("nan"), float("inf"), float("-inf")
    codes, scales = rq.i8_quantize(x)
    assert torch.isnan(scales[:3]).all() and not torch.isnan(scales[3])
    assert (codes[:3] == 0).all() and (codes[3] == 127).all()
    y = rq.i8_dequantize(codes, scales, dtype=DTYPES[dtype])
    assert torch.isnan(y[:3]).all() and torch.isfinite(y[3]).all()


def test_a_nan_with_any_payload_has_zero_codes():
    x = np.ones((2, 64), dtype=np.float32)
    x[0, 7] = np.array([0x7FC000FF], dtype=np.uint32).view(np.float32)[0]
    x[1, 8] = np.array([0xFF8000AA], dtype=np.uint32).view(np.float32)[0]
    codes, scales = rq.i8_quantize(_gpu(x))
    assert (codes == 0).all() and torch.isnan(scales).all()


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("offset,ld", [(0, 192), (1, 192), (0, 193), (3, 197)])
def test_quantize_reads_any_rows(offset, ld, dtype):
    x, _ = _values(9, 192, 3, DTYPES[dtype])
    room = torch.full((9 * 200,), float("nan"), dtype=DTYPES[dtype], device=DEV)
    view = room.as_strided((9, 192), (ld, 1), offset)
    view.copy_(x)
    for a, b in zip(rq.i8_quantize(view), rq.i8_quantize(x)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("K", [256, 251])
def test_dequantize(K, dtype):
    codes = np.tile(np.arange(-128, 128).astype(np.int8)[:K], (7, 1))
    scales = np.array([1.0, 0.3, 2.0 ** -126, 1e-3, 1e30, np.nan, 0.0], dtype=np.float32)
    _same(rq.i8_dequantize(_gpu(codes), _gpu(scales), dtype=DTYPES[dtype]), codes.astype(np.float32) * scales[:, None])


def test_dequantize_takes_more_dimensions_and_slices():
    codes, scales = _weights((3, 5), 96, 1)
    want = codes.astype(np.float32) * scales[..., None]
    _same(rq.i8_dequantize(_gpu(codes), _gpu(scales)), want)
    _same(rq.i8_dequantize(_gpu(codes)[1:, 1:3, 1:], _gpu(scales)[1:, 1:3]), want[1:, 1:3, 1:])


def test_empty_tensors():
    codes, scales = rq.i8_quantize(torch.empty((0, 64), device=DEV))
    assert codes.shape == (0, 64) and scales.shape == (0,)
    assert rq.i8_dequantize(codes, scales).shape == (0, 64)
    W = rq.I8Weight(*(_gpu(a) for a in _weights((9,), 64, 1)))
    assert rq.i8_mul_mat(W, torch.empty((0, 64), device=DEV)).shape == (0, 9)


# ---- product ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (1, 64, 16), (2, 63, 33), (1, 5120, 100), (5, 200, 16), (13, 4099, 77), (16, 128, 640),
                                   (17, 65, 65), (33, 1000, 130), (64, 576, 64), (65, 640, 200), (100, 31, 129), (129, 2048, 257),
                                   (257, 100, 300), (300, 1472, 513)])
def test_product_is_the_definition(M, K, N, dtype):
    x, x64 = _values(M, K, M + K + N, DTYPES[dtype])
    codes, scales = _weights((N,), K, K)
    W = rq.I8Weight(_gpu(codes), _gpu(scales))
    a, s = ref.quantize(x64)
    want = ref.scaled(a, codes, s, scales)
    y = rq.i8_mul_mat(W, x)
    assert y.dtype == DTYPES[dtype]
    _same(y, want)
    _same(rq.i8_mul_mat(W, _gpu(a), scales=_gpu(s), dtype=DTYPES[dtype]), want)
    _same(rq.i8_mul_mat(W, _gpu(a), scales=_gpu(s)), want)


@pytest.mark.parametrize("M", [1, 16, 40, 300])
def test_product_of_the_longest_rows(M):
    """the sum of K = 131071 products of -128 by -128 stays below 2^31"""
    K, N = 131071, 33
    a = np.full((M, K), -128, dtype=np.int8)
    a[M // 2, ::3] = 127
    w = np.full((N, K), -128, dtype=np.int8)
    w[N - 1] = np.random.default_rng(1).integers(-128, 128, size=K)
    s, t = np.linspace(0.5, 2, M).astype(np.float32), np.linspace(1e-9, 2e-9, N).astype(np.float32)
    _same(rq.i8_mul_mat(rq.I8Weight(_gpu(w), _gpu(t)), _gpu(a), scales=_gpu(s)), ref.scaled(a, w, s, t))


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("M", [3, 40, 150])
@pytest.mark.parametrize("offset,ld", [(0, 200), (1, 200), (0, 193), (5, 197)])
def test_product_reads_and_writes_any_rows(M, offset, ld, dtype):
    K, N = 192, 70
    x, x64 = _values(M, K, 5, DTYPES[dtype])
    codes, scales = _weights((N,), K, 6)
    W = rq.I8Weight(_gpu(codes), _gpu(scales))
    a, s = ref.quantize(x64)
    want = ref.scaled(a, codes, s, scales)
    room = torch.full((M * ld + 8,), float("nan"), dtype=DTYPES[dtype], device=DEV)
    view = room.as_strided((M, K), (ld, 1), offset)
    view.copy_(x)
    out = torch.full((M * 100 + 8,), 7.0, dtype=DTYPES[dtype], device=DEV)
    y = out.as_strided((M, N), (N + offset, 1), offset)
    assert rq.i8_mul_mat(W, view, out=y) is y
    _same(y, want)
    kept = torch.ones_like(out, dtype=torch.bool)
    kept.as_strided((M, N), (N + offset, 1), offset)[:] = False
    assert (out[kept] == 7).all()
    given = torch.zeros((M * ld + 8,), dtype=torch.int8, device=DEV).as_strided((M, K), (ld, 1), offset)
    given.copy_(_gpu(a))
    _same(rq.i8_mul_mat(W, given, scales=_gpu(s), dtype=DTYPES[dtype]), want)


@pytest.mark.parametrize("M", [4, 30, 200])
def test_a_nan_stays_its_tokens_and_rows_own(M):
    x, x64 = _values(M, 300, 8)
    x[1, 7], x[M - 1, 299] = float("nan"), float("inf")
    x64 = _host(x)
    codes, scales = _weights((50,), 300, 9)
    scales[3] = np.nan
    a, s = ref.quantize(x64)
    y = rq.i8_mul_mat(rq.I8Weight(_gpu(codes), _gpu(scales)), x)
    _same(y, ref.scaled(a, codes, s, scales))
    assert torch.isnan(y[1]).all() and torch.isnan(y[:, 3]).all() and torch.isfinite(y[0, :3]).all()


@pytest.mark.parametrize("M", [1, 16, 70, 400])
def test_what_a_workspace_held_does_not_matter(M):
    x, x64 = _values(M, 1000, 2)
    codes, scales = _weights((200,), 1000, 3)
    W = rq.I8Weight(_gpu(codes), _gpu(scales))
    want = rq.i8_mul_mat(W, x)
    ws = W.workspace(M)
    for fill in (0, 255, 127):
        ws.fill_(fill)
        assert torch.equal(rq.i8_mul_mat(W, x, workspace=ws), want)
    a, s = ref.quantize(x64)
    _same(want, ref.scaled(a, codes, s, scales))


# ---- sort ------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("M,top,E", [(1, 1, 1), (1, 8, 64), (3, 2, 5), (37, 4, 60), (1000, 1, 3), (1024, 8, 1024), (1025, 8, 256), (8191, 1, 7),
                                     (16384, 8, 256), (70001, 3, 33), (0, 2, 4)])
def test_sort(M, top, E):
    rng = np.random.default_rng(M + E)
    ids = rng.integers(0, E, size=(M, top)).astype(np.int32)
    ids[rng.random((M, top)) < 0.2] = -1
    ids[rng.random((M, top)) < 0.1] = E
    ids[rng.random((M, top)) < 0.05] = np.iinfo(np.int32).max
    ids[rng.random((M, top)) < 0.05] = np.iinfo(np.int32).min
    got = rq.sort_slots(_gpu(ids), E)
    for g, w in zip(got, ref.sort(ids, E)):
        assert g.dtype == torch.int32 and (g.cpu().numpy() == w).all()


@pytest.mark.parametrize("which", [0, -1, 511])
def test_sort_of_one_expert(which):
    ids = np.full((5000, 8), which, dtype=np.int32)
    for g, w in zip(rq.sort_slots(_gpu(ids), 512), ref.sort(ids, 512)):
        assert (g.cpu().numpy() == w).all()


# ---- products grouped by expert ------------------------------------------------------------------------------------------

def _sizes(kind, E, seed):
    rng = np.random.default_rng(seed)
    if kind == "ones":
        return np.ones(E, dtype=np.int64)
    if kind == "few":
        return rng.integers(0, 4, size=E)
    if kind == "one_has_all":
        return np.where(np.arange(E) == E // 2, 333, 0)
    if kind == "ragged":
        return rng.choice([0, 0, 1, 2, 15, 16, 17, 31, 33, 64, 65, 100, 129], size=E)
    return rng.integers(100, 300, size=E)


class _Case:
    """x, weights, offsets and what comes out, for int8 (bits) and 16-bit weights (values and bounds)"""

    def __init__(self, kind, type_, K, N, sizes, M, seed, dtype=None):
        rng = np.random.default_rng(seed)
        E = len(sizes)
        self.E, self.N, self.P = E, N, int(sizes.sum())
        self.type = type_
        self.offsets = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
        self.M = M or self.P
        self.x, self.x64 = _values(self.M, K, seed + 1, dtype or DTYPES.get(type_, torch.float32))
        self.rows = rng.integers(0, self.M, size=self.P).astype(np.int32) if M else np.arange(self.P, dtype=np.int32)
        self.expert = np.repeat(np.arange(E), sizes)
        if type_ == "int8":
            self.codes, self.scales = _weights((E, N), K, seed + 2)
            self.weight = rq.I8Weight(_gpu(self.codes), _gpu(self.scales))
            a, s = ref.quantize(self.x64)
            self.given = _gpu(a), _gpu(s)
            self.want = np.zeros((self.P, N), dtype=np.float32)
            for e in np.unique(self.expert):
                p = np.flatnonzero(self.expert == e)
                self.want[p] = ref.scaled(a[self.rows[p]], self.codes[e], s[self.rows[p]], self.scales[e])
        else:
            w = _gpu(rng.standard_normal((E, N, K)).astype(np.float32) * K ** -0.5, DTYPES[type_])
            self.weight, w64 = rq.HalfWeight(w), _host(w)
            self.want, self.size = np.zeros((self.P, N)), np.zeros((self.P, N))
            for e in np.unique(self.expert):
                p = np.flatnonzero(self.expert == e)
                self.want[p] = self.x64[self.rows[p]] @ w64[e].T
                self.size[p] = np.abs(self.x64[self.rows[p]]) @ np.abs(w64[e]).T
        self.K = K

    def check(self, y, places=None):
        """rows `places` of y (all) are positions 0 .."""
        y = y if places is None else y[torch.from_numpy(places.astype(np.int64)).to(DEV)]
        if self.type == "int8":
            return _same(y, self.want)
        # Products of two 16-bit numbers are exact in fp32. One matrix instruction adds at most 32 of them to a sum, and a sum passes at most
        # K / 16 instructions and the join of 8 wavefronts; each addition is within 2^-24 of what it adds up, twice that if it cuts.
        bound = 2 * (self.K / 16 + 48) * 2.0 ** -24 * self.size + ROUNDING[y.dtype] * 1.01 * np.abs(self.want)
        if y.dtype == torch.float16:
            bound = bound + 2.0 ** -25
        off = np.abs(_host(y) - self.want)
        assert y.shape == self.want.shape and (off <= bound).all(), "off by %g times the bound" % (off / bound).max()


@pytest.mark.parametrize("type_", ["int8", "fp16", "bf16"])
@pytest.mark.parametrize("kind,E,K,N", [("ones", 8, 256, 48), ("few", 64, 129, 100), ("one_has_all", 5, 64, 64), ("ragged", 60, 264, 130),
                                        ("ragged", 7, 1001, 33), ("many", 3, 512, 257), ("ragged", 1, 72, 16), ("few", 1024, 32, 17)])
def test_grouped(kind, E, K, N, type_):
    c = _Case(kind, type_, K, N, _sizes(kind, E, E + K), 0, K + N)
    y = rq.grouped_mul_mat(c.weight, c.x, _gpu(c.offsets))
    assert y.dtype == c.x.dtype
    c.check(y)


@pytest.mark.parametrize("type_", ["int8", "fp16", "bf16"])
@pytest.mark.parametrize("kind,E", [("few", 40), ("ragged", 24), ("many", 4)])
def test_grouped_reads_rows_where_they_lie_and_writes_to_places(kind, E, type_):
    c = _Case(kind, type_, 200, 90, _sizes(kind, E, E), 61, E)
    rng = np.random.default_rng(E)
    places = rng.permutation(c.P + 40)[:c.P].astype(np.int32)
    for dtype in (torch.float32, c.x.dtype, torch.bfloat16):
        out = torch.full((c.P + 40, 90), 7.0, dtype=dtype, device=DEV)
        y = rq.grouped_mul_mat(c.weight, c.x, _gpu(c.offsets), rows=_gpu(c.rows), out_rows=_gpu(places), out=out)
        assert y is out
        c.check(y, places)
        left = np.setdiff1d(np.arange(c.P + 40), places)
        assert (y[torch.from_numpy(left).to(DEV)] == 7).all()
    c.check(rq.grouped_mul_mat(c.weight, c.x, _gpu(c.offsets), rows=_gpu(c.rows)))


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("kind,E", [("few", 30), ("many", 3)])
def test_grouped_int8_takes_every_type_and_given_codes(kind, E, dtype):
    c = _Case(kind, "int8", 333, 50, _sizes(kind, E, E), 40, E, dtype=DTYPES[dtype])
    c.check(rq.grouped_mul_mat(c.weight, c.x, _gpu(c.offsets), rows=_gpu(c.rows)))
    a, s = c.given
    c.check(rq.grouped_mul_mat(c.weight, a, _gpu(c.offsets), rows=_gpu(c.rows), scales=s, dtype=DTYPES[dtype]))
    c.check(rq.grouped_mul_mat(c.weight, a, _gpu(c.offsets), rows=_gpu(c.rows), scales=s))


@pytest.mark.parametrize("type_", ["int8", "fp16"])
@pytest.mark.parametrize("kind,E", [("few", 16), ("many", 2)])
def test_indices_outside(kind, E, type_):
    """a row that is not there reads as zeros, a place that is not there is not written"""
    c = _Case(kind, type_, 96, 40, _sizes(kind, E, E), 20, E)
    rows, places = c.rows.copy(), np.arange(c.P, dtype=np.int32)
    rows[0], rows[1], rows[2] = -1, 20, np.iinfo(np.int32).max
    places[3], places[4], places[5] = -1, c.P, np.iinfo(np.int32).min
    out = torch.full((c.P, 40), 7.0, device=DEV)
    c.x[5] = float("nan")
    rows[6:] = np.where(rows[6:] == 5, 4, rows[6:])
    rq.grouped_mul_mat(c.weight, c.x, _gpu(c.offsets), rows=_gpu(rows), out_rows=_gpu(places), out=out)
    assert (out[:3] == 0).all() and (out[3:6] == 7).all()
    assert torch.isfinite(out).all() and (out[6:] != 7).any()


@pytest.mark.parametrize("type_", ["int8", "bf16"])
@pytest.mark.parametrize("few", [True, False])
def test_rows_of_no_group_are_left(few, type_):
    sizes = np.array([3, 0, 2, 1]) if few else np.array([70, 0, 33, 129])
    c = _Case("", type_, 128, 64, sizes, 0, 5)
    x = torch.cat([c.x, torch.full((50, 128), float("nan"), dtype=c.x.dtype, device=DEV)])
    out = torch.full((c.P + 50, 64), 7.0, dtype=c.x.dtype, device=DEV)
    rq.grouped_mul_mat(c.weight, x, _gpu(c.offsets), out=out)
    c.check(out[:c.P])
    assert (out[c.P:] == 7).all()


@pytest.mark.parametrize("type_", ["int8", "bf16"])
def test_offsets_are_clamped(type_):
    """ends behind the last position end there, starts in front of the first start there, groups that end in front of their start are empty"""
    c = _Case("", type_, 64, 32, np.array([4, 6, 10, 0]), 0, 7)
    offsets = np.array([-5, 4, 10, 1000, 900], dtype=np.int32)
    c.check(rq.grouped_mul_mat(c.weight, c.x, _gpu(offsets)))


def test_no_group_has_rows():
    c = _Case("", "int8", 64, 32, np.array([4, 6]), 0, 7)
    out = torch.full((10, 32), 7.0, device=DEV)
    rq.grouped_mul_mat(c.weight, c.x, _gpu(np.zeros(3, dtype=np.int32)), out=out)
    assert (out == 7).all()
    assert rq.grouped_mul_mat(c.weight, c.x[:0], _gpu(np.zeros(3, dtype=np.int32))).shape == (0, 32)


@pytest.mark.parametrize("type_", ["int8", "fp16", "bf16"])
@pytest.mark.parametrize("kind,E", [("few", 16), ("many", 2)])
@pytest.mark.parametrize("offset,ld", [(0, 200), (1, 200), (0, 193), (8, 208)])
def test_grouped_reads_and_writes_any_rows(kind, E, offset, ld, type_):
    c = _Case(kind, type_, 192, 70, _sizes(kind, E, E), 0, E)
    room = torch.full((c.P * ld + 16,), float("nan"), dtype=c.x.dtype, device=DEV)
    view = room.as_strided((c.P, 192), (ld, 1), offset)
    view.copy_(c.x)
    out = torch.full((c.P * 100 + 8,), 7.0, dtype=c.x.dtype, device=DEV)
    y = out.as_strided((c.P, 70), (70 + offset, 1), offset)
    c.check(rq.grouped_mul_mat(c.weight, view, _gpu(c.offsets), out=y))
    kept = torch.ones_like(out, dtype=torch.bool)
    kept.as_strided((c.P, 70), (70 + offset, 1), offset)[:] = False
    assert (out[kept] == 7).all()


@pytest.mark.parametrize("type_", ["fp16", "bf16"])
@pytest.mark.parametrize("kind,E", [("few", 16), ("many", 2)])
def test_what_lies_behind_a_row_is_not_looked_at(kind, E, type_):
    """rows of 40 elements, which end inside a step, with NaN behind them"""
    c = _Case(kind, type_, 40, 70, _sizes(kind, E, E), 0, E)
    room = torch.full((c.P, 64), float("nan"), dtype=c.x.dtype, device=DEV)
    room[:, :40] = c.x
    c.check(rq.grouped_mul_mat(c.weight, room[:, :40], _gpu(c.offsets)))


# ---- graphs, streams, all of them together --------------------------------------------------------------------------------------

class _Layer:
    """a mixture layer's step on the framework's calls: route, sort, up, an activation, down, weighted sum"""

    def __init__(self, E, K, F, top, kind):
        self.E, self.top, self.kind = E, top, kind
        rng = np.random.default_rng(E)
        self.router = _gpu((rng.standard_normal((K, E)) * K ** -0.5).astype(np.float32))
        self.up64, self.down64 = rng.standard_normal((E, F, K)) * K ** -0.5, rng.standard_normal((E, K, F)) * F ** -0.5
        self.up, self.down = self._weight(self.up64), self._weight(self.down64)

    def _weight(self, w):
        if self.kind != "int8":
            return rq.HalfWeight(_gpu(w.astype(np.float32), DTYPES[self.kind]))
        codes, scales = rq.i8_quantize(_gpu(w.astype(np.float32)).flatten(0, 1))
        return rq.I8Weight(codes.view(w.shape), scales.view(w.shape[:2]))

    def __call__(self, x):
        ids, weights = rq.route(x.float() @ self.router, self.top)
        offsets, slots, tokens = rq.sort_slots(ids, self.E)
        h = rq.grouped_mul_mat(self.up, x, offsets, rows=tokens)
        h = torch.relu(h)
        y = rq.grouped_mul_mat(self.down, h, offsets, out_rows=slots, dtype=torch.float32)
        y = (y.view(*ids.shape, -1) * weights[:, :, None]).sum(dim=1)
        return y, ids, weights


@pytest.mark.parametrize("kind", ["int8", "bf16"])
@pytest.mark.parametrize("M", [1, 50, 400])
def test_a_layer_of_them(M, kind):
    layer = _Layer(12, 256, 96, 3, kind)
    x, x64 = _values(M, 256, 1, DTYPES.get(kind, torch.float32))
    y, ids, weights = layer(x)
    ids, weights = ids.cpu().numpy(), _host(weights)
    want = np.zeros((M, 256))
    for m in range(M):
        for j in range(3):
            e = ids[m, j]
            want[m] += weights[m, j] * (layer.down64[e] @ np.maximum(layer.up64[e] @ x64[m], 0))
    off = np.linalg.norm(_host(y) - want, axis=1) / np.linalg.norm(want, axis=1)
    # Every rounding moves an operand by a vector of random direction: a row's int8 rounding by at most half a step, 1 / 254 of its largest element, which is at most
    # 64 deviations of a row of these (some elements are 8 times the others): 64 / 254 / sqrt(3) = 0.15 of the row's norm at the very worst; four roundings. bf16's: 2^-8 each.
    assert (off < (4 * 0.15 if kind == "int8" else 6 * 2.0 ** -8)).all(), off.max()


@pytest.mark.parametrize("kind", ["int8", "bf16"])
@pytest.mark.parametrize("M", [1, 50, 400])
def test_a_captured_layer_replays(M, kind):
    layer = _Layer(12, 256, 96, 3, kind)
    dtype = DTYPES.get(kind, torch.float32)
    inputs = [_values(M, 256, seed, dtype)[0] for seed in range(3)]
    want = [layer(x) for x in inputs]
    x = inputs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer(x)
    for i in (1, 2, 0, 1):
        x.copy_(inputs[i])
        graph.replay()
        torch.cuda.synchronize()
        for g, w in zip(got, want[i]):
            assert torch.equal(g, w)


@pytest.mark.parametrize("M", [2, 40, 300])
def test_calls_on_another_stream(M):
    x, x64 = _values(M, 512, 4)
    codes, scales = _weights((300,), 512, 5)
    W = rq.I8Weight(_gpu(codes), _gpu(scales))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        big = torch.randn((2048, 2048), device=DEV)
        for _ in range(5):
            big = big @ big * 1e-3
        late = x * 1.0   # (behind the products on this stream)
        y = rq.i8_mul_mat(W, late)
    side.synchronize()
    a, s = ref.quantize(x64)
    _same(y, ref.scaled(a, codes, s, scales))
