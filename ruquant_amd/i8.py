"""Products in 8-bit integers, products grouped by expert (weights in int8, fp16 or bf16) and the sort that makes such groups, over the
C ABI of include/rq_i8.h.

An int8 row of K numbers is K codes and one fp32 scale; a code c stands for c times the scale. Rounding a row: the scale is its largest
magnitude times 1 / 127, in fp32 (at least 2 ** -126), the codes are the whole numbers nearest to x times the scale's fp32 reciprocal, ties to
even. A row that holds an infinity or a NaN becomes NaN.

As in the rest of the package torch owns device memory and the stream, and every computation happens inside librq_w4a4.so, on the
current stream of the inputs' device. With `out` and `workspace` given the products allocate nothing; the other calls make their
outputs. All of them can be captured in a graph.
"""
import torch

from .lib import load_library
from .mx import _DTYPES, _dtype, _elsewhere, _output, _rows, _workspace_bytes
from .w4a4 import RqError, _check, _device_bytes, _on_device_of

_I8 = 3   # RQ_I8


def i8_quantize(x):
    """x[M, K] (fp32, fp16 or bf16) -> codes [M, K] int8, scales [M] fp32, a scale per row."""
    M, K, ldx = _rows(x, "i8_quantize")
    dt = _dtype(x.dtype, "i8_quantize")
    if K == 0:
        raise RqError("i8_quantize: rows of no elements have no scale")
    codes = x.new_empty((M, K), dtype=torch.int8)
    scales = x.new_empty((M,), dtype=torch.float32)
    if M:
        rc = _on_device_of(x, load_library().rq_i8_quantize, dt, x.data_ptr(), ldx, M, K, codes.data_ptr(), scales.data_ptr())
        if rc != 0:
            _check(rc, "rq_i8_quantize")
    return codes, scales


def _check_codes(codes, scales, least):
    if (codes.dtype != torch.int8 or scales.dtype != torch.float32 or codes.dim() < least or codes.shape[:-1] != scales.shape
            or not codes.is_cuda or codes.get_device() != scales.get_device()):
        raise RqError("codes [.., K] are int8 and scales [..] fp32, on one GPU, got %s %s on %s and %s %s on %s"
                      % (codes.dtype, tuple(codes.shape), codes.device, scales.dtype, tuple(scales.shape), scales.device))


def i8_dequantize(codes, scales, dtype=torch.float32):
    """codes [.., K] and scales [..] -> codes times scales [.., K]: the fp32 products, rounded to dtype."""
    _check_codes(codes, scales, 1)
    dt = _dtype(dtype, "i8_dequantize")
    K = codes.shape[-1]
    out = codes.new_empty(codes.shape, dtype=dtype)
    if out.numel():
        codes, scales = codes.contiguous(), scales.contiguous()
        rc = _on_device_of(codes, load_library().rq_i8_dequantize, dt, codes.data_ptr(), scales.data_ptr(), out.numel() // K, K,
                           out.data_ptr(), K)
        if rc != 0:
            _check(rc, "rq_i8_dequantize")
    return out


class _Weight:
    """A weight [N, K], or E experts' [E, N, K], on the GPU in the form that the products stream."""

    def _prepare(self, kind, w, scales):
        if w.dim() not in (2, 3):
            raise RqError("%s: a weight [N, K] or experts' weights [E, N, K], got %s" % (type(self).__name__, tuple(w.shape)))
        self.kind = kind
        self.E = w.shape[0] if w.dim() == 3 else 1
        self.N, self.K = w.shape[-2:]
        self.device = w.device
        self._index = w.get_device()
        L = load_library()
        n = L.rq_weight_prepared_bytes(kind, self.E, self.N, self.K)
        if n == 0:
            raise RqError("%s: unsupported shape E=%d N=%d K=%d" % (type(self).__name__, self.E, self.N, self.K))
        w = w.contiguous()
        self.prepared = _device_bytes(n, self.device)
        _check(_on_device_of(w, L.rq_weight_prepare, kind, w.data_ptr(), None if scales is None else scales.data_ptr(), self.E, self.N,
                             self.K, self.prepared.data_ptr(), n), "rq_weight_prepare")
        self._ptr = self.prepared.data_ptr()

    def get_device(self):
        return self._index


class I8Weight(_Weight):
    """A weight in int8: codes [N, K] and scales [N] as i8_quantize gives them, or [E, N, K] and [E, N]. The tensors it is made from are
    not needed afterwards."""

    def __init__(self, codes, scales):
        _check_codes(codes, scales, 2)
        self._prepare(_I8, codes, scales.contiguous())

    def workspace(self, M):
        """of i8_mul_mat, for up to M rows"""
        if self.E != 1:
            raise RqError("I8Weight.workspace: of a weight [N, K], not of %d experts' (grouped_workspace_bytes(weight, M, P))" % self.E)
        return _device_bytes(load_library().rq_i8_workspace_bytes(self.K, self.N, M), self.device)


class HalfWeight(_Weight):
    """A weight in fp16 or bf16 for grouped_mul_mat: [E, N, K], or [N, K] as one expert's. The tensor it is made from is not needed
    afterwards."""

    def __init__(self, w):
        if w.dtype not in (torch.float16, torch.bfloat16) or not w.is_cuda:
            raise RqError("HalfWeight: a float16 or bfloat16 tensor on the GPU, got %s on %s" % (w.dtype, w.device))
        self.dtype = w.dtype
        self._prepare(_DTYPES[w.dtype], w, None)


def _described(weight):
    shape = [getattr(weight, name, "?") for name in ("E", "N", "K")]
    return "a %s of E=%s N=%s K=%s" % (type(weight).__name__, *shape)


def _given(x, scales, dtype, what):
    """(type of x, default type of the output) of activations that may be int8 already, checked"""
    if x.dtype != torch.int8:
        if scales is not None:
            raise RqError("%s: scales belong to int8 activations, got %s" % (what, x.dtype))
        return _dtype(x.dtype, what), x.dtype if dtype is None else dtype
    if scales is None or scales.dtype != torch.float32 or scales.shape != x.shape[:1] or not scales.is_contiguous():
        raise RqError("%s: int8 activations [%d, %d] come with fp32 scales [%d]" % (what, *x.shape, x.shape[0]))
    return _I8, torch.float32 if dtype is None else dtype


def i8_mul_mat(weight, x, scales=None, dtype=None, out=None, workspace=None):
    """y[M, N] = x^[M, K] . W^T with int8 products and exact sums. x in fp32, fp16 or bf16 is rounded as by i8_quantize; int8 x with its
    scales [M] is taken as it is. y = (sum * the weight's scale) * the token's scale in fp32, rounded to out's type, or to dtype
    (x's by default, fp32 for int8 x). `out` shares no memory with x."""
    M, K, ldx = _rows(x, "i8_mul_mat")
    if not isinstance(weight, I8Weight) or weight.E != 1 or K != weight.K:
        raise RqError("i8_mul_mat: activations of %d inputs against %s, not an I8Weight [N, %d]" % (K, _described(weight), K))
    N = weight.N
    dt, dtype = _given(x, scales, dtype, "i8_mul_mat")
    ldy = N
    if out is None:
        odt = _dtype(dtype, "i8_mul_mat")
        out = x.new_empty((M, N), dtype=dtype)
    else:
        ldy, odt = _output(out, M, N, "i8_mul_mat")
    if M == 0:
        return out
    L = load_library()
    index = x.get_device()
    if workspace is None:
        n, at = L.rq_i8_workspace_bytes(K, N, M), None
        if n > 256:   # (256: nothing that the call looks at)
            workspace = x.new_empty((n,), dtype=torch.uint8)
            at = workspace.data_ptr()
    else:
        n, at = _workspace_bytes(workspace), workspace.data_ptr()
    _elsewhere(index, weight=weight, scales=scales, out=out, workspace=workspace)
    rc = _on_device_of(x, L.rq_i8_mul_mat, weight._ptr, K, N, dt, x.data_ptr(), ldx, None if scales is None else scales.data_ptr(), M,
                       odt, out.data_ptr(), ldy, at, n)
    if rc != 0:
        _check(rc, "rq_i8_mul_mat")
    return out


def sort_slots(ids, E, workspace=None):
    """ids[M, top] int32 as route gives them -> offsets [E + 1], slots [M * top], tokens [M * top], int32. Slot m * top + j is the j-th
    choice of token m. `slots` has them in the order of their experts, those of one expert in rising order, and tokens = slots // top;
    expert e's are at offsets[e] .. offsets[e + 1] - 1. Slots with an id outside 0 .. E - 1 stand behind offsets[E]."""
    if ids.dtype != torch.int32 or ids.dim() != 2 or not ids.is_contiguous() or not ids.is_cuda:
        raise RqError("sort_slots: ids int32 [M, top] on the GPU, contiguous, got %s %s on %s" % (ids.dtype, tuple(ids.shape), ids.device))
    M, top = ids.shape
    L = load_library()
    if not 1 <= E <= 1024:
        raise RqError("sort_slots: 1 to 1024 experts, got %d" % E)
    offsets, slots, tokens = ids.new_empty((E + 1 + 2 * M * top,)).split((E + 1, M * top, M * top))   # (one allocation: a small call is the host's time)
    n = L.rq_sort_workspace_bytes(M, top, E)
    at = None
    if workspace is None:
        if n:
            workspace = ids.new_empty((n,), dtype=torch.uint8)
            at = workspace.data_ptr()
    else:
        n, at = _workspace_bytes(workspace), workspace.data_ptr()
        _elsewhere(ids.get_device(), workspace=workspace)
    rc = _on_device_of(ids, L.rq_sort_slots, ids.data_ptr(), M, top, E, offsets.data_ptr(), slots.data_ptr(), tokens.data_ptr(), at, n)
    if rc != 0:
        _check(rc, "rq_sort_slots")
    return offsets, slots, tokens


def _places(t, P, what):
    if t is not None and (t.dtype != torch.int32 or t.shape != (P,) or not t.is_contiguous()):
        raise RqError("grouped_mul_mat: %s int32 [%d], contiguous, got %s %s" % (what, P, t.dtype, tuple(t.shape)))


def grouped_mul_mat(weight, x, offsets, rows=None, out_rows=None, scales=None, dtype=None, out=None, workspace=None):
    """Products of ragged groups of rows with their experts' weights (I8Weight or HalfWeight [E, N, K]). Of P positions, those from offsets[e] up to
    offsets[e + 1] (int32 [E + 1], not falling) belong to expert e:

        y[out_rows[p]] = W_e x[rows[p]]

    where p itself stands for rows[p] or out_rows[p] if that is None. rows (int32 [P]) lets positions read tokens where they lie, out_rows
    (int32 [P], no row twice) write to the slots' places; without rows P is the number of x's rows. An index of rows outside x gives zeros, one
    of out_rows outside `out` is not written. Rows of `out` that no position writes are left as they were (so undefined where the call makes
    `out`, [P, N]): among them, without out_rows, those from offsets[E] on, and with sort_slots' slots for out_rows those of experts that are not
    here; an `out` of zeros keeps them out of later sums.

    With int8 weights x in fp32, fp16 or bf16 is rounded as by i8_quantize, int8 x with its scales is taken as it is, and products are scaled as by
    i8_mul_mat; with 16-bit weights x has the weight's type. Sums are exact or in fp32; y is rounded to out's type, or to dtype (x's by default, fp32 for
    int8 x). `out` shares no memory with the inputs."""
    M, K, ldx = _rows(x, "grouped_mul_mat")
    if not isinstance(weight, _Weight) or K != weight.K:
        raise RqError("grouped_mul_mat: x of %d inputs against %s, not an I8Weight or HalfWeight [E, N, %d]" % (K, _described(weight), K))
    E, N = weight.E, weight.N
    if weight.kind != _I8 and x.dtype != weight.dtype:
        raise RqError("grouped_mul_mat: x has to be of the weight's type %s, got %s" % (weight.dtype, x.dtype))
    if offsets.dtype != torch.int32 or offsets.shape != (E + 1,) or not offsets.is_contiguous():
        raise RqError("grouped_mul_mat: offsets int32 [%d], contiguous, got %s %s" % (E + 1, offsets.dtype, tuple(offsets.shape)))
    P = M if rows is None else rows.numel()
    _places(rows, P, "rows")
    _places(out_rows, P, "out_rows")
    dt, dtype = _given(x, scales, dtype, "grouped_mul_mat")
    ldy, Y = N, P
    if out is None:
        odt = _dtype(dtype, "grouped_mul_mat")
        out = x.new_empty((P, N), dtype=dtype)
    else:
        if out.dim() == 2 and out_rows is not None:
            Y = out.shape[0]
        ldy, odt = _output(out, Y, N, "grouped_mul_mat")
    if P == 0 or Y == 0:
        return out
    L = load_library()
    index = x.get_device()
    if workspace is None:
        n, at = L.rq_grouped_workspace_bytes(weight.kind, E, K, N, M, P), None
        if n > 256:
            workspace = x.new_empty((n,), dtype=torch.uint8)
            at = workspace.data_ptr()
    else:
        n, at = _workspace_bytes(workspace), workspace.data_ptr()
    _elsewhere(index, weight=weight, offsets=offsets, rows=rows, out_rows=out_rows, scales=scales, out=out, workspace=workspace)
    pointer = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    rc = _on_device_of(x, L.rq_grouped_mul_mat, weight.kind, weight._ptr, E, K, N, dt, x.data_ptr(), ldx, pointer(scales), M,
                       offsets.data_ptr(), P, pointer(rows), pointer(out_rows), odt, out.data_ptr(), ldy, Y, at, n)
    if rc != 0:
        _check(rc, "rq_grouped_mul_mat")
    return out


def grouped_workspace_bytes(weight, M, P):
    """Workspace of grouped_mul_mat for x of M rows and P positions; it grows with both."""
    return load_library().rq_grouped_workspace_bytes(weight.kind, weight.E, weight.K, weight.N, M, P)
