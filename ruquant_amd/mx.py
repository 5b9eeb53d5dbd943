"""MXFP4 weights and activations, the routing to experts and the experts' feed-forward, over the C ABI of include/rq_mx4.h.

MXFP4 (microscaled 4-bit floating point): 32 consecutive elements of a row share a scale. Elements are e2m1 (0, 0.5, 1, 1.5, 2, 3,
4, 6 and their negatives), two per byte, the even one in the low half; a scale is a byte X that stands for 2 ** (X - 127), 255 for
NaN. A tensor [.., K] is codes [.., K / 2] and scales [.., K / 32], both uint8.

As in the rest of the package torch owns device memory and the stream, and every computation happens inside librq_w4a4.so, on the
current stream of the inputs' device. With `out` and `workspace` given the product and the experts allocate nothing; the other calls
make their outputs. All of them can be captured in a graph.
"""
import torch

from .lib import load_library
from .w4a4 import RqError, _check, _device_bytes, _on_device_of

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
SCORINGS = {"softmax": 0, "sigmoid": 1}


def _dtype(t, what):
    code = _DTYPES.get(t)
    if code is None:
        raise RqError("%s: float32, float16 or bfloat16, got %s" % (what, t))
    return code


def _rows(x, what):
    """(rows, length, row stride) of a matrix on the GPU whose rows' elements are consecutive"""
    # (a decode step's calls are a few microseconds each on the GPU: every attribute that is asked for shows)
    if x.dim() == 2 and x.is_cuda:
        M, K = x.shape
        ld, one = x.stride()
        if one == 1 or K == 1:
            return M, K, ld if M > 1 else K
    raise RqError("%s: a matrix on the GPU with consecutive elements in its rows, got %s on %s with strides %s"
                  % (what, tuple(x.shape), x.device, x.stride()))


def _elsewhere(index, **others):
    """The error for a tensor or weight that is not on GPU `index`"""
    for name, t in others.items():
        if t is not None and t.get_device() != index:
            raise RqError("%s is on GPU %d, the activations are on %d" % (name, t.get_device(), index))


def _check_codes(codes, scales):
    shape, blocks = codes.shape, scales.shape
    if (codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or len(shape) < 2 or shape[:-1] != blocks[:-1]
            or shape[-1] != 16 * blocks[-1] or not codes.is_cuda or codes.get_device() != scales.get_device()):
        raise RqError("codes [.., K / 2] and scales [.., K / 32] are uint8 tensors on one GPU, got %s %s on %s and %s %s on %s"
                      % (codes.dtype, tuple(codes.shape), codes.device, scales.dtype, tuple(scales.shape), scales.device))


def _aligned(t, n):
    t = t.contiguous()
    return t if t.data_ptr() % n == 0 else t.clone()


def mx_quantize(x):
    """x[M, K] (fp32, fp16 or bf16) -> codes [M, K / 2], scales [M, K / 32]. The scale is the exponent of the block's largest
    magnitude less two; elements go to the nearest, ties to the even code, and saturate at 6 units. A block that holds an infinity
    or a NaN becomes NaN."""
    M, K, ldx = _rows(x, "mx_quantize")
    dt = _dtype(x.dtype, "mx_quantize")
    if K % 32 or K == 0:
        raise RqError("mx_quantize: rows of whole blocks of 32, got %d" % K)
    codes = x.new_empty((M, K // 2), dtype=torch.uint8)
    scales = x.new_empty((M, K // 32), dtype=torch.uint8)
    if M:
        rc = _on_device_of(x, load_library().rq_mx4_quantize, dt, x.data_ptr(), ldx, M, K, codes.data_ptr(), scales.data_ptr())
        if rc != 0:
            _check(rc, "rq_mx4_quantize")
    return codes, scales


def mx_dequantize(codes, scales, dtype=torch.float32):
    """codes [.., K / 2] and scales [.., K / 32] -> values [.., K], rounded once to dtype."""
    _check_codes(codes, scales)
    dt = _dtype(dtype, "mx_dequantize")
    K = 2 * codes.shape[-1]
    out = codes.new_empty((*codes.shape[:-1], K), dtype=dtype)
    if out.numel():
        codes, scales = _aligned(codes, 4), scales.contiguous()
        rc = _on_device_of(codes, load_library().rq_mx4_dequantize, dt, codes.data_ptr(), scales.data_ptr(), out.numel() // K, K,
                           out.data_ptr(), K)
        if rc != 0:
            _check(rc, "rq_mx4_dequantize")
    return out


class MXWeight:
    """A weight [N, K], or E experts' weights [E, N, K], in MXFP4 on the GPU: its codes and scales in the form that the products
    stream. The tensors it is made from are not needed afterwards."""

    def __init__(self, codes, scales):
        _check_codes(codes, scales)
        if codes.dim() not in (2, 3):
            raise RqError("MXWeight: a weight [N, K] or experts' weights [E, N, K], got codes %s" % (tuple(codes.shape),))
        self.E = codes.shape[0] if codes.dim() == 3 else 1
        self.N, self.K = codes.shape[-2], 2 * codes.shape[-1]
        self.device = codes.device
        self._index = codes.get_device()
        L = load_library()
        n = L.rq_mx4_prepared_bytes(self.E, self.N, self.K)
        if n == 0:
            raise RqError("MXWeight: unsupported shape E=%d N=%d K=%d" % (self.E, self.N, self.K))
        codes, scales = _aligned(codes, 256), _aligned(scales, 256)
        self.prepared = _device_bytes(n, self.device)
        _check(_on_device_of(codes, L.rq_mx4_prepare, codes.data_ptr(), scales.data_ptr(), self.E, self.N, self.K,
                             self.prepared.data_ptr(), n), "rq_mx4_prepare")
        self._ptr = self.prepared.data_ptr()

    def get_device(self):
        return self._index

    def workspace(self, M):
        return _device_bytes(load_library().rq_mx4_workspace_bytes(self.K, self.N, M), self.device)


def _output(out, M, N, what):
    """row stride and type of `out`, checked"""
    if out.shape == (M, N) and out.is_cuda:
        ld, one = out.stride()
        if (one == 1 or N == 1) and (M == 1 or ld >= N):
            return ld if M > 1 else N, _dtype(out.dtype, what)
    raise RqError("%s: out has to be [%d, %d] on the GPU with consecutive elements in its rows, got %s with strides %s"
                  % (what, M, N, tuple(out.shape), out.stride()))


def _workspace_bytes(workspace):
    if not workspace.is_contiguous():
        raise RqError("a workspace is one run of memory, got strides %s" % (workspace.stride(),))
    return workspace.numel() * workspace.element_size()


def mx_mul_mat(weight, x, out=None, workspace=None):
    """y[M, N] = x^[M, K] . W^T, x^ = x rounded as by mx_quantize, sums in fp32, rounded once to out's type (x's by default).
    `out` shares no memory with x."""
    M, K, ldx = _rows(x, "mx_mul_mat")
    N = weight.N
    if weight.E != 1 or K != weight.K:
        raise RqError("mx_mul_mat: activations of %d inputs against a weight of E=%d N=%d K=%d" % (K, weight.E, N, weight.K))
    odt = dt = _dtype(x.dtype, "mx_mul_mat")
    ldy = N
    if out is None:
        out = x.new_empty((M, N))
    else:
        ldy, odt = _output(out, M, N, "mx_mul_mat")
    if M == 0:
        return out
    L = load_library()
    index = x.get_device()
    if workspace is None:
        n, at = L.rq_mx4_workspace_bytes(K, N, M), None
        if n > 256:   # (256: nothing that the call looks at)
            workspace = x.new_empty((n,), dtype=torch.uint8)
            at = workspace.data_ptr()
    else:
        n, at = _workspace_bytes(workspace), workspace.data_ptr()
        _elsewhere(index, workspace=workspace)
    if weight._index != index or out.get_device() != index:
        _elsewhere(index, weight=weight, out=out)
    rc = _on_device_of(x, L.rq_mx4_mul_mat, weight._ptr, K, N, dt, x.data_ptr(), ldx, M, odt, out.data_ptr(), ldy, at, n)
    if rc != 0:
        _check(rc, "rq_mx4_mul_mat")
    return out


def route(logits, top, scoring="softmax", bias=None, groups=1, top_groups=1, renormalize=True, scale=1.0):
    """Each row of logits[M, E] chooses `top` experts -> ids [M, top] int32 in falling order of choice, weights [M, top] fp32.

    The scores are softmax(logits) or sigmoid(logits). The choice goes by score + bias (bias[E] fp32, as balances the experts' load);
    with groups > 1 only the experts of the top_groups runs of E / groups whose two best add up to most can be chosen. Ties go to the
    lowest index. The weights are the chosen scores without the bias, divided by their sum if renormalize, times scale."""
    M, E, ldl = _rows(logits, "route")
    dt = _dtype(logits.dtype, "route")
    if scoring not in SCORINGS:
        raise RqError("route: scoring %r is none of %s" % (scoring, sorted(SCORINGS)))
    if groups < 1 or E % groups or not 1 <= top_groups <= groups or not 1 <= top <= top_groups * (E // groups):
        raise RqError("route: %d of %d experts from %d of %d groups" % (top, E, top_groups, groups))
    if bias is not None:
        if bias.dtype != torch.float32 or bias.shape != (E,) or not bias.is_contiguous():
            raise RqError("route: bias is fp32 [%d], got %s %s" % (E, bias.dtype, tuple(bias.shape)))
        _elsewhere(logits.get_device(), bias=bias)
    ids = logits.new_empty((M, top), dtype=torch.int32)
    weights = logits.new_empty((M, top), dtype=torch.float32)
    if M:
        rc = _on_device_of(logits, load_library().rq_route, dt, logits.data_ptr(), ldl, M, E, SCORINGS[scoring],
                           None if bias is None else bias.data_ptr(), groups, top_groups, top, int(renormalize), float(scale),
                           ids.data_ptr(), weights.data_ptr())
        if rc != 0:
            _check(rc, "rq_route")
    return ids, weights


def expert_workspace_bytes(gate, down, M, top):
    """Workspace of expert_ffn for M tokens with `top` experts each."""
    return load_library().rq_mx4_experts_workspace_bytes(gate.E, gate.K, gate.N, down.N, M, top)


def expert_ffn(gate, up, down, x, ids, weights, out=None, workspace=None):
    """y[m] = sum_j weights[m, j] * down_e(silu(gate_e(x[m])) * up_e(x[m])), e = ids[m, j], with MXFP4 products: x and the hidden
    values are rounded as by mx_quantize, sums are fp32, y is rounded once to out's type (x's by default).

    gate, up: MXWeight [E, F, K]; down: MXWeight [E, N, F]; ids [M, top] int32 and weights [M, top] fp32 as route gives them. An id
    outside 0 .. E - 1 adds nothing (an expert that another device holds, a token that is padding). `out` shares no memory with the inputs."""
    M, K, ldx = _rows(x, "expert_ffn")
    E, F, N = gate.E, gate.N, down.N
    if (up.E, up.N, up.K, down.E, down.K, gate.K) != (E, F, K, E, F, K):
        raise RqError("expert_ffn: x of %d inputs, gate E=%d N=%d K=%d, up E=%d N=%d K=%d, down E=%d N=%d K=%d do not fit"
                      % (K, E, F, gate.K, up.E, up.N, up.K, down.E, N, down.K))
    if (ids.dtype != torch.int32 or weights.dtype != torch.float32 or ids.dim() != 2 or ids.shape[0] != M or weights.shape != ids.shape
            or not ids.is_contiguous() or not weights.is_contiguous()):
        raise RqError("expert_ffn: ids int32 and weights fp32 [%d, top], contiguous, got %s %s and %s %s"
                      % (M, ids.dtype, tuple(ids.shape), weights.dtype, tuple(weights.shape)))
    odt = dt = _dtype(x.dtype, "expert_ffn")
    ldy = N
    if out is None:
        out = x.new_empty((M, N))
    else:
        ldy, odt = _output(out, M, N, "expert_ffn")
    if M == 0:
        return out
    L = load_library()
    index, top = x.get_device(), ids.shape[1]
    if workspace is None:
        n = L.rq_mx4_experts_workspace_bytes(E, K, F, N, M, top)
        workspace = x.new_empty((n,), dtype=torch.uint8)
    else:
        n = _workspace_bytes(workspace)
    _elsewhere(index, gate=gate, up=up, down=down, ids=ids, weights=weights, out=out, workspace=workspace)
    rc = _on_device_of(x, L.rq_mx4_experts, gate._ptr, up._ptr, down._ptr, E, K, F, N, dt, x.data_ptr(), ldx, M, ids.data_ptr(),
                       weights.data_ptr(), top, odt, out.data_ptr(), ldy, workspace.data_ptr(), n)
    if rc != 0:
        _check(rc, "rq_mx4_experts")
    return out
