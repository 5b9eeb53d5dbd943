"""int8 rows, their products, the sort of slots and the products grouped by expert from their definitions, in 64 bits on the host."""
import numpy as np


def quantize(x):
    """x [M, K] float64 (values of a float type) -> codes int8 [M, K], scales fp32 [M]"""
    finite = np.isfinite(x).all(axis=1)
    v = np.where(finite[:, None], x, 0.0)
    scales = np.maximum(np.abs(v).max(axis=1).astype(np.float32) * np.float32(1 / 127), np.float32(2.0 ** -126))
    r = (1.0 / scales.astype(np.float64)).astype(np.float32)
    codes = np.rint(v * r.astype(np.float64)[:, None]).astype(np.int8)   # (the product of two 24-bit numbers is exact)
    return codes, np.where(finite, scales, np.float32(np.nan))


def scaled(a, w, s, t):
    """the fp32 numbers ((sum of a w) t) s: a [M, K], w [N, K] int8, s [M], t [N]"""
    total = a.astype(np.float64) @ w.astype(np.float64).T   # (whole numbers below 2^31: exact)
    with np.errstate(invalid="ignore"):
        return total.astype(np.float32) * t[None, :] * s[:, None]


def sort(ids, E):
    flat = ids.reshape(-1).astype(np.int64)
    expert = np.where((flat >= 0) & (flat < E), flat, E)
    slots = np.argsort(expert, kind="stable")
    offsets = np.searchsorted(expert[slots], np.arange(E + 1))
    return offsets.astype(np.int32), slots.astype(np.int32), (slots // max(1, ids.shape[1])).astype(np.int32)
