"""The plans of the int8 product and of the products grouped by expert, as the library tells them."""
import ctypes

import ruquant_amd as rq

F32, F16, BF16, I8 = 0, 1, 2, 3
ROUNDS, STREAM, TILES = 1, 2, 3


def product(K, N, M, dtype=I8):
    p = (ctypes.c_int64 * 8)()
    assert rq.load_library().rq_i8_product_plan(K, N, dtype, M, p) == 0
    return list(p)


def grouped(kind, E, K, N, M, P, dtype=None):
    p = (ctypes.c_int64 * 8)()
    assert rq.load_library().rq_grouped_plan(kind, E, K, N, kind if dtype is None else dtype, M, P, p) == 0
    return list(p)
