"""What the plans of the int8 and grouped products say at the ends of their rules, asked without a GPU."""
import pytest

import ruquant_amd as rq
from tests import i8_plan_util as plan
from tests.i8_plan_util import BF16, F16, F32, I8, ROUNDS, STREAM

# Of a workgroup that rounds rows: 2 x 8 maxima and 16 scales, 4 bytes each, beside the rows, which have 16 bytes behind their steps of 64.
FIXED, LDS = 128, 65536


def _lengths():
    """rows around every length at which one row less fits, and the longest"""
    for rows in range(1, 9):
        last = LDS // rows - 16
        yield from range(last // 64 * 64 - 130, last // 64 * 64 + 66)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_rounded_rows_fit_the_memory_that_a_launch_has_without_asking(dtype):
    reached = set()
    for K in _lengths():
        plans = [plan.product(K, 32, M, dtype) for M in (1, 2)] + [plan.grouped(I8, 8, K, 32, P, P, dtype) for P in range(1, 9)]
        for p in plans:
            assert p[0] in (ROUNDS, STREAM)
            if p[0] == ROUNDS:
                reached.add(p[1])
                assert FIXED + p[1] * ((K + 63) // 64 * 64 + 16) <= LDS, (K, p[1])
    assert reached == set(range(1, 9))


def test_calls_on_both_sides_of_the_longest_rounded_row():
    """a call that needs no workspace says so, and the one that is one element longer asks for its rounded row"""
    L = rq.load_library()
    last = max(K for K in _lengths() if plan.product(K, 32, 1, F32)[0] == ROUNDS)
    assert plan.product(last + 1, 32, 1, F32)[0] == STREAM
    assert L.rq_i8_workspace_bytes(last, 32, 1) == 256 and L.rq_i8_workspace_bytes(last + 1, 32, 1) > last
    assert L.rq_grouped_workspace_bytes(I8, 8, last, 32, 1, 1) == 256 and L.rq_grouped_workspace_bytes(I8, 8, last + 1, 32, 1, 1) > last


def test_a_dense_workspace_is_of_a_dense_weight():
    """experts' weights have no product of their own: what their workspace takes depends on the positions too"""
    W = object.__new__(rq.I8Weight)
    W.E, W.N, W.K, W.device = 8, 1000, 5000, "cpu"
    with pytest.raises(rq.RqError, match="grouped_workspace_bytes"):
        W.workspace(40)
