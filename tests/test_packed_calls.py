"""Calls over a cache in 4 bits that its other tests do not make: plans whose rows lie anywhere, calls without what they need, rows and heads of noughts, numbers
at both ends of their range, groups that are no numbers in portions, rows over chosen pages beside others, and the room that a portion takes."""
import math

import pytest
import torch

from test_packed import BF16, F32, GPU, chosen, make_pool, make_table, near, places, plain_attention, poison, tiles_bytes

from beglin_b200.csrc import ops


# ------------------------------------------------------------------------------------------------ plans
@pytest.mark.parametrize("lens,row_start", [([1, 1], [0, 100]), ([1, 1], [0, -1]), ([1, 1], [0, 0]), ([2, 2], [0, 1]), ([1, 1], [1, 2]), ([3], [1]), ([70, 1], [2, 0]),
                                            ([0, 1], [0, 1]), ([1] * 70, list(range(1, 71)))], ids=str)
def test_a_plan_refuses_rows_that_the_step_does_not_have(lens, row_start):
    """Every row of the step is one request's: none lies outside, none is in two requests."""
    with pytest.raises(ops.KernelError, match="first row"):
        ops.packed_plan(lens, 4, 2, 64, BF16, 64, device="cpu", row_start=row_start)


def test_a_plan_takes_rows_in_any_order():
    plan = ops.packed_plan([1, 0, 2, 1], 4, 2, 64, BF16, 64, device="cpu", row_start=[3, -7, 0, 2])
    assert plan.short.view(-1, 3).tolist() == [[0, 3, 1], [2, 0, 2], [3, 2, 1]]


# ------------------------------------------------------------------------------------------------ calls without what they need
def test_rows_need_their_requests(monkeypatch):
    """Only attention knows whose a row is without a list of requests."""
    monkeypatch.setattr(ops, "_here", lambda *a: None)                         # (nothing is launched)
    hd, page, T = 64, 16, 3
    pool, table, positions = make_pool(2, 1, hd, page, True), torch.zeros((T, 1), dtype=torch.int32), torch.zeros(T, dtype=torch.int32)
    src, q = torch.zeros((T, 3 * hd), dtype=BF16), torch.zeros((T, hd), dtype=BF16)
    for call in (lambda: ops.packed_append(src, q, 1, 1, hd, 0, False, None, positions, None, table, pool, page, None),
                 lambda: ops.packed_bounds(pool, positions, None, table, hd, page, None),
                 lambda: ops.packed_rows(pool, positions, None, table, hd, page, torch.empty((T, 2, 1, hd)), None)):
        with pytest.raises(ops.KernelError, match="a request for every row"):
            call()
