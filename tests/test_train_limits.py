"""What training calls decide on the host, without a GPU: rows of no segment, and what a capture may begin with."""
import itertools

import pytest

import torch

from dan_amd import _grad, _native, workloads
from dan_amd.attention import Batch, _uncovered, segment
from dan_amd.plan import TilePlan


@pytest.mark.parametrize("spans", [[], [(0, 9)], [(2, 9)], [(0, 4), (4, 9)], [(6, 9), (1, 3)], [(0, 3), (5, 6), (8, 11)], [(3, 3), (4, 9)], [(2, 7), (3, 5)]])
def test_rows_of_no_segment(spans):
    n = 11
    for order in itertools.permutations(spans):
        segs = Batch(segment(a, workloads.branch_ids(b - a, []), None, 0, 0, "cpu") for a, b in order)
        runs = _uncovered(segs, n)
        assert all(a < b for a, b in runs)
        rows = [r for a, b in runs for r in range(a, b)]
        assert rows == [r for r in range(n) if not any(a <= r < b for a, b in spans)]


def test_what_a_capture_may_begin_with():
    """Nothing that the capture itself would have to upload or copy."""
    def make(count, entry):
        segs, at = Batch(), 0
        for _ in range(count):
            segs.append(segment(at, workloads.branch_ids(4, []), {0: entry, 1: entry}, 0, 3, "cpu"))
            at += 4
        return TilePlan.build(segs, at, 64, "cpu")

    layout, aligned = (4, 2, 64), tuple(torch.zeros(2, 3, 64, dtype=torch.bfloat16) for _ in range(2))
    assert not _grad.capturable(None, 0, layout)
    plan = make(3, aligned)
    assert not _grad.capturable(plan, 0, layout)  # the backward pass's tables are missing
    plan.grad_tables[layout] = None
    assert _grad.capturable(plan, 0, layout) and not _grad.capturable(plan, 0, (8, 2, 64))
    odd = torch.zeros(2, 3, 65, dtype=torch.bfloat16)[..., 1:]
    copied = make(1, (aligned[0], odd))
    long = make(_native.INLINE_PASTS + 1, aligned)
    for plan in (copied, long):
        plan.grad_tables[layout] = None
        assert not _grad.capturable(plan, 0, layout)
        plan.past_tables[0], plan.past_hosts[0] = None, None if plan is long else 0
        if plan is long:
            assert not _grad.capturable(plan, 0, layout)
            plan.past_uploaded.add(0)
        assert _grad.capturable(plan, 0, layout) and not _grad.capturable(plan, 1, layout)
