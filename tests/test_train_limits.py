"""What training calls decide on the host, without a GPU: rows of no segment, and which sizes are too many for a launch."""
import itertools

import pytest

from dan_amd import workloads
from dan_amd.attention import Batch, _uncovered, segment


@pytest.mark.parametrize("spans", [[], [(0, 9)], [(2, 9)], [(0, 4), (4, 9)], [(6, 9), (1, 3)], [(0, 3), (5, 6), (8, 11)], [(3, 3), (4, 9)], [(2, 7), (3, 5)]])
def test_rows_of_no_segment(spans):
    n = 11
    for order in itertools.permutations(spans):
        segs = Batch(segment(a, workloads.branch_ids(b - a, []), None, 0, 0, "cpu") for a, b in order)
        runs = _uncovered(segs, n)
        assert all(a < b for a, b in runs)
        rows = [r for a, b in runs for r in range(a, b)]
        assert rows == [r for r in range(n) if not any(a <= r < b for a, b in spans)]
