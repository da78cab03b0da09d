"""What training calls decide on the host, without a GPU: rows of no segment, what a capture may begin with, and
which sizes a launch holds."""
import ctypes
import itertools

import pytest

import torch

from dan_amd import _grad, _layer, _native, workloads
from dan_amd.attention import Batch, _uncovered, segment
from dan_amd.plan import TilePlan
from test_abi import lib  # noqa: F401  -- the library fixture


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
    assert not _grad.capturable(plan, 0, layout)  # a prefix table in the capture's own memory
    plan.make_spare(3 * 72)
    assert set(plan.spare) == {0, 1} and all(t.shape == (3 * 72,) for t in plan.spare.values())
    assert _grad.capturable(plan, 0, layout) and not _grad.capturable(plan, 0, (8, 2, 64))
    odd = torch.zeros(2, 3, 65, dtype=torch.bfloat16)[..., 1:]
    copied = make(1, (aligned[0], odd))
    long = make(_native.INLINE_PASTS + 1, aligned)
    for plan in (copied, long):
        plan.grad_tables[layout] = None
        plan.make_spare(72 * len(plan.past_dicts))
        assert not _grad.capturable(plan, 0, layout)
        plan.past_tables[0], plan.past_hosts[0] = None, None if plan is long else 0
        if plan is long:
            assert not _grad.capturable(plan, 0, layout)
            plan.past_uploaded.add(0)
        assert _grad.capturable(plan, 0, layout) and not _grad.capturable(plan, 1, layout)


P = 4096  # an aligned address that no call reads


def adapt_args(cls, rows, n_in, n_out, rank, adapters):
    a = cls()
    a.abi_version, a.dtype, a.scale_value = _layer.ADAPT_ABI_VERSION, _native.DTYPE_BF16, 1.0
    a.rows, a.n_in, a.n_out, a.rank, a.adapters = rows, n_in, n_out, rank, adapters
    return a  # (x is missing: sizes that are taken end there)


@pytest.mark.parametrize("rows,n_in,n_out,rank,adapters,forward,gradient", [
    # up to what a launch of the kernels for many rows holds, a thread for 128 values
    (1 << 20, 8, 8192, 16, 1, True, True), (1 << 19, 4096, 28672, 64, 8, True, True), (131072, 64, 65536, 16, 3, True, True),
    (1 << 20, 1 << 18, 8, 8, 1, True, True), (1 << 20, 8, (1 << 19) - 1024, 1, 1, True, True), (1 << 20, 8, 1 << 19, 1, 1, False, False),
    (1 << 20, 1 << 20, 32, 8, 1, False, False), (1 << 19, 8, (1 << 20) - 1024, 1, 1, True, True), (1 << 19, 8, 1 << 20, 1, 1, False, False),
    # few rows: a thread for 2 values, always held
    (640, 1 << 20, 1 << 20, 16, 1, True, True), (768, 1 << 20, 1 << 20, 16, 5, True, True),
    # many adapters are the gradient's limit
    (64, 8192, 28672, 1, 65535, True, False), (64, 8192, 4096, 1, 65535, True, True), (64, 8192, 8192, 128, 16383, True, True), (64, 8192, 8192, 128, 16400, True, False)])
def test_adapts_sizes(lib, rows, n_in, n_out, rank, adapters, forward, gradient):  # noqa: F811
    for name, cls, taken in (("dan_adapt", _layer.DanAdaptArgs, forward), ("dan_adapt_grad", _layer.DanAdaptGradArgs, gradient)):
        a = adapt_args(cls, rows, n_in, n_out, rank, adapters)
        assert lib[name](ctypes.byref(a), None) == (_native.ERR_INVALID_ARGUMENT if taken else _native.ERR_UNSUPPORTED)
        assert ("NULL" if taken else "one launch") in _native.last_error(lib)
    assert (_layer.adapt_grad_workspace_size(rows, n_in, n_out, rank, adapters) > 0) == gradient


@pytest.mark.parametrize("rows,cols,layout,taken", [
    ((1 << 24) - 1, 4096, 0, True), ((1 << 24) - 256, 4096, 1, True), ((1 << 24) - 255, 4096, 1, False), ((1 << 24) - 1, 1040, 1, False), ((1 << 24) - 1, 1024, 1, True)])
def test_add_norms_rows(lib, rows, cols, layout, taken):  # noqa: F811
    """With tiled codes whole panels of 256 rows are launched, a work group each row (four up to 1024 columns): 2^24 of them are more than a
    launch holds. (What is taken ends at its weight's alignment.)"""
    a = _layer.DanNormArgs()
    a.abi_version, a.dtype, a.rows, a.cols, a.eps, a.layout = _layer.NORM_ABI_VERSION, _native.DTYPE_BF16, rows, cols, 1e-6, layout
    a.x = a.codes = a.scale = P
    a.weight, a.x_stride = P + 2, cols
    assert lib.dan_add_norm(ctypes.byref(a), None) == _native.ERR_INVALID_ARGUMENT
    assert ("aligned" if taken else "2^24 - 256") in _native.last_error(lib)
