"""attend_train in fp16 beside a segment that overflowed: its infinities change nothing of another segment's gradients, which share
the batch's power of 2 (dan_amd/csrc/tree_attn_grad.hip, ds_factor)."""
import math

import pytest
import torch

import test_gpu_attend_train
from oracle import training as oracle

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def say(*a):
    print("[gpu-case]", *a, flush=True)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("which", ["v", "grad", "prefix"])
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(4, 2, 64), (4, 1, 128), (2, 1, 256)])
def test_a_segments_infinity_stays_in_it(gpu, heads, kv_heads, head_dim, which, bad, dtype):
    """Bit for bit what the others get where that row is zeros; and with gradients of 2^-12, which fp16 would not hold dS of as it
    is, as close to the oracle as ever (test_gpu_train_edges' tolerance for such gradients)."""
    say("attend_train: infinite", which, bad, heads, kv_heads, head_dim, dtype)
    q, k, v, grad, segs = test_gpu_attend_train.make(gpu, [(70, [5, 40]), (33, [30]), (64, [2])], heads, kv_heads, head_dim, dtype, pasts=[12, 20, 0])
    grad = (grad.float() * 2.0 ** -12).to(dtype)
    s = segs[1]
    at = {"v": v[:, s.start + 3], "grad": grad[:, s.start + 3], "prefix": s.past[0][1][:, 7]}[which]
    at.zero_()
    want = test_gpu_attend_train.train(q, k, v, grad, segs)
    at[..., 5] = bad
    got = test_gpu_attend_train.train(q, k, v, grad, segs)
    assert not got[1][:, s.start:s.end].isfinite().all()
    u = torch.finfo(dtype).eps / 2
    ref = oracle.attend(q, k, v, [segs[0], segs[2]], 0, grad=grad)
    for name, a, b in zip(("out", "dq", "dk", "dv"), got, want, strict=True):
        for t in (segs[0], segs[2]):
            rows = slice(t.start, t.end)
            assert torch.equal(a[:, rows], b[:, rows]), name
            x, r, bound = a[:, rows].double().cpu(), ref[name][:, rows], ref["abs_" + name][:, rows]
            assert ((x - r).abs() <= 6 * u * bound + 2 ** -12 * bound + (2 ** -24 if dtype is FP16 else torch.finfo(dtype).tiny)).all(), name
