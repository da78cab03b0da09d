"""attend_train over batches that change or that training and other calls share: rows of no segment where nothing needs a
gradient.

Results are compared bit for bit with those of the same kernels on the same values."""
import math

import pytest
import torch
import torch.utils.checkpoint

import test_gpu_attend_train
from dan_amd.attention import Batch, attend_train, segment
from test_gpu_train_calls import same, say

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def poison(like, value=math.nan):
    """Fills memory of `like`'s size, many times over, and gives it back to the allocator: an empty tensor of that size holds `value`."""
    blocks = [torch.full((like.numel(),), value, dtype=like.dtype, device=like.device) for _ in range(32)]
    torch.cuda.synchronize()
    del blocks


# ---------------------------------------------------------------- rows of no segment
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("structure,gap", [([(40, [5, 9]), (7, [30]), (1, [])], 5), ([(64, [3])], 1), ([(300, [40, 3])], 200)])
@pytest.mark.parametrize("how", ["no_grad", "frozen", "inference"])
def test_rows_of_no_segment_give_zeros_without_a_gradient(gpu, how, structure, gap, dtype):
    say("attend_train with gaps,", how, dtype)
    q, k, v, grad, segs = test_gpu_attend_train.make(gpu, structure, 4, 2, 64, dtype, gap=gap)
    want = test_gpu_attend_train.train(q, k, v, grad, segs)[0]
    inside = torch.zeros(q.shape[1], dtype=torch.bool, device=gpu)
    for s in segs:
        inside[s.start:s.end] = True
    assert (want[:, ~inside] == 0).all()
    for _ in range(2):  # (a plan made before, and for the second batch by this call)
        poison(want)
        if how == "frozen":
            out = attend_train(q, k, v, segs, 0)
        else:
            with torch.no_grad() if how == "no_grad" else torch.inference_mode():
                out = attend_train(*(x.detach().requires_grad_() for x in (q, k, v)), segs, 0)
        assert torch.equal(out, want) and not out.requires_grad
        segs = Batch(segment(s.start, s.branch_ids, None, 0, 0, str(gpu)) for s in segs)


def test_no_segment_at_all_gives_zeros_without_a_gradient(gpu):
    say("attend_train, no segment, no gradient")
    q, k = torch.randn(4, 5, 64, device=gpu).to(BF16), torch.randn(2, 5, 64, device=gpu).to(BF16)
    poison(q)
    out = attend_train(q, k, k, Batch(), 0)
    assert out.shape == q.shape and (out == 0).all()


def test_gaps_under_a_reentrant_checkpoint(gpu):
    """Its first forward pass runs without a gradient: what it hands on is what the second one does."""
    say("attend_train with gaps, reentrant checkpoint")
    q, k, v, grad, segs = test_gpu_attend_train.make(gpu, [(40, [5, 9]), (7, [30])], 4, 2, 64, BF16, gap=5)
    want = test_gpu_attend_train.train(q, k, v, grad, segs)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    poison(want[0])
    out = torch.utils.checkpoint.checkpoint(lambda *xs: attend_train(*xs, segs, 0), *leaves, use_reentrant=True)
    assert torch.equal(out, want[0])
    out.backward(grad)
    assert same([x.grad for x in leaves], want[1:])
