"""attend_train (dan_amd/csrc/tree_attn_grad.hip) against the fp64 oracle, row by row.

Tolerances, derived before the first run. u is half a step of the inputs' type (bf16 2^-9
.. 2^-8: eps / 2). Rounded to the type: P and dS where they enter a product (u each), the
output where delta reads it (u of |O|, which moves dS by P u sum |G O|), the result itself
(u of its value). The logsumexp's sum is of P rounded to fp16 (2^-11 of each term, which is
at most u), and moves P by as much. So every result lies within 4 u of its bound, the sum of its terms'
magnitudes (the oracle's abs_*), with one u more for the result's own rounding; fp32's
sums and exponentials (2^-24 a step, some hundred steps, scores up to some tens) stay below
2^-12 of it, which one more u covers for bf16 and is added for fp16."""
import math

import pytest
import torch

from dan_amd import workloads
from dan_amd.attention import Batch, attend, attend_train, segment
from oracle import training as oracle

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def say(*a):
    print(*a, flush=True)


def make(gpu, structure, heads, kv_heads, head_dim, dtype, seed=0, pasts=None, std=1.0, gap=0):
    """(q, k, v, G on the GPU, the batch); ``pasts``: a prefix length of each segment; ``gap``: rows of no segment between them."""
    g = torch.Generator().manual_seed(seed)
    n = sum(t + sum(ls) + gap for t, ls in structure)
    rows = (torch.randn(n, heads + 2 * kv_heads, head_dim, generator=g) * std).to(dtype).to(gpu)
    q, k, v = (rows[:, a:b].transpose(0, 1) for a, b in ((0, heads), (heads, heads + kv_heads), (heads + kv_heads, heads + 2 * kv_heads)))
    grad = torch.randn(n, heads, head_dim, generator=g).to(dtype).to(gpu).transpose(0, 1)
    segs, at = Batch(), gap
    for i, (t, ls) in enumerate(structure):
        past = None
        p = pasts[i] if pasts else 0
        if p:
            past = {0: tuple((torch.randn(kv_heads, p, head_dim, generator=g) * std).to(dtype).to(gpu) for _ in range(2))}
        ids = workloads.branch_ids(t, ls)
        segs.append(segment(at, ids, past, 0, p, str(gpu)))
        at += len(ids) + gap
    return q, k, v, grad, segs


def train(q, k, v, grad, segs, scale=None):
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    out = attend_train(*leaves, segs, 0, scale)
    return (out.detach(), *torch.autograd.grad(out, leaves, grad))


def check(got, ref, dtype, names=("out", "dq", "dk", "dv")):
    u = torch.finfo(dtype).eps / 2
    for name, x in zip(names, got, strict=True):
        x, r, bound = x.double().cpu(), ref[name], ref["abs_" + name]
        tol = 6 * u * bound + 2 ** -12 * bound + torch.finfo(dtype).tiny
        worst = ((x - r).abs() / tol).max().item()
        say(f"  {name}: {worst:.3f} of the tolerance")
        assert worst <= 1, (name, worst)


STRUCTURES = {
    "one": [(1, [])],
    "pair": [(1, [1])],
    "trunk": [(64, [])],
    "odd": [(33, [5, 9, 1])],
    "tiles": [(128, [32, 32])],
    "long": [(257, [40, 3, 70])],
    "no_trunk": [(0, [3, 40, 2]), (31, [])],
    "mixed": [(40, [5, 9, 1]), (7, [30]), (1, [3] * 6), (64, []), (13, [17, 2])],
}


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(8, 2, 64), (4, 1, 128), (2, 1, 256), (3, 3, 128), (7, 1, 64), (4, 2, 128)])
@pytest.mark.parametrize("name", STRUCTURES)
def test_against_the_oracle(gpu, name, heads, kv_heads, head_dim, dtype):
    say(f"attend_train {name} {heads}/{kv_heads} x {head_dim} {dtype}")
    q, k, v, grad, segs = make(gpu, STRUCTURES[name], heads, kv_heads, head_dim, dtype)
    check(train(q, k, v, grad, segs), oracle.attend(q, k, v, segs, 0, grad=grad), dtype)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(8, 2, 64), (4, 1, 128), (4, 2, 256)])
def test_behind_a_prefix(gpu, heads, kv_heads, head_dim, dtype):
    say(f"attend_train with prefixes {heads}/{kv_heads} x {head_dim} {dtype}")
    q, k, v, grad, segs = make(gpu, [(40, [5, 9, 1]), (7, [30]), (0, [3, 4]), (13, [17, 2])], heads, kv_heads, head_dim, dtype, pasts=[12, 0, 33, 64])
    check(train(q, k, v, grad, segs), oracle.attend(q, k, v, segs, 0, grad=grad), dtype)
