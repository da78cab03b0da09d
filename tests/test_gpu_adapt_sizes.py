"""adapt and its gradient at sizes that only the kernels for many rows hold in one launch: 2^33 values and more."""
import pytest
import torch

import test_gpu_adapt
from dan_amd.adapters import adapt
from oracle import training as oracle

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def say(*a):
    print("[gpu-case]", *a, flush=True)


def test_2_to_the_20_rows(gpu):
    """x repeats every 1024 rows and y is one row (of stride 0), so the output repeats, bit for bit; a period and the
    gradients against fp64. dB is one row of G by the sum of all h: fp32 sums of up to 2^13 products in a row, 2^-11 of their magnitudes."""
    n, n_in, n_out, period = 1 << 20, 8, 8192, 1024
    say("adapt:", n, "rows,", n_out, "columns")
    _, x, a, b, index, scale, _ = test_gpu_adapt.make(gpu, period, n_in, n_out, 8, 3, BF16)
    y, grad = (torch.randn(1, n_out, device=gpu, generator=torch.Generator(device=gpu).manual_seed(i)).to(BF16) for i in (1, 2))
    rows, idx = x.repeat(n // period, 1), index.repeat(n // period)
    out = adapt(y.expand(n, -1), rows, a, b, idx, scale)
    blocks = out.view(n // period, period, n_out)
    assert all(torch.equal(blocks[i], blocks[0]) for i in range(1, n // period))
    ref = oracle.adapt(y.expand(period, -1), x, a, b, index.tolist(), scale, grad.expand(period, -1))
    test_gpu_adapt.check([blocks[0]], ref, BF16, ["out"])
    del out, blocks

    leaves = [t.detach().requires_grad_() for t in (rows, a, b)]
    dx, da, db = torch.autograd.grad(adapt(y.expand(n, -1), *leaves, idx, scale), leaves, grad.expand(n, -1))
    blocks = dx.view(n // period, period, n_in)
    assert all(torch.equal(blocks[i], blocks[0]) for i in range(1, n // period))
    test_gpu_adapt.check([blocks[0]], ref, BF16, ["dx"])
    u, times = torch.finfo(BF16).eps / 2, n // period
    for name, t in (("da", da), ("db", db)):
        r, bound = times * ref[name], times * ref["abs_" + name]
        assert ((t.double().cpu() - r).abs() <= u * r.abs() + 2 ** -11 * bound).all(), name
