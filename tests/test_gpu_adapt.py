"""adapt (dan_amd/csrc/adapt.hip) against the fp64 oracle, row by row.

Tolerances, derived before the first run: a stored value is off by half a step of its type (u = eps /
2) of itself. Between the two products a value is the sum of two 16-bit numbers: off by 2^-18 (bf16:
2^-9 of 2^-9) of itself, less in fp16, and sums of at most 600 terms in fp32 by 600 x 2^-24 < 2^-14.7
of their terms' magnitudes, twice: 2^-13 of the bound (the oracle's abs_*) covers them."""
import pytest
import torch

from dan_amd.adapters import AdaptedLinear, adapt
from oracle import training as oracle

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def say(*a):
    print(*a, flush=True)


def make(gpu, n, n_in, n_out, rank, count, dtype, seed=0, order="mixed"):
    g = torch.Generator().manual_seed(seed)
    x, y = torch.randn(n, n_in, generator=g).to(dtype), torch.randn(n, n_out, generator=g).to(dtype)
    a, b = (torch.randn(count, rank, n_in, generator=g) * n_in ** -0.5).to(dtype), torch.randn(count, n_out, rank, generator=g).to(dtype)
    if order == "mixed":
        index = torch.randint(-1, count, (n,), generator=g)
    else:
        index = torch.arange(n) * count // max(n, 1)
    scale = torch.rand(count, generator=g) + 0.5
    grad = torch.randn(n, n_out, generator=g).to(dtype)
    return [t.to(gpu) for t in (y, x, a, b, index.int(), scale, grad)]


def check(got, ref, dtype, names):
    u = torch.finfo(dtype).eps / 2
    for name, t in zip(names, got, strict=True):
        t, r, bound = t.detach().double().cpu(), ref[name], ref["abs_" + name]
        tol = u * r.abs() + 2 ** -13 * bound + torch.finfo(dtype).tiny
        worst = ((t - r).abs() / tol).max().item() if t.numel() else 0.0
        say(f"  {name}: {worst:.3f} of the tolerance")
        assert worst <= 1, (name, worst)


def run(y, x, a, b, index, scale, grad):
    leaves = [t.detach().requires_grad_() for t in (x, a, b)]
    out = adapt(y, *leaves, index, scale)
    return (out, *torch.autograd.grad(out, leaves, grad))


SHAPES = [  # rows, n_in, n_out, rank, adapters
    (1, 8, 8, 8, 1), (1, 512, 264, 16, 3), (2, 136, 72, 16, 2), (15, 600, 200, 8, 4), (16, 128, 256, 24, 16), (17, 264, 264, 32, 40),
    (33, 256, 520, 40, 5), (64, 512, 512, 64, 24), (70, 384, 136, 72, 3), (40, 200, 64, 128, 3), (600, 136, 96, 16, 7), (530, 64, 72, 64, 3),
    (130, 600, 600, 1, 2), (50, 64, 64, 3, 2), (20, 128, 128, 100, 2)]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("order", ["mixed", "runs"])
@pytest.mark.parametrize("n,n_in,n_out,rank,count", SHAPES)
def test_against_the_oracle(gpu, n, n_in, n_out, rank, count, dtype, order):
    say(f"adapt {n} rows {n_in} -> {n_out} rank {rank} x {count} {dtype} {order}")
    args = make(gpu, n, n_in, n_out, rank, count, dtype, order=order)
    y, x, a, b, index, scale, grad = args
    ref = oracle.adapt(y, x, a, b, index.tolist(), scale, grad)
    check([adapt(y, x, a, b, index, scale)], ref, dtype, ["out"])
    check(run(*args), ref, dtype, ["out", "dx", "da", "db"])
