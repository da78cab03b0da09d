"""add_norm (dan_amd/csrc/add_norm.hip) against the fp64 oracle.

Tolerances, derived before the first run, with u half a step of the type (eps / 2): a stored
16-bit value is off by u of itself, after fp32 sums of at most some thousand terms (added
pairwise over 64 lanes and more: 2^-18 of the result covers them, the root and the products).
An e4m3 code is off by 2^-4 of its value, or by half of the smallest step (2^-10) near zero.
The gradient reads the sum rounded to 16 bits: each of its two terms moves by at most 2 u."""
import pytest
import torch

from dan_amd.norm import add_norm
from dan_amd.quant import fp8_gemm, fp8_quantize, tile_codes
from oracle import training as oracle

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def say(*a):
    print(*a, flush=True)


def make(gpu, n, k, dtype, seed=0, residual=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, k, generator=g).to(dtype)
    r = (torch.randn(n, k, generator=g) * 3).to(dtype) if residual else None
    w = (torch.randn(k, generator=g) * 0.2 + 1).to(dtype)
    return x.to(gpu), None if r is None else r.to(gpu), w.to(gpu)


def close(name, got, ref, tol):
    got = got.detach().double().cpu()
    worst = ((got - ref).abs() / tol.clamp(min=1e-300)).max().item() if ref.numel() else 0.0
    say(f"  {name}: {worst:.3f} of the tolerance")
    assert worst <= 1, (name, worst)


def check(r, ref, dtype):
    u = torch.finfo(dtype).eps / 2
    for f in ("stream", "out"):
        if getattr(r, f) is not None:
            close(f, getattr(r, f), ref[f], (u + 2 ** -18) * ref[f].abs() + torch.finfo(dtype).tiny * u)
    if r.scale is not None:
        close("scale", r.scale, ref["scale"], 2 ** -18 * ref["scale"])


SHAPES = [(1, 8), (3, 512), (5, 520), (2, 1024), (7, 1032), (33, 2048), (4, 2056), (9, 4096), (3, 4104), (2, 8192), (3, 14336), (2, 16384)]


@pytest.mark.parametrize("norm", ["rms", "zero_centered"])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("n,k", SHAPES)
@pytest.mark.parametrize("residual", [True, False])
def test_forward_and_gradient(gpu, n, k, dtype, norm, residual):
    say(f"add_norm {n} x {k} {dtype} {norm} residual {residual}")
    x, r, w = make(gpu, n, k, dtype, residual=residual)
    g = torch.Generator().manual_seed(1)
    go, gs = (torch.randn(n, k, generator=g).to(dtype).to(gpu) for _ in range(2))
    ref = oracle.add_norm(x, r, w, norm=norm, grad=go, grad_stream=gs if residual else None)
    check(add_norm(x, r, w, norm=norm), ref, dtype)
    leaves = [t.detach().requires_grad_() for t in ((x, r, w) if residual else (x, w))]
    got = add_norm(leaves[0], leaves[1] if residual else None, leaves[-1], norm=norm)
    check(got, ref, dtype)
    outs, grads = ((got.out, got.stream), (go, gs)) if residual else ((got.out,), (go,))
    d = torch.autograd.grad(outs, leaves, grads)
    u = torch.finfo(dtype).eps / 2
    for t in d[:-1]:
        close("ds", t, ref["ds"], (3 * u + 2 ** -17) * ref["abs_ds"] + torch.finfo(dtype).tiny)
    close("dw", d[-1], ref["dw"], (u + 2 ** -17) * ref["abs_dw"] + u * ref["dw"].abs() + torch.finfo(dtype).tiny)


@pytest.mark.parametrize("layout", ["rows", "tiled"])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("n,k", [(1, 16), (5, 528), (7, 1040), (300, 512), (255, 2048), (33, 4112), (2, 14336)])
def test_codes(gpu, n, k, dtype, layout):
    say(f"add_norm codes {n} x {k} {dtype} {layout}")
    x, r, w = make(gpu, n, k, dtype)
    ref = oracle.add_norm(x, r, w)
    rows = add_norm(x, r, w, fp8="rows", out=True)
    check(rows, ref, dtype)
    value = rows.codes.float().double().cpu() * rows.scale.double().cpu()
    close("codes", value, ref["out"], 2 ** -4 * ref["out"].abs() * (1 + 2 ** -10) + 2 ** -10 * ref["scale"] * (1 + 2 ** -10))
    if layout == "tiled":
        tiled = add_norm(x, r, w, fp8="tiled")
        assert tiled.out is None and tiled.codes.shape == (n, k)
        assert torch.equal(tiled.codes.data, tile_codes(rows.codes).data) and torch.equal(tiled.scale, rows.scale)
        wq, ws = fp8_quantize(torch.randn(32, k, device=gpu, dtype=dtype), tiled=True)
        a, b = (fp8_gemm(t.codes, t.scale, wq, ws.reshape(1, -1)) for t in (rows, tiled))
        assert torch.equal(a, b)
