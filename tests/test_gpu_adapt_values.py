"""adapt and its gradient on values far apart from each other, and on infinities between the two products.

A value v between the two products enters the second one as the sum of two 16-bit numbers. In fp16 it is multiplied before by a power of
2 that is one for a row (out, dx) or a tile of 32 rows (the gradients of a and b) and brings the largest |v| to 2^14 or
above: 2^-25 of a number that is 2^-20 of the largest's size is 2^-25 / 2^(14 - 20) = 2^-19 of it, and what is above that
scale has 22 bits. test_gpu_adapt's tolerance (2^-13 of the sum of magnitudes) holds for it as it stands."""
import math

import pytest
import torch

import test_gpu_adapt
from dan_amd.adapters import adapt
from oracle import training as oracle

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def say(*a):
    print("[gpu-case]", *a, flush=True)


# ---------------------------------------------------------------- values far apart
@pytest.mark.parametrize("rank", [5, 16, 64, 128])
@pytest.mark.parametrize("n", [40, 600])
def test_fp16_rows_of_very_different_size(gpu, n, rank):
    """Rows whose G is 2^20 times the others', and whose x (or the other way round) is zero in the columns looked at: those columns'
    gradients are sums of the small rows' products alone."""
    say("adapt fp16, rows of very different size", n, rank)
    y, x, a, b, _, _, grad = test_gpu_adapt.make(gpu, n, 136, 200, rank, 1, FP16)
    a, big = a * 0.25, torch.arange(n, device=gpu) % 8 == 3
    for name in ("da", "db"):
        z, w = x.clone(), grad.clone()
        if name == "da":  # g of the large rows reaches the last 8 columns of a alone
            w[big], w[~big] = w[big] * 2.0 ** 8, w[~big] * 2.0 ** -12
            z[big, :-8], z[big, -8:] = 0, z[big, -8:] * 2.0 ** -12
            z[~big] *= 2.0 ** 6
        else:  # h of the large rows reaches the last 8 rows of b alone
            z[big], z[~big] = z[big] * 2.0 ** 8, z[~big] * 2.0 ** -12
            w[big, :-8], w[big, -8:] = 0, w[big, -8:] * 2.0 ** -12
            w[~big] *= 2.0 ** 8
        ref = oracle.adapt(y, z, a, b, [0] * n, 0.5, w)
        small = ref[name][0, :, :-8] if name == "da" else ref[name][0, :-8]
        assert small.abs().mean() > 2 ** -9 and all(r.isfinite().all() for r in ref.values())
        test_gpu_adapt.check(test_gpu_adapt.run(y, z, a, b, None, 0.5, w), ref, FP16, ["out", "dx", "da", "db"])


@pytest.mark.parametrize("rank", [5, 16, 64, 128])
@pytest.mark.parametrize("n", [40, 600])
def test_fp16_ranks_of_very_different_size(gpu, n, rank):
    """Ranks whose h is 2^20 times the others' and that some rows of b (or whose g and columns of a) leave out."""
    say("adapt fp16, ranks of very different size", n, rank)
    y, x, a, b, _, _, grad = test_gpu_adapt.make(gpu, n, 136, 200, rank, 1, FP16)
    big = torch.arange(rank, device=gpu) % 4 == 1
    y = y * 0
    for name in ("out", "dx"):
        p, q, w, z = a.clone(), b.clone() * 0.25, grad.clone(), x.clone()
        if name == "out":
            p[0, big], p[0, ~big] = p[0, big] * 2.0 ** 9, p[0, ~big] * 2.0 ** -11
            q[0, :-8, big], q[0, -8:, big] = 0, q[0, -8:, big] * 2.0 ** -9
            q[0, :, ~big] *= 2.0 ** 9
            w *= 2.0 ** -10
        else:
            q[0, :, big], q[0, :, ~big] = q[0, :, big] * 2.0 ** 7, q[0, :, ~big] * 2.0 ** -13
            p[0, big, :-8], p[0, big, -8:] = 0, p[0, big, -8:] * 2.0 ** -9
            p[0, ~big] *= 2.0 ** 11
            z *= 2.0 ** -10
        ref = oracle.adapt(y, z, p, q, [0] * n, 0.5, w)
        small = ref[name][:, :-8]
        assert small.abs().mean() > 2 ** -9 and all(r.abs().max() < 65504 for r in ref.values())
        test_gpu_adapt.check(test_gpu_adapt.run(y, z, p, q, None, 0.5, w), ref, FP16, ["out", "dx", "da", "db"])


# ---------------------------------------------------------------- infinities
def alike(got, ref, dtype, name, bound):
    """Infinities and NaN where the reference has them; within test_gpu_adapt's tolerance elsewhere."""
    got = got.detach().double().cpu()
    assert torch.equal(got.isnan(), ref.isnan()), name
    assert torch.equal(got.isposinf(), ref.isposinf()) and torch.equal(got.isneginf(), ref.isneginf()), name
    rest = ref.isfinite() & bound.isfinite()
    assert torch.equal(rest, ref.isfinite())
    u = torch.finfo(dtype).eps / 2
    tol = u * ref[rest].abs() + 2 ** -13 * bound[rest] + torch.finfo(dtype).tiny
    assert ((got[rest] - ref[rest]).abs() <= tol).all(), name


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("where", ["x", "a", "g"])
@pytest.mark.parametrize("n_in,n_out", [(136, 200), (256, 512)])  # the wide side ends inside a chunk, or with one
@pytest.mark.parametrize("n,rank", [(40, 16), (600, 16), (40, 5), (600, 64), (40, 128), (600, 128)])
def test_infinities_between_the_products(gpu, n, rank, n_in, n_out, where, dtype):
    """x A^T (or G B) of infinities gives what the formula gives: infinities, where no sum meets both of them or a zero."""
    say("adapt: infinite", where, n, rank, n_in, n_out, dtype)
    y, x, a, b, index, scale, grad = test_gpu_adapt.make(gpu, n, n_in, n_out, rank, 3, dtype)
    index[::5] = 1
    a[1], b[1] = a[1].abs() + 2.0 ** -6, b[1].abs() + 2.0 ** -6  # sums of one sign
    hit = index == 1
    row = int(hit.nonzero()[2])
    if where == "x":
        x[row, n_in - 3] = math.inf
    elif where == "a":
        a[1, :, n_in - 3] = math.inf
        x[hit, n_in - 3] = x[hit, n_in - 3].abs() + 2.0 ** -6
    else:
        grad[row, n_out - 3] = math.inf
    ref = oracle.adapt(y, x, a, b, index.tolist(), scale, grad)
    got = dict(zip(("out", "dx", "da", "db"), test_gpu_adapt.run(y, x, a, b, index, scale, grad)))
    assert torch.equal(got["out"], adapt(y, x, a, b, index, scale))
    # what an infinity reaches as an operand of the second product itself may be infinite or NaN: it is left out below
    direct = {"x": ("da",), "a": ("dx",), "g": ("db",)}[where]
    assert any(ref[f].isinf().any() for f in got if f not in direct)
    for f, t in got.items():
        r, bound = ref[f], ref["abs_" + f]
        if f in direct:
            i = (slice(1, 2), slice(None), n_in - 3) if f == "da" else (1, n_out - 3) if f == "db" else (hit.cpu(), n_in - 3)
            keep = torch.ones_like(r, dtype=torch.bool)
            keep[i] = False
            assert not t.detach().cpu()[i].isfinite().any()
            t, r, bound = t.detach().cpu()[keep], r[keep], bound[keep]
        alike(t, r, dtype, f, bound)


@pytest.mark.parametrize("where", ["x", "g"])
@pytest.mark.parametrize("n,n_out,rank", [(6200, 8200, 8), (12300, 4104, 13)])
def test_infinities_in_gradients_of_wide_outputs(gpu, n, n_out, rank, where):
    """The same where dB and g come from one pass: an infinity reaches its own row of dx, and its sums of dA and dB."""
    say("adapt: infinite", where, "wide", n, n_out, rank)
    g = torch.Generator(device=gpu).manual_seed(0)

    def new(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device=gpu) * std).to(BF16)

    x, y, grad, a, b = new(n, 64), new(n, n_out), new(n, n_out), new(1, rank, 64).abs(), new(1, n_out, rank).abs()
    for t in (x, grad, a, b):
        t[t == 0] = 0.5
    want = test_gpu_adapt.run(y, x, a, b, None, 0.5, grad)
    row = 4097
    (x if where == "x" else grad)[row, 13] = math.inf
    out, dx, da, db = test_gpu_adapt.run(y, x, a, b, None, 0.5, grad)
    rest = torch.arange(n, device=gpu) != row
    assert torch.equal(out[rest], want[0][rest]) and torch.equal(dx[rest], want[1][rest])
    if where == "x":  # h = inf: dB is G's sign; dA's column 13 meets x itself
        assert out[row].isposinf().all() and torch.equal(dx, want[1])
        assert torch.equal(db[0], (grad[row].float().sign() * math.inf).to(BF16)[:, None].expand(n_out, rank))
        keep = torch.arange(64, device=gpu) != 13
        assert torch.equal(da[..., keep], want[2][..., keep]) and not da[..., 13].isfinite().any()
    else:  # g = inf: dx, and dA is x's sign; dB's row 13 meets G itself
        assert dx[row].isposinf().all()
        assert torch.equal(da[0], (x[row].float().sign() * math.inf).to(BF16)[None].expand(rank, 64))
        keep = torch.arange(n_out, device=gpu) != 13
        assert torch.equal(db[:, keep], want[3][:, keep]) and not db[:, 13].isfinite().any()
