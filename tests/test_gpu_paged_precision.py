"""attend_paged: how exactly its weights and scores are held, at inputs that show it. The oracle is arithmetic in 64 bits,
written out here. u = finfo(dtype).eps / 2 is the rounding of a stored output (bf16 2^-8, fp16 2^-11)."""
import math

import pytest
import torch

from dan_amd.paged import attend_paged

pytestmark = pytest.mark.gpu
BF16, F16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
HALF = {BF16: 2.0 ** -8, F16: 2.0 ** -11}
TYPES = [(BF16, BF16), (F16, F16), (BF16, E4M3), (F16, E4M3)]


def say(msg):
    print(f"[gpu-case] {msg}", flush=True)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def cached(rows, gpu, cache, page=16):
    """Sequences' rows [B, n, Hkv, D] as pages and a table."""
    b, n, hkv, d = rows.shape
    width = -(-n // page)
    full = torch.zeros(b, width * page, hkv, d)
    full[:, :n] = rows
    return full.view(b * width, page, hkv, d).transpose(1, 2).to(cache).contiguous().to(gpu), torch.arange(b * width, dtype=torch.int32).view(b, width).to(gpu)


def call(q, k, v, gpu, cache, ks=1.0, vs=1.0, scale=1.0, **kw):
    """q [B, H, D]; k, v [B, n, Hkv, D] in fp32 (the codes' values of an e4m3 cache)."""
    kc, table = cached(k, gpu, cache)
    vc, _ = cached(v, gpu, cache)
    if cache == E4M3:
        kw.update(k_scale=torch.full((1,), ks, device=gpu), v_scale=torch.full((1,), vs, device=gpu))
    lens = torch.full((q.shape[0],), k.shape[1], dtype=torch.int32, device=gpu)
    out, lse = attend_paged(q.to(gpu).transpose(0, 1), kc, vc, table, lens, scale, return_lse=True, **kw)
    torch.cuda.synchronize()
    return out.transpose(0, 1).cpu().double(), lse.t().cpu().double()


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_weights_have_the_bits_of_fp32(gpu, d, dtype, cache):
    """Three keys: weight 1 on value 0, w on 1 and w e^x on -1, x around 2^-12: what is left of the difference shows the
    weights' own errors. Scores are exact (q a + q x of single products); an exponent's product is off by 1.5 units of 2^-24 times
    its size (<= 1.5), the exponential by 2^-23, so a weight by 2^-22 at most; at most 8 sums of 2^-24 of a weight follow: 2^-20.9
    of (w1 + w2) / Z in all, and the output's own rounding."""
    g = gen(d)
    b, h = 16, 64
    a = -(torch.rand(b, h, generator=g) * 0.8 + 0.7).to(dtype)
    x = ((torch.rand(b, h, generator=g) - 0.5) * 2.0 ** -11).to(dtype)
    q = torch.zeros(b, h, d, dtype=dtype)
    q[..., 3], q[..., 40] = a, x
    k, v = torch.zeros(b, 3, 4, d), torch.zeros(b, 3, 4, d)
    k[:, 1:, :, 3], k[:, 2, :, 40] = 1, 1
    v[:, 1], v[:, 2] = 1, -1
    out, lse = call(q, k, v, gpu, cache)
    w1, w2 = torch.exp(a.double()), torch.exp(a.double() + x.double())
    z = 1 + w1 + w2
    ref = ((w1 - w2) / z)[..., None]
    tol = HALF[dtype] * ref.abs() + (2.0 ** -20.9 * (w1 + w2) / z)[..., None] + (2.0 ** -25 if dtype == F16 else 0.0)
    worst = ((out - ref).abs() / tol).max().item()
    lerr = ((lse - torch.log(z)).abs() / 2.0 ** -21).max().item()
    say(f"weights {dtype} cache={cache} x {d}: {worst:.3f} of the tolerance, lse {lerr:.3f}")
    assert worst <= 1.0 and lerr <= 1.0


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("n", [700, 8193])
def test_many_small_weights_beside_a_large_one(gpu, n, dtype, cache):
    """A first key that takes nearly all (value 0) and n - 1 of weight e^-18 = 2^-26 each (value 1): their sum is the whole output, which
    fp16's subnormals (steps of 2^-24) would not hold. One weight is off by 2^-18 (three roundings of 2^-24 of an exponent of 18, and the
    exponential's own), the sum of n by n 2^-24 more. The sum of all weights is 1 and something: each of its n + 64 additions rounds by up to half a unit of 1, 2^-24,
    and its logarithm is off by as much."""
    d, h = 128, 4
    q = torch.zeros(2, h, d, dtype=dtype)
    q[..., 5] = 1
    k, v = torch.zeros(2, n, 2, d), torch.ones(2, n, 2, d)
    k[:, 1:, :, 5] = -288.0 if cache == E4M3 else -18.0
    v[:, 0] = 0
    out, lse = call(q, k, v, gpu, cache, ks=1 / 16)
    total = (n - 1) * math.exp(-18)
    ref = total / (1 + total)
    tol = (HALF[dtype] + 2.0 ** -18 + (n + 64) * 2.0 ** -24) * ref + (2.0 ** -25 if dtype == F16 else 0.0)
    worst = (out - ref).abs().max().item() / tol
    say(f"small weights {dtype} cache={cache} n={n}: {worst:.3f} of the tolerance")
    assert worst <= 1.0 and (lse - math.log1p(total)).abs().max() <= (n + 64) * 2.0 ** -24


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("d,n", [(64, 5), (128, 40), (256, 40), (64, 3001), (128, 9000), (256, 9000)])
def test_finite_scores_of_any_size(gpu, d, n, dtype, cache):
    """Scores of up to 2^29 (fp16) to 2^40, far apart: the largest takes all, equal ones share, in one range and in several. Products are single and
    exact; the weights are 1 and 0, so that only the output rounds (a sum of two and a quotient by 2 are exact: u |o|), and the logsumexp by 2^-22."""
    g = gen(n + d)
    b, h = 6, 8
    size = 2.0 ** (15 if dtype == F16 else 20)
    q = torch.zeros(b, h, d, dtype=dtype)
    q[..., 7] = torch.where(torch.arange(h) % 2 == 0, size, -size).to(dtype)
    k = torch.zeros(b, n, 2, d)
    steps = torch.randint(-100, 100, (b, n, 2), generator=g).float()
    steps = torch.where(steps == 0, 1.0, steps)
    steps[0, 0], steps[0, n - 1] = 110, 110       # two at the top
    steps[1, n // 2] = 120
    steps[2] = 96                                  # all alike
    steps[3] = -steps[3].abs() - 1                 # all of one sign
    unit = 1.0 if cache == E4M3 else 2.0 ** 8 if dtype == F16 else 2.0 ** 13
    k[..., 7] = (steps * unit).to(cache).float()
    v = torch.randint(-8, 9, (b, n, 2, d), generator=g).float()
    ks = 2.0 ** 12
    out, lse = call(q, k, v, gpu, cache, ks=ks, vs=1.0)
    s = torch.einsum("bhd,bnhd->bhn", q.double(), k.double().repeat_interleave(h // 2, 2)) * (ks if cache == E4M3 else 1.0)
    p = torch.softmax(s, -1)
    assert s.abs().max() >= 2.0 ** 29
    ref = torch.einsum("bhn,bnhd->bhd", p, v.double().repeat_interleave(h // 2, 2))
    some = (p > 0).sum(-1).double()[..., None]     # of many equal ones the sum's quotient by their number rounds, too
    tol = HALF[dtype] * ref.abs() + torch.where(some > 2, 2.0 ** -21, 0.0) * 8
    worst = torch.where(out == ref, 0.0, (out - ref).abs() / tol)
    assert not worst.isnan().any()
    rl = torch.logsumexp(s, -1)
    lerr = ((lse - rl).abs() / (rl.abs() * 2.0 ** -22 + 2.0 ** -21)).max().item()
    say(f"scores to {s.abs().max().item():.3g} {dtype} cache={cache} x {d}, {n} keys: {worst.max().item():.3f} of the tolerance, lse {lerr:.3f}")
    assert worst.max() <= 1.0 and lerr <= 1.0


@pytest.mark.parametrize("n", [5, 64, 700, 9000])
@pytest.mark.parametrize("d", [64, 256])
def test_a_cache_of_scale_zero(gpu, d, n):
    """k_scale 0 makes every score 0: the mean of the values, whole numbers of up to 8 whose sums are exact; u |o| for the output, 2^-23 for the quotient.
    v_scale 0 makes every output 0."""
    g = gen(n)
    q = torch.randn(2, 4, d, generator=g).to(BF16)
    k, v = torch.randint(-8, 9, (2, n, 2, d), generator=g).float(), torch.randint(-8, 9, (2, n, 2, d), generator=g).float()
    out, lse = call(q, k, v, gpu, E4M3, ks=0.0)
    ref = v.double().mean(1).repeat_interleave(2, 1)
    say(f"k_scale 0, {n} keys x {d}: {(out - ref).abs().max().item():.3g}")
    assert ((out - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -20).all() and (lse - math.log(n)).abs().max() <= 2.0 ** -20
    out, lse = call(q, k, v, gpu, E4M3, ks=0.25, vs=0.0)
    assert (out == 0).all() and lse.isfinite().all()
