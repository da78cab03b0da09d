"""token_logprobs on the GPU against the CPU oracle in float64 (oracle/readout.py).

Tolerances. A sum of e^(x - M) takes at most 64 additions in a lane, 6 across lanes and 2 x 16 in the
joins, each term off by 4 units for the exponential and 2^-23 |x - M| e^(x - M) <= 2^-24 for its argument:
relative 128 x 2^-24 = 2^-17, which the logarithm makes absolute. logsumexp and a log probability add the
rounding of their own size and of M's: 2^-22 (|value| + |M|). The entropy's second sum has terms of weight |log2 p|:
its error is 2^-17 (1 + E|log p|) + 2^-22 log V, E|log p| being the entropy itself (plus |log| of the sum's l >= 1, at
most log V). The gradient is rounded to its type once (u = eps / 2, fp16 subnormals 2^-25), after fp32 products that are off by
2^-16 of p (|pull| + |g_H| (|log p| + H)) and 2^-22 of the given tokens' own gradients."""
import math

import pytest
import torch

from dan_amd.readout import token_logprobs
from oracle import readout as OR

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def say(msg):
    print(f"[gpu-case] {msg}", flush=True)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def within(got, ref, tol):
    got, ref, tol = got.double().cpu(), ref.double(), torch.as_tensor(tol, dtype=torch.float64)
    ref = torch.where(ref.abs() > torch.finfo(F32).max, ref.sign() * math.inf, ref)  # no fp32 holds it: lowest - highest is -inf
    same = (got == ref) | (got.isnan() & ref.isnan())
    over = torch.where(same, 0.0, (got - ref).abs() / tol)
    assert not over.isnan().any() and not torch.isinf(over).any(), "infinities or NaN differ"
    return over.max().item() if over.numel() else 0.0


def check_forward(x, tokens, top, gpu, entropy=True, xd=None):
    r = token_logprobs(x.to(gpu) if xd is None else xd, tokens.to(gpu), top=top, entropy=entropy)
    torch.cuda.synchronize()
    t2 = tokens if tokens.dim() == 2 else tokens[:, None]
    lp, lse, ent, tlp, ids = OR.token_logprobs(x, t2, top)
    m = x.double().amax(1)
    m = torch.where(m.isinf(), 0.0, m).abs()
    row = 2.0 ** -17 + 2.0 ** -22 * (m + torch.where(lse.isinf(), 0.0, lse).abs())
    worst = within(r.logsumexp, lse, row)
    assert r.logprobs.shape == tokens.shape and r.logprobs.dtype == F32
    worst = max(worst, within(r.logprobs.reshape(lp.shape), lp, row[:, None] + 2.0 ** -22 * torch.where(lp.isfinite(), lp.abs(), 0.0)))
    if entropy:
        worst = max(worst, within(r.entropy, ent, 2.0 ** -17 * (1 + ent.nan_to_num() + math.log(x.shape[1])) + 2.0 ** -22 * m))
    else:
        assert r.entropy is None
    if top:
        assert torch.equal(r.top_ids.cpu(), ids), "top ids"
        worst = max(worst, within(r.top_logprobs, tlp, row[:, None] + 2.0 ** -22 * torch.where(tlp.isfinite(), tlp.abs(), 0.0)))
    else:
        assert r.top_ids is None and r.top_logprobs is None
    say(f"logprobs {tuple(x.shape)} {x.dtype} L={t2.shape[1]} top={top}: {worst:.3f} of the tolerance")
    assert worst <= 1.0
    return r


SIZES = [1, 2, 3, 7, 8, 9, 31, 64, 65, 100, 511, 512, 513, 1000, 4095, 4096, 4097, 8191, 50257]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("vocab", SIZES)
def test_forward(gpu, vocab, dtype):
    g = gen(vocab)
    x = (torch.randn(5, vocab, generator=g) * 3).to(dtype)
    check_forward(x, torch.randint(0, vocab, (5,), generator=g), 0, gpu)
    for top in {1, min(vocab, 5), min(vocab, 32)}:
        check_forward(x, torch.randint(-1, vocab, (5, 3), generator=g), top, gpu, entropy=top != 5)


@pytest.mark.parametrize("vocab,dtype", [(128256, BF16), (151936, F16), (262144, F32), (524288, BF16), (524288, F32)])
def test_large_vocabularies(gpu, vocab, dtype):
    g = gen(vocab)
    x = (torch.randn(3, vocab, generator=g) * 2.5).to(dtype)
    check_forward(x, torch.randint(0, vocab, (3, 40), generator=g), 20, gpu)


def test_many_rows(gpu):
    g = gen(1)
    check_forward((torch.randn(700, 1003, generator=g) * 2).to(BF16), torch.randint(0, 1003, (700,), generator=g), 5, gpu)
    check_forward((torch.randn(700, 1003, generator=g) * 2).to(F32), torch.randint(0, 1003, (700, 2), generator=g), 0, gpu)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("vocab", [300, 2048, 4096, 5001, 16384, 16385, 32768, 32769])
def test_few_and_many_rows_agree(gpu, vocab, dtype):
    """Short rows go through one launch or two, by how many there are: to the same bits."""
    g = gen(vocab)
    x = (torch.randn(40, vocab, generator=g) * 2.5).to(dtype)
    t = torch.randint(0, vocab, (40, 2), generator=g)
    xd, td = x.to(gpu).repeat(28, 1), t.to(gpu).repeat(28, 1)
    for top in (0, 5, 32):
        few = check_forward(x, t, top, gpu)
        many = token_logprobs(xd, td, top=top, entropy=True)
        for a, b in zip(few, many):
            assert a is None and b is None or torch.equal(a.repeat(28, *[1] * (a.dim() - 1)), b)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("vocab", [20, 300, 9000, 40000])
def test_equal_and_clustered_logits(gpu, vocab, dtype):
    """Rows of one value, of few values, sorted up and down, signed zeros: ties to the lowest id."""
    g = gen(2)
    rows = [torch.zeros(vocab), torch.full((vocab,), -3.5), torch.randint(0, 2, (vocab,), generator=g).float(),
            torch.randint(0, 7, (vocab,), generator=g).float(), torch.arange(vocab).float() / 64, -torch.arange(vocab).float() / 64,
            torch.where(torch.arange(vocab) % 2 == 0, 0.0, -0.0), torch.where(torch.arange(vocab) == vocab - 1, 9.0, 1.0)]
    x = torch.stack(rows).to(dtype)
    for top in (1, 7, 20):
        check_forward(x, torch.zeros(len(rows), dtype=torch.long), top, gpu)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("vocab", [37, 5000, 33333])
def test_masked_logits(gpu, vocab, dtype):
    """-inf and the type's lowest value in masked places: few tokens left, one, none, all of them lowest."""
    g = gen(vocab)
    x = (torch.randn(8, vocab, generator=g) * 3).to(dtype)
    lowest = torch.finfo(dtype).min
    keep = torch.rand(8, vocab, generator=g) < 0.02
    keep[:, 11] = True
    x[0] = torch.where(keep[0], x[0], -math.inf)
    x[1] = torch.where(keep[1], x[1], lowest)
    x[2] = torch.where(torch.arange(vocab) == 11, x[2], -math.inf)
    x[3] = torch.where(torch.arange(vocab) == 11, x[3], lowest)
    x[4] = -math.inf
    x[5] = lowest
    x[6, 1:] = lowest
    x[6, 0] = -lowest
    x[7, : vocab // 2] = -math.inf
    tokens = torch.tensor([[11, 0, 3]]).repeat(8, 1)
    for top in (0, 5, 20):
        check_forward(x, tokens, top, gpu)


def test_nan_and_infinity_reach_their_row_only(gpu):
    say("logprobs: NaN and +inf")
    x = torch.randn(6, 9001, generator=gen(3)).to(BF16)
    x[1, 8999], x[2, 17], x[3], x[4, 3:] = math.nan, math.inf, math.nan, math.nan
    t = torch.randint(0, 9001, (6,), generator=gen(4))
    for top in (0, 5):
        r = token_logprobs(x.to(gpu), t.to(gpu), top=top, entropy=True)
        for out in (r.logprobs, r.logsumexp, r.entropy) + ((r.top_logprobs.sum(1),) if top else ()):
            assert torch.isnan(out).tolist() == [False, True, True, True, True, False]
        if top:
            assert ((r.top_ids >= 0) & (r.top_ids < 9001)).all()
        good = token_logprobs(x[[0, 5]].to(gpu), t[[0, 5]].to(gpu), top=top, entropy=True)
        assert torch.equal(r.logprobs[[0, 5]], good.logprobs) and torch.equal(r.entropy[[0, 5]], good.entropy)


def test_tokens_padding_and_outside(gpu):
    say("logprobs: padding, tokens past the vocabulary, int32, strided")
    x = torch.randn(4, 50, generator=gen(5)).to(BF16)
    t = torch.tensor([[-1, 3, 49], [50, 3, 3], [-(1 << 62), 1 << 40, 0], [7, 7, 7]])
    r = check_forward(x, t, 3, gpu)
    assert torch.isnan(r.logprobs[1, 0]) and torch.isnan(r.logprobs[2, 1]) and r.logprobs[0, 0] == 0
    small = t.clamp(-1, 60)
    assert torch.equal(token_logprobs(x.to(gpu), small.int().to(gpu)).logprobs.nan_to_num(), token_logprobs(x.to(gpu), small.to(gpu)).logprobs.nan_to_num())
    strided = small.to(gpu).repeat_interleave(2, 1)[:, ::2]
    assert torch.equal(token_logprobs(x.to(gpu), strided).logprobs.nan_to_num(), r.logprobs.nan_to_num())
    column = small.to(gpu)[:, 1]
    assert torch.equal(token_logprobs(x.to(gpu), column).logprobs.nan_to_num(), r.logprobs[:, 1].nan_to_num())
    assert token_logprobs(x.to(gpu), small[:, :0].to(gpu)).logprobs.shape == (4, 0)
    assert token_logprobs(x[:0].to(gpu), small[:0].to(gpu), top=2, entropy=True).top_ids.shape == (0, 2)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strides_and_alignment(gpu, dtype):
    g = gen(6)
    wide = (torch.randn(9, 1100, generator=g) * 2).to(dtype)
    t = torch.randint(0, 1000, (9,), generator=g)
    wd = wide.to(gpu)
    for a in (0, 1, 3, 8):
        check_forward(wide[:, a:a + 1000], t, 5, gpu, xd=wd[:, a:a + 1000])
    check_forward(wide[::2, 5:1006], t[::2], 5, gpu, xd=wd[::2, 5:1006])
    check_forward(wide[:1].expand(9, -1), t, 5, gpu, xd=wd[:1].expand(9, -1))
    check_forward(wide.t()[:9], t % 9, 5, gpu, xd=wd.t()[:9])


# ------------------------------------------------------------------ gradients


def check_gradient(x, tokens, top, gpu, use=("g", "g_lse", "g_entropy", "g_top"), seed=0, xd=None):
    g = gen(seed)
    n, vocab = x.shape
    leaf = (x.to(gpu) if xd is None else xd).detach().requires_grad_()
    r = token_logprobs(leaf, tokens.to(gpu), top=top, entropy="g_entropy" in use)
    w = dict(g=torch.randn(tokens.shape, generator=g), g_lse=torch.randn(n, generator=g), g_entropy=torch.randn(n, generator=g),
             g_top=torch.randn(n, top, generator=g) if top else None)
    w = {k: (v if k in use else None) for k, v in w.items()}
    outs = dict(g=r.logprobs, g_lse=r.logsumexp, g_entropy=r.entropy, g_top=r.top_logprobs)
    pairs = [(outs[k], v.to(gpu)) for k, v in w.items() if v is not None]
    got = torch.autograd.grad([p[0] for p in pairs], leaf, [p[1] for p in pairs])[0]
    torch.cuda.synchronize()
    assert got.dtype == x.dtype and got.shape == x.shape
    t2 = tokens if tokens.dim() == 2 else tokens[:, None]
    if w["g"] is not None:
        w["g"] = w["g"].reshape(t2.shape)
    _, lse, ent, _, ids = OR.token_logprobs(x, t2, top)
    ref = OR.gradient(x, t2, ids, **w)
    logp = x.double() - lse[:, None]
    p = torch.where(lse[:, None] == -math.inf, 0.0, logp.exp())
    zero = torch.zeros(n, 1, dtype=torch.float64)
    pull = sum((w[k].double().abs().reshape(n, -1).sum(1, keepdim=True) if w[k] is not None else zero) for k in ("g", "g_lse", "g_top"))
    if w["g_entropy"] is not None:
        pull = pull + w["g_entropy"].double().abs()[:, None] * (torch.where(p > 0, logp.abs(), 0.0) + ent[:, None])
    own = OR.gradient(torch.zeros_like(x, dtype=torch.float64), t2, ids, g=None if w["g"] is None else w["g"].abs(),
                      g_top=None if w["g_top"] is None else w["g_top"].abs()).abs()
    tol = torch.finfo(x.dtype).eps / 2 * ref.abs() + 2.0 ** -16 * p * pull + 2.0 ** -22 * own + (2.0 ** -25 if x.dtype == F16 else 1e-37)
    worst = within(got, ref, tol)
    say(f"gradient {tuple(x.shape)} {x.dtype} L={t2.shape[1]} top={top} {'+'.join(use)}: {worst:.3f} of the tolerance")
    assert worst <= 1.0
    return got


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("vocab", [1, 7, 8, 9, 513, 4097, 50257])
def test_gradient(gpu, vocab, dtype):
    g = gen(vocab)
    x = (torch.randn(5, vocab, generator=g) * 2).to(dtype)
    top = min(vocab, 4)
    check_gradient(x, torch.randint(0, vocab, (5,), generator=g), 0, gpu, ("g",))
    check_gradient(x, torch.randint(-1, vocab, (5, 3), generator=g), top, gpu)
    for one in ("g_lse", "g_entropy", "g_top"):
        check_gradient(x, torch.randint(0, vocab, (5,), generator=g), top, gpu, (one,))


def test_gradient_of_many_and_equal_labels(gpu):
    """More labels than a wave has lanes, every one of them given several times: they add up."""
    g = gen(9)
    x = torch.randn(3, 600, generator=g)
    check_gradient(x, torch.randint(-1, 20, (3, 150), generator=g), 0, gpu, ("g",))
    check_gradient(x, torch.full((3, 70), 5), 3, gpu)


def test_gradient_of_masked_rows(gpu):
    x = torch.randn(4, 300, generator=gen(10))
    x[0, 20:] = -math.inf
    x[1] = -math.inf
    x[2, 5:] = torch.finfo(F32).min
    t = torch.tensor([[3, 200], [0, 1], [4, -1], [0, 0]])
    got = check_gradient(x, t, 0, gpu, ("g", "g_lse", "g_entropy"))
    assert (got[1] == 0).all() and (got[0, 21:200] == 0).all() and torch.isfinite(got).all()


def test_gradient_layouts(gpu):
    """A padded row stride (the gradient itself is contiguous), an expanded row, a transposed leaf."""
    g = gen(11)
    wide = torch.randn(6, 1037, generator=g).to(BF16)
    t = torch.randint(0, 1001, (6,), generator=g)
    check_gradient(wide[:, 3:1004], t, 3, gpu, xd=wide.to(gpu)[:, 3:1004])
    row = torch.randn(1, 50, generator=g).to(gpu).requires_grad_()
    token_logprobs(row.expand(4, -1), torch.arange(4, device=gpu)).logprobs.sum().backward()
    want = torch.zeros(50, dtype=torch.float64)
    want[:4] += 1
    want -= 4 * torch.softmax(row.detach().cpu().double()[0], 0)
    assert (row.grad.cpu().double()[0] - want).abs().max() < 4 * 2.0 ** -16
    col = torch.randn(50, 4, generator=g).to(gpu).requires_grad_()
    token_logprobs(col.t(), torch.arange(4, device=gpu)).logprobs.sum().backward()
    want = -torch.softmax(col.detach().cpu().double(), 0)
    want[torch.arange(4), torch.arange(4)] += 1
    assert (col.grad.cpu().double() - want).abs().max() < 2.0 ** -16


def test_gradient_against_differences(gpu):
    """Central differences of the kernel's own fp32 forward: truncation h^2 / 6 |f'''| <= 6e-5 with h = 0.02 and weights up to 4, rounding
    2 x 2^-17 x 4 / (2 h) = 1.6e-3."""
    g = gen(12)
    vocab, h = 23, 0.02
    x = torch.randn(vocab, generator=g)
    t = torch.tensor([[3, 7, 7]])

    def f(rows):
        r = token_logprobs(rows, t.expand(rows.shape[0], -1).contiguous().to(gpu), top=4, entropy=True)
        return 0.7 * r.logprobs.sum(1) + 0.4 * r.logsumexp - 0.9 * r.entropy + 0.3 * r.top_logprobs.sum(1)

    leaf = x[None].to(gpu).requires_grad_()
    got = torch.autograd.grad(f(leaf).sum(), leaf)[0][0].cpu()
    step = torch.eye(vocab) * h
    diff = (f((x + step).to(gpu)) - f((x - step).to(gpu))).cpu() / (2 * h)
    assert (got - diff).abs().max() < 1.7e-3


def test_autograd_manners(gpu):
    say("readout: autograd")
    x = torch.randn(3, 40, generator=gen(13)).to(gpu)
    t = torch.tensor([1, 2, 3], device=gpu)
    leaf = x.clone().requires_grad_()
    r = token_logprobs(leaf, t, top=2, entropy=True)
    assert r.logprobs.requires_grad and r.entropy.requires_grad and not r.top_ids.requires_grad
    with torch.no_grad():
        assert not token_logprobs(leaf, t).logprobs.requires_grad
    grad = torch.autograd.grad(r.logprobs.sum(), leaf, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        grad.sum().backward()
    r = token_logprobs(leaf, t)
    with torch.no_grad():
        leaf.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        r.logprobs.sum().backward()
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            token_logprobs(torch.autograd.forward_ad.make_dual(x, x), t)


def test_refusals(gpu):
    say("readout: refusals")
    x, t = torch.zeros(3, 40, device=gpu), torch.zeros(3, dtype=torch.long, device=gpu)
    for bad in ((x.double(), t), (x[0], t), (x[:, :0], t), (x, t[:2]), (x, t.float()), (x, t[:, None, None]), (x, t.cpu())):
        with pytest.raises(ValueError):
            token_logprobs(*bad)
    for top in (-1, 33, 41):
        with pytest.raises(ValueError):
            token_logprobs(x, t, top=top)
    with pytest.raises(ValueError):
        token_logprobs(torch.zeros(1, 524289, device=gpu), t[:1], top=1)
