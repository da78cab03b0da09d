"""token_logprobs at logits of every finite size: masks of -1e9 to -1e37 over whole chunks and whole rows, maxima as large, rows at an offset.

The oracle subtracts the row's maximum before anything else, in 64 bits, so that no logit's size costs it bits. Neither does it the kernel, which
holds x - M and log(sum) apart: tolerances have no term in M but for the logsumexp itself. A sum has terms off by 2^-17 in all (as in
test_gpu_readout.py: 128 roundings of 2^-24 of it), which the logarithm makes absolute; a log probability adds 2^-22 of its own size; the
entropy's sum has terms of weight |log p|: 2^-17 (1 + H + log V)."""
import math

import numpy as np
import pytest
import torch

from dan_amd.readout import token_logprobs

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
SIZES = [9e5, 1.2e6, 1e9, 5e9, 1e10, 1e20, 1e30, 1e37]


def say(msg):
    print(f"[gpu-case] {msg}", flush=True)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def exact(x):
    """log p [N, V] and log(sum e^(x - M)) in 64 bits, the maximum M, and the entropy."""
    x = x.double()
    m = x.amax(1, keepdim=True)
    z = torch.log(torch.exp(x - m).sum(1, keepdim=True))
    logp = (x - m) - z
    p = logp.exp()
    return logp, z[:, 0], m[:, 0], -torch.where(p == 0, 0.0, p * logp).sum(1)


def ordered(x, top):
    return torch.sort(x.double() + 0.0, dim=1, descending=True, stable=True).indices[:, :top]


def rows_of(vocab, size, dtype, g):
    """Rows of finite logits with values of `size` in them."""
    at = torch.arange(vocab)
    x = torch.randn(9, vocab, generator=g) * 3
    few = at < 13
    x[0] = torch.where(few, x[0], -size)                                      # all chunks but the first masked
    x[1] = torch.where(at >= vocab - 2, x[1], -size)                          # all but the last
    x[2] = -size
    x[3] = size
    x[4] = torch.where(torch.rand(vocab, generator=g) < 0.02, x[4], -size)
    x[5] = torch.where(at == vocab // 2, size, x[5])                          # one far above the rest
    x[6] = torch.where(at < vocab // 2, size, -size)
    x[7] = -size + x[7] * (size * 2.0 ** -7)                                   # all of that size, none equal
    x[8] = torch.where(few, x[8], torch.where(at % 2 == 0, -size, -size / 16))
    return x.to(dtype)


def check(x, tokens, top, gpu, entropy=True):
    r = token_logprobs(x.to(gpu), tokens.to(gpu), top=top, entropy=entropy)
    torch.cuda.synchronize()
    logp, z, m, ent = exact(x)
    lowest = -torch.finfo(F32).max
    worst = {}

    def within(name, got, ref, tol):
        got, ref = got.double().cpu(), torch.where(ref < lowest, -math.inf, ref)  # no fp32 holds it: lowest - highest
        err = torch.where(got == ref, 0.0, (got - ref).abs() / tol)
        assert not err.isnan().any(), name
        worst[name] = err.max().item()

    finite = logp.clamp(min=lowest).abs()
    within("logsumexp", r.logsumexp, m + z, 2.0 ** -17 + 2.0 ** -23 * (m + z).abs())
    within("logprobs", r.logprobs, logp.gather(1, tokens), 2.0 ** -17 + 2.0 ** -22 * finite.gather(1, tokens))
    if entropy:
        within("entropy", r.entropy, ent, 2.0 ** -17 * (1 + ent + math.log(x.shape[1])))
    if top:
        ids = ordered(x, top)
        assert torch.equal(r.top_ids.cpu(), ids)
        within("top", r.top_logprobs, logp.gather(1, ids), 2.0 ** -17 + 2.0 ** -22 * finite.gather(1, ids))
    say(f"logprobs {tuple(x.shape)} {x.dtype} top={top}: " + ", ".join(f"{k} {v:.3f}" for k, v in worst.items()) + " of the tolerance")
    assert max(worst.values()) <= 1.0, worst


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("vocab", [300, 5000, 16384, 70000])
def test_finite_logits_of_any_size(gpu, vocab, size, dtype):
    """One chunk a row, a few (one launch), and many (two launches)."""
    g = gen(vocab)
    x = rows_of(vocab, size, dtype, g)
    tokens = torch.stack([torch.randint(0, vocab, (9,), generator=g), torch.full((9,), 5), torch.full((9,), vocab - 1), torch.full((9,), vocab // 2)], 1)
    check(x, tokens, 0, gpu)
    check(x, tokens, 0, gpu, entropy=False)
    check(x, tokens, 7, gpu)
    many = 1100 if vocab <= 16384 else 0  # more rows than one launch takes whole
    if many:
        check(x.repeat(many // 9, 1), tokens.repeat(many // 9, 1), 0, gpu)


@pytest.mark.parametrize("offset", [0.0, 6e4, -6e4])
def test_finite_logits_fp16(gpu, offset):
    x = (torch.randn(9, 9000, generator=gen(3)) * 3)
    x[:4, 100:] = offset
    x[4:] += offset / 2
    check(x.to(F16), torch.randint(0, 9000, (9, 4), generator=gen(4)), 5, gpu)


def test_top_is_a_whole_number(gpu):
    """A fraction is refused, not cut; whole numbers of any type are taken."""
    say("logprobs: top of other types")
    x, t = torch.randn(2, 50, device=gpu), torch.tensor([3, 4], device=gpu)
    want = token_logprobs(x, t, top=3)
    for top in (np.int64(3), torch.tensor(3), 3.0):
        assert torch.equal(token_logprobs(x, t, top=top).top_ids, want.top_ids)
    for top in (2.5, "3", None):
        with pytest.raises((TypeError, ValueError)):
            token_logprobs(x, t, top=top)


# ------------------------------------------------------------------ gradients


class _Rest:
    """Stands for the host module: makes no call, so that the Python functions make every one."""

    append = attend = logprobs = staticmethod(lambda *args: None)


def check_gradient(x, tokens, top, gpu, seed=0):
    """Against the formula in 64 bits with x - M - log(sum) for log p. p is off by 2^-17 for the sum in it, 2^-24 |log p| < 2^-17 for the
    exponent's rounding: 2^-16 of p (|pull| + |g_H| (|log p| + H)), as in test_gpu_readout.py, whatever the logits' size.
    A p below 2^-126, fp32's smallest normal value, is 0 on the hardware: off by less than 2^-126 of what it is a factor of."""
    g = gen(seed)
    n, vocab = x.shape
    leaf = x.to(gpu).requires_grad_()
    r = token_logprobs(leaf, tokens.to(gpu), top=top, entropy=True)
    w = [torch.randn(s, generator=g) for s in (tokens.shape, (n,), (n,), (n, top))]
    outs = [r.logprobs, r.logsumexp, r.entropy] + ([r.top_logprobs] if top else [])
    got = torch.autograd.grad(outs, leaf, [t.to(gpu) for t, _ in zip(w, outs)])[0]
    torch.cuda.synchronize()
    logp, _, _, ent = exact(x)
    p = logp.exp()
    own, mag = torch.zeros_like(logp), torch.zeros_like(logp)
    for ids, h in ((tokens, w[0]), (ordered(x, top), w[3])):
        own.scatter_add_(1, ids, h.double())
        mag.scatter_add_(1, ids, h.double().abs())
    weight = torch.where(p > 0, logp + ent[:, None], 0.0)
    ge = w[2].double()[:, None]
    ref = own + p * (w[1].double()[:, None] - own.sum(1, keepdim=True) - ge * weight)
    pull = w[1].double().abs()[:, None] + mag.sum(1, keepdim=True) + ge.abs() * (torch.where(p > 0, logp.abs(), 0.0) + ent[:, None])
    tol = torch.finfo(x.dtype).eps / 2 * ref.abs() + (2.0 ** -16 * p + 2.0 ** -126) * pull + 2.0 ** -22 * mag + (2.0 ** -25 if x.dtype == F16 else 1e-37)
    worst = ((got.double().cpu() - ref).abs() / tol).max().item()
    say(f"gradient {tuple(x.shape)} {x.dtype} top={top}: {worst:.3f} of the tolerance")
    assert worst <= 1.0
    return got


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size", [1e3, 1e5] + SIZES + [3.3e38])
@pytest.mark.parametrize("vocab", [300, 5000, 33333])
def test_gradient_of_finite_logits_of_any_size(gpu, vocab, size, dtype):
    g = gen(vocab + 1)
    x = rows_of(vocab, size, dtype, g)
    tokens = torch.stack([torch.randint(0, vocab, (9,), generator=g), torch.full((9,), 5)], 1)
    check_gradient(x, tokens, 0, gpu)
    check_gradient(x, tokens, 4, gpu)


@pytest.mark.parametrize("offset", [-1e6, -1e4, -300.0, 77.0, 1e4, 1e6, 1.6e7])
def test_gradient_at_an_offset(gpu, offset):
    """Logits of ordinary spread around an offset, and one value in all places: sum p is 1, not e^(what rounding takes from logsumexp)."""
    vocab = 32000
    x = torch.randn(4, vocab, generator=gen(7)) * 2 + offset
    x[3] = offset
    t = torch.randint(0, vocab, (4, 1), generator=gen(8))
    check_gradient(x, t, 0, gpu)
    leaf = x.to(gpu).requires_grad_()
    (grad,) = torch.autograd.grad(token_logprobs(leaf, t.to(gpu)).logsumexp.sum(), leaf)
    assert (grad.double().sum(1) - 1).abs().max() <= 2.0 ** -16


def test_gradient_of_lowest_rows_through_python(gpu, monkeypatch):
    """The calls that go on in Python keep the same two parts of logsumexp."""
    from dan_amd import _decode

    x = torch.full((3, 700), torch.finfo(F32).min)
    x[1] = 1e6
    x[2, :5] = -1e10
    t = torch.tensor([[3, 200], [0, 699], [4, 9]])
    first = check_gradient(x, t, 2, gpu)
    monkeypatch.setattr(_decode, "calls", lambda: _Rest)
    assert torch.equal(first, check_gradient(x, t, 2, gpu))
