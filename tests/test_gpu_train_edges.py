"""add_norm, adapt and attend_train where they can go wrong: rows that hold infinities or NaN beside rows that do not,
no rows at all, indexes of no adapter, offsets past 32 bits, gradients that fp16 barely holds, buffers behind the last
row, and larger batches; then all of them in one training step and one serving step.

Tolerances as in test_gpu_norm, test_gpu_adapt and test_gpu_attend_train, unless derived where they stand."""
import math

import pytest
import torch
from torch import nn

import test_gpu_adapt
import test_gpu_attend_train
import test_gpu_norm
from dan_amd import _grad, _layer, _native, workloads
from dan_amd.adapters import AdaptedLinear, adapt
from dan_amd.attention import Batch, attend_train, segment
from dan_amd.norm import add_norm
from dan_amd.quant import FP8Linear, fp8_gemm, fp8_quantize
from dan_amd.readout import token_logprobs
from oracle import training as oracle

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def say(*a):
    print("[gpu-case]", *a, flush=True)


# ---------------------------------------------------------------- attend_train
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_rows_of_no_segment_give_zeros(gpu, dtype):
    say("attend_train with gaps", dtype)
    q, k, v, grad, segs = test_gpu_attend_train.make(gpu, [(40, [5, 9]), (7, [30]), (1, [])], 4, 2, 64, dtype, gap=5)
    inside = torch.zeros(q.shape[1], dtype=torch.bool, device=gpu)
    for s in segs:
        inside[s.start:s.end] = True
    # what lies in the gaps reaches nothing: not the power of 2 that fp16's dS is scaled by, either
    grad = (grad.float() * 2.0 ** -10).to(dtype)
    want = test_gpu_attend_train.train(q, k, v, grad, segs)
    for value in (math.nan, math.inf, 6e4):
        poison = [x.clone() for x in (q, k, v, grad)]
        for x in poison:
            x[:, ~inside] = value
        got = test_gpu_attend_train.train(*poison, segs)
        for x, w in zip(got, want):
            assert (x[:, ~inside] == 0).all() and torch.equal(x, w)
    test_gpu_attend_train.check(got, oracle.attend(q, k, v, segs, 0, grad=grad), dtype)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_a_segments_nan_stays_in_it(gpu, dtype):
    say("attend_train: NaN in one segment", dtype)
    q, k, v, grad, segs = test_gpu_attend_train.make(gpu, [(70, [5, 40]), (33, [30]), (64, [2])], 4, 2, 64, dtype)
    want = test_gpu_attend_train.train(q, k, v, grad, segs)
    s = segs[1]
    for i in range(4):
        bad = [x.clone() for x in (q, k, v, grad)]
        bad[i][:, s.start + 3] = math.nan
        got = test_gpu_attend_train.train(*bad, segs)
        for a, b in zip(got, want):
            for t in (segs[0], segs[2]):
                assert torch.equal(a[:, t.start:t.end], b[:, t.start:t.end])


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_no_rows(gpu, dtype):
    say("no rows", dtype)
    q, k = torch.empty(4, 0, 64, dtype=dtype, device=gpu), torch.empty(2, 0, 64, dtype=dtype, device=gpu)
    got = test_gpu_attend_train.train(q, k, k, q, Batch())
    assert [x.shape for x in got] == [q.shape, q.shape, k.shape, k.shape]
    q, k = torch.randn(4, 5, 64, device=gpu).to(dtype), torch.randn(2, 5, 64, device=gpu).to(dtype)  # rows, but no segment
    assert all((x == 0).all() for x in test_gpu_attend_train.train(q, k, k, q, Batch()))
    leaves = [x.requires_grad_() for x in (torch.empty(0, 64, dtype=dtype, device=gpu), torch.ones(64, dtype=dtype, device=gpu))]
    out = add_norm(leaves[0], None, leaves[1])
    dx, dw = torch.autograd.grad(out.out, leaves, torch.empty_like(out.out))
    assert dx.shape == (0, 64) and (dw == 0).all()
    assert add_norm(leaves[0].detach(), None, leaves[1].detach(), fp8="rows").codes.shape == (0, 64)
    x, a, b = torch.empty(0, 64, dtype=dtype, device=gpu), torch.ones(2, 8, 64, dtype=dtype, device=gpu), torch.ones(2, 32, 8, dtype=dtype, device=gpu)
    leaves = [t.requires_grad_() for t in (x, a, b)]
    out = adapt(torch.empty(0, 32, dtype=dtype, device=gpu), *leaves, torch.empty(0, dtype=torch.int32, device=gpu))
    assert out.shape == (0, 32)
    for t, d in zip(leaves, torch.autograd.grad(out, leaves, torch.empty_like(out))):
        assert d.shape == t.shape and (d == 0).all()


def dense(q, k, v, segs, grad, scale):
    """The oracle's results in fp64 on the GPU, whole segments at a time, for batches too large for it row by row."""
    q, k, v, grad = (x.double() for x in (q, k, v, grad))
    h, hkv = q.shape[0], k.shape[0]
    r = {f: torch.zeros_like(x) for f, x in (("out", q), ("abs_out", q), ("dq", q), ("abs_dq", q), ("dk", k), ("abs_dk", k), ("dv", v), ("abs_dv", v))}
    for s in segs:
        a, m = slice(s.start, s.end), s.end - s.start
        see = torch.zeros(m, m, dtype=torch.bool, device=q.device)
        see[:, :s.trunk] = True
        for x, y in s.branches:
            see[x - s.start:y - s.start, x - s.start:y - s.start] = True
        see &= torch.ones_like(see).tril()
        for head in range(h):
            g = head * hkv // h
            qq, kk, vv, gg = q[head, a], k[g, a], v[g, a], grad[head, a]
            p = (qq @ kk.T * scale).masked_fill(~see, -math.inf).softmax(1)
            dp, ap = gg @ vv.T, gg.abs() @ vv.abs().T
            ds = p * (dp - (p * dp).sum(1, keepdim=True))
            ads = p * (dp.abs() + (p * ap).sum(1, keepdim=True))
            r["out"][head, a], r["abs_out"][head, a] = p @ vv, p @ vv.abs()
            r["dq"][head, a], r["abs_dq"][head, a] = scale * (ds @ kk), scale * (ads @ kk.abs())
            r["dk"][g, a] += scale * (ds.T @ qq)
            r["abs_dk"][g, a] += scale * (ads.T @ qq.abs())
            r["dv"][g, a] += p.T @ gg
            r["abs_dv"][g, a] += p.T @ gg.abs()
    return {f: x.cpu() for f, x in r.items()}


def test_the_dense_reference_is_the_oracle(gpu):
    q, k, v, grad, segs = test_gpu_attend_train.make(gpu, [(20, [5, 9]), (0, [3, 4])], 4, 2, 64, BF16)
    want, got = oracle.attend(q, k, v, segs, 0, grad=grad), dense(q, k, v, segs, grad, 0.125)
    for f in got:
        assert (got[f] - want[f]).abs().max().item() <= 1e-12 * max(1.0, want[f].abs().max().item())


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("heads,kv_heads,head_dim,structure", [
    (4, 1, 64, [(1500, [300, 41, 200])]), (4, 2, 128, [(900, [64] * 9), (1023, [])]), (2, 1, 256, [(700, [500, 33]), (0, [129, 257])]),
    (8, 8, 64, [(257, [90] * 4)] * 3)])
def test_longer_batches(gpu, heads, kv_heads, head_dim, structure, dtype):
    say(f"attend_train {heads}/{kv_heads} x {head_dim} {dtype} {structure}")
    q, k, v, grad, segs = test_gpu_attend_train.make(gpu, structure, heads, kv_heads, head_dim, dtype)
    test_gpu_attend_train.check(test_gpu_attend_train.train(q, k, v, grad, segs), dense(q, k, v, segs, grad, head_dim ** -0.5), dtype)


@pytest.mark.parametrize("power", [-12, -6, 8])
def test_fp16_gradients_far_from_1(gpu, power):
    """dS is scaled by a power of 2 before it becomes fp16, so a gradient of 2^power times another's gives 2^power times
    its results, but for what fp16 itself does not hold of them: half a step of its smallest numbers (2^-25)."""
    say("attend_train fp16, gradient times 2 **", power)
    q, k, v, grad, segs = test_gpu_attend_train.make(gpu, [(70, [5, 40]), (33, [30])], 4, 2, 64, FP16)
    grad = (grad.float() / 16).half()
    got = test_gpu_attend_train.train(q, k, v, (grad.double() * 2.0 ** power).half(), segs)
    ref = oracle.attend(q, k, v, segs, 0, grad=(grad.double() * 2.0 ** power).half())
    u = 2 ** -11
    for name, x in zip(("out", "dq", "dk", "dv"), got):
        x, r, bound = x.double().cpu(), ref[name], ref["abs_" + name]
        assert ((x - r).abs() <= 6 * u * bound + 2 ** -12 * bound + 2 ** -24).all(), name


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_scores_that_single_out_one_key(gpu, dtype):
    """Scores of some hundreds: a row's weights are 1 and zeros, and nothing overflows. (fp32 holds a score of 500 to 2^-15,
    which moves P by as much: it is added to the tolerance's share of the bound.)

    Weights this small leave the types' normal numbers, where a rounding is no longer relative. P is off by up to 2^-126
    (bf16: flushed) or 2^-39 (fp16, which holds 2^14 P: half of 2^-24 2^-14), dS, below B = 2 max |G| max |V| (2-norms of rows,
    Cauchy-Schwarz), by 2^-126 more, or by 2^-39 B (fp16: brought to 2^14 and above first). A term of dK or dQ is scale dS times a
    number of q or k, one of dV is P times one of G, and there are at most 2 n of them. The forward pass holds P as fp16 in
    both types: 2^-25 times n numbers of v."""
    say("attend_train, large scores", dtype)
    q, k, v, grad, segs = test_gpu_attend_train.make(gpu, [(70, [5, 40]), (33, [30])], 4, 2, 64, dtype, std=6.0)
    got, ref = test_gpu_attend_train.train(q, k, v, grad, segs), oracle.attend(q, k, v, segs, 0, grad=grad)
    u, n = torch.finfo(dtype).eps / 2, q.shape[1]
    size = {f: x.double().abs().max().item() for f, x in (("q", q), ("k", k), ("v", v), ("g", grad))}
    top = 2 * grad.double().norm(dim=2).max().item() * v.double().norm(dim=2).max().item()
    dp = 2 ** -39 if dtype is FP16 else 2 ** -126
    ds = dp * top + (2 ** -39 * top if dtype is FP16 else 2 ** -126)
    least = dict(out=n * 2 ** -25 * size["v"], dq=2 * n * 0.125 * ds * size["k"], dk=2 * n * 0.125 * ds * size["q"], dv=2 * n * dp * size["g"])
    for name, x in zip(("out", "dq", "dk", "dv"), got):
        tol = (6 * u + 2 ** -11) * ref["abs_" + name] + least[name] + torch.finfo(dtype).tiny
        worst = (x.double().cpu() - ref[name]).abs() / tol
        say(f"  {name}: {worst.max().item():.3f} of the tolerance, where the bound is {ref['abs_' + name].flatten()[worst.argmax()].item():.3g}")
        assert worst.max().item() <= 1, name


@pytest.mark.parametrize("wide", [1 << 24, 1 << 25])
def test_prefixes_with_wide_rows_and_large_offsets(gpu, wide):
    """A prefix whose rows lie 2^24 elements apart, and inputs whose rows do: offsets within a tile pass 2^30 bytes, and
    those of the whole pass 2^32. From 2^25 on they are copied."""
    say(f"attend_train, rows {wide} elements apart")
    q, k, v, grad, segs = test_gpu_attend_train.make(gpu, [(40, [30])], 2, 1, 64, BF16, pasts=[70])
    want = test_gpu_attend_train.train(q, k, v, grad, segs)

    def spread(x):  # [heads, n, d] with token strides of `wide`
        out = torch.empty(x.shape[1] * wide, dtype=x.dtype, device=gpu).as_strided(x.shape, (x.shape[2], wide, 1))
        return out.copy_(x)

    past = {0: tuple(spread(x) for x in segs[0].past[0])}
    far = Batch([segment(0, workloads.branch_ids(40, [30]), past, 0, 70, str(gpu))])
    for a, b in zip(test_gpu_attend_train.train(spread(q), spread(k), spread(v), spread(grad), far), want):
        assert torch.equal(a, b)


def test_backward_leaves_rows_of_no_unit_alone(gpu):
    """The C ABI's own promise: rows outside every unit are left as they are, and nothing is written behind the last row."""
    say("dan_tree_attn_bwd: rows of no segment")
    from dan_amd import attention as A

    q, k, v, grad, segs = test_gpu_attend_train.make(gpu, [(40, [5, 9]), (7, [30])], 4, 2, 64, BF16, gap=3)
    h, n, d = q.shape
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    out = attend_train(*leaves, segs, 0)
    want = torch.autograd.grad(out, leaves, grad)
    t = segs.tile_plan.grad_tables[h, 2, d]
    lse = torch.zeros(h, n, device=gpu)
    args, pasts_host, _ = A._call_args(q, k, v, segs, 0, None, None, _native.PHASES_ALL, False, upload=False)
    A._launch_tree_attn(*args, None, pasts_host, launch=lambda *a: _grad.call_forward_lse(lse.data_ptr(), *a), zero=True)
    buffers = [torch.full((n + 4, x.shape[0], d), 7.0, dtype=BF16, device=gpu) for x in (q, k, v)]
    ws = torch.empty(_grad.workspace_size(h, 2, d, n, t.key_splits), dtype=torch.uint8, device=gpu)
    o = out.detach()
    _grad.call_backward(_native.stream(gpu), _grad.GRAD_ABI_VERSION, _native.DTYPE_BF16, h, 2, d, n, _native.f32(d ** -0.5), t.key_rows,
                        *[f for x in (q, k, v, o, grad) for f in (x.data_ptr(), x.stride(1), x.stride(0))], lse.data_ptr(),
                        *[f for x in buffers for f in (x.data_ptr(), x.stride(0), x.stride(1))], t.keys, t.num_keys, t.queries, t.num_queries,
                        t.row_lo, t.row_end, segs.tile_plan.past_tables[0][0].data_ptr(), 0, ws.data_ptr(), ws.numel(), t.key_splits, 0)
    torch.cuda.synchronize()
    inside = torch.zeros(n + 4, dtype=torch.bool, device=gpu)
    for s in segs:
        inside[s.start:s.end] = True
    for x, w in zip(buffers, want):
        assert (x[~inside] == 7).all() and torch.equal(x[:n][inside[:n]], w.transpose(0, 1)[inside[:n]])


# ---------------------------------------------------------------- adapt
@pytest.mark.parametrize("n", [40, 600])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_indexes_of_no_adapter(gpu, n, dtype):
    say("adapt: negative indexes and ones past the last", n, dtype)
    y, x, a, b, index, scale, grad = test_gpu_adapt.make(gpu, n, 136, 200, 16, 3, dtype)
    index[::7] = -1 - torch.arange(len(index[::7]), device=gpu).int()
    index[3], index[n - 1] = 3, 2 ** 31 - 1
    keep = [i for i in range(n) if i not in (3, n - 1)]
    ref = oracle.adapt(y, x, a, b, index.tolist(), scale, grad)
    for idx in (index, index.long(), torch.where(index == 3, 2 ** 40, index.long())):
        got = test_gpu_adapt.run(y, x, a, b, idx, scale, grad)
        assert got[0][[3, n - 1]].isnan().all() and got[1][[3, n - 1]].isnan().all()
        assert torch.equal(got[0][index < 0], y[index < 0]) and (got[1][index < 0] == 0).all()
        test_gpu_adapt.check([got[0][keep], got[1][keep], *got[2:]],
                             {f: t[keep] if f.endswith(("out", "dx")) else t for f, t in ref.items()}, dtype, ["out", "dx", "da", "db"])


@pytest.mark.parametrize("n", [40, 600])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_an_adapters_nan_stays_with_its_rows(gpu, n, bad, dtype):
    say("adapt: an adapter of", bad, n, dtype)
    y, x, a, b, index, scale, grad = test_gpu_adapt.make(gpu, n, 136, 200, 16, 4, dtype)
    want = test_gpu_adapt.run(y, x, a, b, index, scale, grad)
    a, b, x, grad = (t.clone() for t in (a, b, x, grad))
    a[2, 5], b[2, 7], scale[2] = bad, bad, bad
    x[index == 2], grad[index == 2] = bad, bad
    got = test_gpu_adapt.run(y, x, a, b, index, scale, grad)
    rest = index != 2
    for g, w in zip(got[:2], want[:2]):
        assert torch.equal(g[rest], w[rest])
    for g, w in zip(got[2:], want[2:]):
        assert all(torch.equal(g[i], w[i]) for i in (0, 1, 3))
    # a row without an adapter passes through, whatever x holds there
    x[index < 0] = bad
    assert torch.equal(adapt(y, x, a, b, index, scale)[index < 0], y[index < 0])


@pytest.mark.parametrize("n", [1, 17, 530])
def test_one_adapter_without_an_index_and_a_number_for_scale(gpu, n):
    say("adapt: one adapter, no index", n)
    y, x, a, b, _, _, grad = test_gpu_adapt.make(gpu, n, 136, 200, 16, 1, BF16)
    zero = torch.zeros(n, dtype=torch.int32, device=gpu)
    for scale in (1.0, 0.25, -2, 0.0):
        got = test_gpu_adapt.run(y, x, a, b, None, scale, grad)
        want = test_gpu_adapt.run(y, x, a, b, zero, torch.full((1,), float(scale), device=gpu), grad)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        test_gpu_adapt.check(got, oracle.adapt(y, x, a, b, [0] * n, scale, grad), BF16, ["out", "dx", "da", "db"])


@pytest.mark.parametrize("power", [-20, 12])
def test_fp16_adapters_far_from_1(gpu, power):
    """x A^T may leave fp16's range by far; what comes out of it does not here."""
    for n in (40, 600):
        say("adapt fp16: A times 2 **", power, n)
        y, x, a, b, index, scale, grad = test_gpu_adapt.make(gpu, n, 136, 200, 24, 3, FP16)
        a, b = (a.double() * 2.0 ** (power / 2)).half(), (b.double() * 2.0 ** (-power / 2)).half()
        scale = scale * 2.0 ** -4
        x = (x.double() * 2.0 ** (power / 4)).half()
        ref = oracle.adapt(y, x, a, b, index.tolist(), scale, grad)
        test_gpu_adapt.check(test_gpu_adapt.run(y, x, a, b, index, scale, grad), ref, FP16, ["out", "dx", "da", "db"])


def test_adapters_in_other_layouts(gpu):
    say("adapt: adapters that are views")
    y, x, a, b, index, scale, grad = test_gpu_adapt.make(gpu, 40, 136, 200, 24, 3, BF16)
    want = test_gpu_adapt.run(y, x, a, b, index, scale, grad)
    at, bt = a.transpose(1, 2).contiguous().transpose(1, 2), b.transpose(0, 1).contiguous().transpose(0, 1)
    got = test_gpu_adapt.run(y, x, at, bt, torch.stack((index, index), 1)[:, 0], torch.stack((scale, scale), 1)[:, 1], grad)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("order", ["mixed", "runs"])
@pytest.mark.parametrize("n,n_in,n_out,rank,count", [  # on both sides of where the kernels for many rows begin, for each rank
    (384, 136, 72, 16, 2), (385, 136, 72, 16, 2), (769, 136, 72, 16, 5), (256, 264, 72, 32, 3), (257, 264, 72, 32, 3), (193, 600, 136, 64, 1),
    (385, 72, 264, 40, 6), (160, 520, 264, 128, 2), (161, 520, 264, 128, 2), (321, 136, 200, 104, 9), (1100, 8, 8, 8, 1),
    # ranks that are no multiple of 8, or of 4
    (400, 136, 200, 5, 2), (2, 840, 776, 4, 2), (1, 64, 64, 1, 1), (500, 64, 8, 1, 1), (270, 264, 72, 30, 3), (200, 64, 136, 63, 1), (170, 72, 72, 127, 2),
    (40, 72, 136, 18, 5), (40, 136, 72, 61, 3), (30, 72, 72, 125, 2)])
def test_where_many_rows_begin(gpu, n, n_in, n_out, rank, count, order, dtype):
    say(f"adapt {n} rows {n_in} -> {n_out} rank {rank} x {count} {dtype} {order}")
    args = test_gpu_adapt.make(gpu, n, n_in, n_out, rank, count, dtype, order=order)
    y, x, a, b, index, scale, grad = args
    test_gpu_adapt.check(test_gpu_adapt.run(*args), oracle.adapt(y, x, a, b, index.tolist(), scale, grad), dtype, ["out", "dx", "da", "db"])


@pytest.mark.parametrize("order", ["mixed", "runs", "one"])
@pytest.mark.parametrize("n,n_in,n_out,rank,count", [(12300, 64, 4104, 16, 3), (6200, 136, 8200, 8, 1), (49000, 72, 1032, 16, 2), (3080, 64, 16456, 13, 40)])
def test_gradients_of_wide_outputs(gpu, n, n_in, n_out, rank, count, order):
    """From 96 MB of G on, dB and g come from one pass over it. Against fp64 on the GPU, an adapter at a time. Sums over the
    rows are made in fp32 by parts of at most 2^9 rows a wave, and of some tens of those: 2^-24 (2^9 + 2^6) of their magnitudes, which 2^-13 covers with what the two numbers of v leave."""
    say(f"adapt {n} rows {n_in} -> {n_out} rank {rank} x {count} {order}")
    g = torch.Generator(device=gpu).manual_seed(0)

    def new(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device=gpu) * std).to(BF16)

    x, y, grad, a, b = new(n, n_in), new(n, n_out), new(n, n_out), new(count, rank, n_in, std=n_in ** -0.5), new(count, n_out, rank)
    index = torch.randint(-1, count, (n,), generator=g, device=gpu).int() if order == "mixed" else torch.arange(n, device=gpu).mul(count).div(n, rounding_mode="floor").int()
    if order == "one":
        index = None if count == 1 else torch.full_like(index, count - 1)
    scale = torch.rand(count, generator=g, device=gpu) + 0.5
    got = test_gpu_adapt.run(y, x, a, b, index, scale, grad)
    assert all(torch.equal(p, q) for p, q in zip(got, test_gpu_adapt.run(y, x, a, b, index, scale, grad)))
    ref = {f: torch.zeros_like(t, dtype=torch.float64) for f, t in (("dx", x), ("da", a), ("db", b))}
    ref.update({"abs_" + f: torch.zeros_like(t) for f, t in ref.items()})
    for i in range(count):
        rows = torch.arange(n, device=gpu) if index is None else (index == i).nonzero()[:, 0]
        for prefix, (xx, gg, aa, bb) in (("", (x[rows].double(), grad[rows].double(), a[i].double(), b[i].double())),
                                         ("abs_", (x[rows].double().abs(), grad[rows].double().abs(), a[i].double().abs(), b[i].double().abs()))):
            c, h, low = scale[i].double(), xx @ aa.T, gg @ bb
            ref[prefix + "dx"][rows] = c * (low @ aa)
            ref[prefix + "da"][i], ref[prefix + "db"][i] = c * (low.T @ xx), c * (gg.T @ h)
    test_gpu_adapt.check(got[1:], {f: t.cpu() for f, t in ref.items()}, BF16, ["dx", "da", "db"])


def test_many_adapters_and_few_rows_each(gpu):
    say("adapt: 300 adapters")
    args = test_gpu_adapt.make(gpu, 520, 64, 72, 8, 300, BF16)
    y, x, a, b, index, scale, grad = args
    test_gpu_adapt.check(test_gpu_adapt.run(*args), oracle.adapt(y, x, a, b, index.tolist(), scale, grad), BF16, ["out", "dx", "da", "db"])


def test_rows_past_2_to_the_32_bytes(gpu):
    """x and y of more than 2^32 bytes from the first row to the last: the first and the last rows against the oracle, and the
    gradients, to which only those rows contribute, too."""
    n, wide = 600, 1 << 22
    say("adapt: rows", wide, "elements apart")
    y, x, a, b, index, scale, grad = test_gpu_adapt.make(gpu, n, 136, 200, 16, 3, BF16)
    want = test_gpu_adapt.run(y, x, a, b, index, scale, grad)

    def spread(t):
        return torch.empty(n * wide, dtype=t.dtype, device=gpu).as_strided(t.shape, (wide, 1)).copy_(t)

    got = test_gpu_adapt.run(spread(y), spread(x), a, b, index, scale, spread(grad))
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_the_c_entry_writes_in_place_and_no_row_more(gpu):
    for n in (1, 40, 530):
        say("dan_adapt: out is y itself, rows behind the last", n)
        y, x, a, b, index, scale, grad = test_gpu_adapt.make(gpu, n, 136, 200, 16, 3, BF16)
        want = adapt(y, x, a, b, index, scale)
        out = torch.full((n + 3, 208), 7.0, dtype=BF16, device=gpu)
        out[:n, :200] = y
        nbytes = _layer.adapt_workspace_size(n, 136, 16, 3)
        ws = torch.full((nbytes + 64,), 5, dtype=torch.uint8, device=gpu)
        _layer.call_adapt(_native.stream(gpu), _layer.ADAPT_ABI_VERSION, _native.DTYPE_BF16, n, 136, 200, 16, 3, 0, x.data_ptr(), x.stride(0),
                          out.data_ptr(), 208, a.data_ptr(), b.data_ptr(), index.data_ptr(), scale.data_ptr(), 0.0, out.data_ptr(), 208, 0, ws.data_ptr(), nbytes)
        torch.cuda.synchronize()
        assert torch.equal(out[:n, :200], want) and (out[n:] == 7).all() and (out[:, 200:] == 7).all() and (ws[nbytes:] == 5).all()


@pytest.mark.parametrize("fp8", [False, True])
def test_adapted_linear(gpu, fp8):
    say("AdaptedLinear", "on FP8Linear" if fp8 else "on nn.Linear")
    torch.manual_seed(0)
    linear = nn.Linear(128, 96, dtype=BF16, device=gpu)
    layer = AdaptedLinear(FP8Linear(linear) if fp8 else linear, 3, 8, 0.5)
    x = torch.randn(2, 10, 128, device=gpu, dtype=BF16)
    index = torch.randint(-1, 3, (20,), device=gpu, dtype=torch.int32)
    with torch.no_grad():
        assert torch.equal(layer(x, index), layer.base(x))  # an adapter starts as nothing
        layer.b.normal_()
    assert [n for n, p in layer.named_parameters() if p.requires_grad] == ["a", "b"]
    with torch.no_grad():
        y = layer.base(x).view(20, 96)
    grad = torch.randn(2, 10, 96, device=gpu, dtype=BF16)
    ref = oracle.adapt(y, x.view(20, 128), layer.a, layer.b, index.tolist(), 0.5, grad.view(20, 96))
    out = layer(x, index)
    da, db = torch.autograd.grad(out, (layer.a, layer.b), grad)
    test_gpu_adapt.check([out.view(20, 96), da, db], ref, BF16, ["out", "da", "db"])
    assert layer(x[:0], index[:0]).shape == (0, 10, 96)
    if fp8:
        with pytest.raises(NotImplementedError, match="no gradient of its input"):
            layer(x.requires_grad_(), index)


REFUSALS = [
    (dict(x=lambda t: t[:-1]), ValueError, "N, n_in"), (dict(x=lambda t: t.float()), ValueError, "bf16 or fp16"), (dict(y=lambda t: t.half()), ValueError, "must be"),
    (dict(a=lambda t: t[:, :, :-8]), ValueError, "a must be"), (dict(b=lambda t: t[:1]), ValueError, "a must be"), (dict(a=lambda t: t.cpu()), ValueError, "on"),
    (dict(index=lambda t: None), ValueError, "need an index"), (dict(index=lambda t: t[:-1]), ValueError, "index must be"),
    (dict(index=lambda t: t.float()), ValueError, "index must be"), (dict(index=lambda t: t.cpu()), ValueError, "index must be"),
    (dict(scale=lambda t: t[:-1]), ValueError, "scale must be"), (dict(scale=lambda t: t.double()), ValueError, "scale must be"),
    (dict(scale=lambda t: math.inf), ValueError, "finite"), (dict(scale=lambda t: 1e39), ValueError, "finite"),
    (dict(scale=lambda t: t.clone().requires_grad_()), NotImplementedError, "gradient of scale")]


@pytest.mark.parametrize("changes,error,match", REFUSALS)
def test_adapt_refuses(gpu, changes, error, match):
    y, x, a, b, index, scale, _ = test_gpu_adapt.make(gpu, 4, 136, 200, 16, 3, BF16)
    args = dict(y=y, x=x, a=a, b=b, index=index, scale=scale)
    args.update({f: change(args[f]) for f, change in changes.items()})
    with pytest.raises(error, match=match):
        adapt(**args)


def test_adapt_refuses_ranks_and_widths_that_it_does_not_have(gpu):
    for n_in, n_out, rank in ((132, 200, 16), (136, 204, 16), (136, 200, 129), (136, 200, 0)):
        y, x, a, b = (torch.zeros(s, dtype=BF16, device=gpu) for s in ((2, n_out), (2, n_in), (1, rank, n_in), (1, n_out, rank)))
        with pytest.raises(ValueError, match="multiples of 8|of rank"):
            adapt(y, x, a, b)
    with torch.autograd.forward_ad.dual_level():
        y, x, a, b = (torch.zeros(s, dtype=BF16, device=gpu) for s in ((2, 8), (2, 8), (1, 8, 8), (1, 8, 8)))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            adapt(y, torch.autograd.forward_ad.make_dual(x, x), a, b)


# ---------------------------------------------------------------- add_norm
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("k", [512, 4096, 8192])
def test_a_rows_nan_stays_in_it(gpu, k, dtype):
    say("add_norm: rows of NaN, infinities and zeros", k, dtype)
    x, r, w = test_gpu_norm.make(gpu, 9, k, dtype)
    g = torch.randn(9, k, device=gpu).to(dtype)
    clean, rest = add_norm(x, r, w, fp8="rows", out=True), [0, 2, 4, 6, 8]
    x, r = x.clone(), r.clone()
    x[1], x[3, 5], x[5], r[5], x[7, 0] = math.nan, math.inf, 0.0, 0.0, -math.inf
    got = add_norm(x, r, w, fp8="rows", out=True)
    for a, b in ((got.out, clean.out), (got.stream, clean.stream), (got.codes.view(torch.uint8), clean.codes.view(torch.uint8)), (got.scale, clean.scale)):
        assert torch.equal(a[rest], b[rest])
    assert (got.out[5] == 0).all() and (got.codes[5].float() == 0).all() and got.out[1].isnan().all()
    leaves = [t.detach().requires_grad_() for t in (x, r, w)]
    ds = torch.autograd.grad(add_norm(*leaves).out, leaves, g)[0]
    leaves = [t.detach().requires_grad_() for t in test_gpu_norm.make(gpu, 9, k, dtype)]
    assert torch.equal(ds[rest], torch.autograd.grad(add_norm(*leaves).out, leaves, g)[0][rest])


def test_large_values_of_fp16(gpu):
    """Values near fp16's largest: squares and sums are fp32's; a sum past 65504 is infinite as `stream`, not in the norm."""
    say("add_norm fp16: large values")
    x, r, w = test_gpu_norm.make(gpu, 5, 1024, FP16)
    x, r = (x.float() * 15000).clamp(-60000, 60000).half(), (r.float() * 5000).clamp(-60000, 60000).half()
    got, ref = add_norm(x, r, w), oracle.add_norm(x, r, w)
    u = 2 ** -11
    test_gpu_norm.close("out", got.out, ref["out"], (u + 2 ** -18) * ref["out"].abs() + 2 ** -24)
    over = ref["stream"].abs() >= 65520
    assert over.any() and got.stream.cpu()[over].isinf().all()


def test_the_norms_c_entry_writes_in_place_and_no_row_more(gpu):
    for n, k in ((1, 264), (9, 2048), (300, 520)):
        say("dan_add_norm: stream is the residual itself, rows behind the last", n, k)
        x, r, w = test_gpu_norm.make(gpu, n, k, BF16)
        want = add_norm(x, r, w)
        stream = torch.full((n + 3, k + 8), 7.0, dtype=BF16, device=gpu)
        stream[:n, :k] = r
        out = torch.full((n + 3, k + 8), 7.0, dtype=BF16, device=gpu)
        _layer.call_norm(_native.stream(gpu), _layer.NORM_ABI_VERSION, _native.DTYPE_BF16, n, k, 0, 0, _native.f32(1e-6), 0, x.data_ptr(), x.stride(0),
                         stream.data_ptr(), k + 8, w.data_ptr(), stream.data_ptr(), k + 8, out.data_ptr(), k + 8, 0, 0, 0)
        torch.cuda.synchronize()
        for t, u in ((stream, want.stream), (out, want.out)):
            assert torch.equal(t[:n, :k], u) and (t[n:] == 7).all() and (t[:, k:] == 7).all()


@pytest.mark.parametrize("kw,error,match", [
    (dict(norm="layer"), ValueError, "norm"), (dict(fp8="columns"), ValueError, "fp8"), (dict(out=False), ValueError, "nothing is left"),
    (dict(eps=-1.0), ValueError, "eps"), (dict(eps=math.nan), ValueError, "eps"), (dict(eps=math.inf), ValueError, "eps"),
    (dict(x=lambda t: t.float()), ValueError, "bf16 or fp16"), (dict(x=lambda t: t[None]), ValueError, "N, K"), (dict(x=lambda t: t[:, :60]), ValueError, "multiple of 8"),
    (dict(residual=lambda t: t[:2]), ValueError, "residual"), (dict(residual=lambda t: t.half()), ValueError, "residual"),
    (dict(weight=lambda t: t[:8]), ValueError, "weight"), (dict(weight=lambda t: t.float()), ValueError, "weight"), (dict(weight=lambda t: t.cpu()), ValueError, "weight"),
    (dict(fp8="rows", weight=lambda t: t.clone().requires_grad_()), NotImplementedError, "no gradient")])
def test_add_norm_refuses(gpu, kw, error, match):
    x, r, w = test_gpu_norm.make(gpu, 3, 64, BF16)
    args = dict(x=x, residual=r, weight=w)
    for f, change in kw.items():
        args[f] = change(args[f]) if callable(change) else change
    with pytest.raises(error, match=match):
        add_norm(args.pop("x"), args.pop("residual"), args.pop("weight"), **args)


def test_add_norm_refuses_widths_that_it_does_not_have(gpu):
    for k, fp8 in ((0, None), (16392, None), (72, "rows")):
        with pytest.raises(ValueError, match="multiple of"):
            add_norm(torch.zeros(2, k, dtype=BF16, device=gpu), None, torch.ones(k, dtype=BF16, device=gpu), fp8=fp8)


# ---------------------------------------------------------------- together
def steps(p, x, rows, segs, index, tokens, ops):
    """One decoder layer with adapters on two projections and the log probabilities of the next tokens, by `ops`."""
    norm, project, attention, logprobs = ops
    h, hkv, d = 4, 2, 64
    first, stream = norm(x, None, p["norm1"])
    qkv = project(first, "qkv", index)
    q, k, v = (t.view(rows, -1, d).transpose(0, 1) for t in qkv.split((h * d, hkv * d, hkv * d), 1))
    o = attention(q, k, v).transpose(0, 1).reshape(rows, h * d)
    second, stream = norm(project(o, "out", index), stream, p["norm2"])
    return logprobs(second @ p["head"].T), stream


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_a_training_step(gpu, dtype):
    """Against the same step in fp64. Between the loss and a gradient lie about twelve results that are rounded to the type
    on the way forward and as many on the way back, each off by at most two halves of a step (2 u) of its norm, where no
    step makes an error grow by more than the value itself: 48 u in the 2-norm."""
    say("a training step", dtype)
    g = torch.Generator().manual_seed(0)
    structure, model, h, hkv, d, vocab = [(40, [9, 17]), (21, [5, 5, 5])], 128, 4, 2, 64, 200
    segs, n = Batch(), 0
    for t, ls in structure:
        ids = workloads.branch_ids(t, ls)
        segs.append(segment(n, ids, None, 0, 0, str(gpu)))
        n += len(ids)

    def new(*shape, std):
        return (torch.randn(*shape, generator=g) * std).to(dtype)

    wide = (h + 2 * hkv) * d
    p = dict(norm1=new(model, std=0.1) + 1, norm2=new(model, std=0.1) + 1, head=new(vocab, model, std=model ** -0.5),
             qkv=new(wide, model, std=model ** -0.5), out=new(model, h * d, std=(h * d) ** -0.5),
             qkv_a=new(3, 16, model, std=model ** -0.5), qkv_b=new(3, wide, 16, std=0.2), out_a=new(3, 8, h * d, std=(h * d) ** -0.5), out_b=new(3, model, 8, std=0.2))
    x = new(n, model, std=1.0)
    index = torch.cat([torch.full((s.end - s.start,), i, dtype=torch.int32) for i, s in enumerate(segs)])
    index[::11] = -1
    tokens = torch.randint(0, vocab, (n,), generator=g)
    tokens[::9] = -1  # no label there
    learnt = ("norm1", "norm2", "qkv_a", "qkv_b", "out_a", "out_b")

    def run(to, ops_of):
        q = {f: to(t).requires_grad_(f in learnt) for f, t in p.items()}
        rows = to(x).requires_grad_()
        lp, stream = steps(q, rows, n, segs, index, tokens, ops_of(q))
        loss = -lp.sum() / 100 + stream.to(torch.float64).square().sum() / 1e4
        return [lp.detach(), stream.detach()] + list(torch.autograd.grad(loss, [rows] + [q[f] for f in learnt]))

    def here(q):
        idx, tok = index.to(gpu), tokens.to(gpu)
        return (lambda a, b, w: add_norm(a, b, w)[:2], lambda t, name, _: adapt(t @ q[name].T, t, q[name + "_a"], q[name + "_b"], idx, 0.5),
                lambda a, b, c: attend_train(a, b, c, segs, 0), lambda logits: token_logprobs(logits, tok).logprobs)

    def plain(q):
        def norm(a, b, w):
            s = a if b is None else a + b
            return nn.functional.rms_norm(s, (model,), w, 1e-6), s

        def project(t, name, _):
            hot = nn.functional.one_hot(index.long().clamp(min=0), 3).double() * (index >= 0)[:, None]
            low = torch.einsum("nk,rjk->nrj", t, q[name + "_a"])
            return t @ q[name].T + 0.5 * torch.einsum("nrj,rmj,nr->nm", low, q[name + "_b"], hot)

        def attention(a, b, c):
            see = torch.zeros(n, n, dtype=torch.bool)
            for s in segs:
                see[s.start:s.end, s.start:s.start + s.trunk] = True
                for u, w in s.branches:
                    see[u:w, u:w] = True
            see &= torch.ones_like(see).tril()
            b, c = (t.repeat_interleave(h // hkv, 0) for t in (b, c))
            return (a @ b.transpose(1, 2) * d ** -0.5).masked_fill(~see, -math.inf).softmax(2) @ c

        def logprobs(logits):
            lp = logits.log_softmax(1).gather(1, tokens.clamp(min=0)[:, None])[:, 0]
            return torch.where(tokens >= 0, lp, 0.0)

        return norm, project, attention, logprobs

    got, ref = run(lambda t: t.clone().to(gpu), here), run(lambda t: t.double(), plain)
    u = torch.finfo(dtype).eps / 2
    for name, a, b in zip(("logprobs", "stream", "x", *learnt), got, ref, strict=True):
        a = a.double().cpu()
        if name == "logprobs":
            a = torch.where(tokens >= 0, a, 0.0)
        error = ((a - b).norm() / b.norm()).item()
        say(f"  {name}: {error:.4f} of its norm, {48 * u:.4f} allowed")
        assert error <= 48 * u, name
    again = run(lambda t: t.clone().to(gpu), here)
    assert all(torch.equal(a, b) for a, b in zip(got[1:], again[1:]))


def test_a_serving_step_captured(gpu):
    """add_norm as codes and as rows, the e4m3 projection, and each request's adapter beside it, captured and replayed: against the
    calls made eagerly, and adapt's part against the oracle."""
    say("a serving step: add_norm, fp8_gemm, adapt")
    n, k, m = 7, 256, 320
    x, r, w = test_gpu_norm.make(gpu, n, k, BF16)
    wq, ws = fp8_quantize(torch.randn(m, k, device=gpu, dtype=BF16) * k ** -0.5, tiled=True)
    _, _, a, b, index, scale, _ = test_gpu_adapt.make(gpu, n, k, m, 16, 4, BF16)

    def step():
        s = add_norm(x, r, w, fp8="tiled", out=True)
        y = fp8_gemm(s.codes, s.scale, wq, ws.reshape(1, -1))
        return s.out, s.stream, y, adapt(y, s.out, a, b, index, scale)

    with torch.no_grad():
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
            got = step()
        gen = torch.Generator(device=gpu).manual_seed(1)
        for _ in range(3):
            for t in (x, r):
                t.copy_(torch.randn(t.shape, device=gpu, generator=gen).to(BF16))
            index.copy_(torch.randint(-1, 4, (n,), device=gpu, generator=gen))
            graph.replay()
            torch.cuda.synchronize()
            have = [t.clone() for t in got]
            assert all(torch.equal(p, q) for p, q in zip(have, step()))
            test_gpu_adapt.check([have[3]], oracle.adapt(have[2], have[0], a, b, index.tolist(), scale), BF16, ["out"])
