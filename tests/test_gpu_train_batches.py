"""attend_train over batches that change or that training and other calls share: rows of no segment where nothing needs a
gradient, tables uploaded on another stream, first calls in a capture, prefix-cache entries replaced between calls.

Results are compared bit for bit with those of the same kernels on the same values."""
import math

import pytest
import torch
import torch.utils.checkpoint

import test_gpu_attend_train
from dan_amd import workloads
from dan_amd.attention import Batch, attend, attend_train, segment
from oracle import training as oracle
from test_gpu_train_calls import same, say, way, ways  # noqa: F401  -- the fixture of `ways`

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


# ---------------------------------------------------------------- batches
def entry(gpu, seed, length, dtype=BF16, heads=2, d=64, other=False):
    g = torch.Generator().manual_seed(seed)
    new = [torch.randn(heads, length, d, generator=g).to(dtype).to(gpu) for _ in range(2)]
    if other:  # (rows that the kernels read from a copy)
        new = [torch.nn.functional.pad(x, (3, 2))[..., 3:-2] for x in new]
    return tuple(new)


def batch(gpu, lengths, pasts):
    segs, at = Batch(), 0
    for (t, ls), past in zip(lengths, pasts):
        ids = workloads.branch_ids(t, ls)
        segs.append(segment(at, ids, past, 0, past[0][0].shape[1] if past else 0, str(gpu)))
        at += len(ids)
    return segs, at


def train(q, k, v, grad, segs, layer=0):
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    out = attend_train(*leaves, segs, layer)
    return out.detach(), *torch.autograd.grad(out, leaves, grad)


# ---------------------------------------------------------------- streams
def slow(x):
    for _ in range(150):
        torch.mm(x, x)


@pytest.fixture(scope="module")
def big(gpu):
    x = torch.randn(8192, 8192, device=gpu, dtype=BF16)
    slow(x)
    torch.cuda.synchronize()
    return x


def many(gpu, seed, count=12, other=False):
    """(q, k, v, G, a function that makes the batch): each segment behind an entry of its own, more than a launch carries by value."""
    lengths = [(20 + i, [3, 4]) for i in range(count)]
    pasts = [{layer: entry(gpu, 100 * layer + i, 5 + i, other=other) for layer in range(3)} for i in range(count)]
    n = sum(t + sum(ls) for t, ls in lengths)
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(h, n, 64, generator=g).to(BF16).to(gpu) for h in (4, 2, 2, 4)], lambda: batch(gpu, lengths, pasts)[0]


@ways
@pytest.mark.parametrize("other", [False, True])
@pytest.mark.parametrize("count", [3, 12])
def test_a_plan_made_behind_slow_work_on_another_stream(gpu, big, count, other, way):  # noqa: F811
    """attend on one stream makes the plan and a layer's prefix table; attend_train of it and of another layer on a second stream, and
    of the first's layers on a third, wait for what they read, with and without a gradient."""
    say("attend_train on another stream than the plan's", count, other, way)
    x, make = many(gpu, 3, count, other)
    want = [train(*x, make(), layer) for layer in range(3)]
    b, c = torch.cuda.Stream(), torch.cuda.Stream()
    for first, a in (("grad", torch.cuda.Stream()), ("no_grad", torch.cuda.Stream()), ("grad", torch.cuda.default_stream())):
        segs = make()
        torch.cuda.synchronize()
        with torch.cuda.stream(a):
            slow(big)
            out = [attend(*x[:3], segs, 0)]
        with torch.cuda.stream(b):
            if first == "grad":
                got = [train(*x, segs, 0)]
            else:
                with torch.no_grad():
                    out.append(attend_train(*x[:3], segs, 0))
                got = []
            slow(big)
            got.append(train(*x, segs, 1))
        with torch.cuda.stream(c):
            more = [train(*x, segs, 0), train(*x, segs, 1), train(*x, segs, 2)]
        torch.cuda.synchronize()
        assert all(torch.equal(o, want[0][0]) for o in out)
        assert all(same(g, want[i]) for i, g in zip((0, 1) if first == "grad" else (1,), got))
        assert all(same(g, w) for g, w in zip(more, want))


@ways
def test_a_later_layers_table_uploaded_on_another_stream(gpu, big, way):  # noqa: F811
    say("attend_train: a later layer's prefix table behind slow work", way)
    x, make = many(gpu, 4)
    want = [train(*x, make(), layer) for layer in range(2)]
    segs = make()
    assert same(train(*x, segs, 0), want[0])
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(a):
        slow(big)
        first = train(*x, segs, 1)  # (uploads the layer's table)
    with torch.cuda.stream(b):
        second = train(*x, segs, 1)
    torch.cuda.synchronize()
    assert same(first, want[1]) and same(second, want[1])


@ways
@pytest.mark.parametrize("count", [3, 12])
def test_a_table_in_memory_that_its_stream_still_uses(gpu, big, count, way):  # noqa: F811
    """A prefix table takes memory that was given back on its stream, where work that uses it may still be to come: a call on another
    stream, which writes the table (3 entries) or reads it (12), comes behind that work."""
    say("attend_train: a layer's table in memory still in use", count, way)
    x, make = many(gpu, 8, count)
    want = [train(*x, make(), layer) for layer in range(2)]
    segs = make()
    b, c = torch.cuda.Stream(), torch.cuda.Stream()
    nbytes = segs_table_bytes(segs)
    with torch.cuda.stream(b):
        assert same(train(*x, segs, 0), want[0])
        segs.tile_plan.spare.clear()  # (or the layer's table would be there already)
        small = [torch.full((nbytes,), i % 251, dtype=torch.uint8, device=gpu) for i in range(512)]  # (also the holes that were there)
    torch.cuda.synchronize()
    with torch.cuda.stream(b):
        slow(big)
        copies = [t.clone() for t in small[::2]]
        del small[::2]
        first = train(*x, segs, 1)
    with torch.cuda.stream(c):
        second = train(*x, segs, 1)
    torch.cuda.synchronize()
    assert same(first, want[1]) and same(second, want[1])
    assert all((t == 2 * i % 251).all() for i, t in enumerate(copies))


def segs_table_bytes(segs):
    return max(72 * len(segs), 512)  # a DanPastDesc each, and what the allocator rounds to


@ways
@pytest.mark.parametrize("needs", [True, False])
def test_a_batch_dropped_before_another_stream_has_read_it(gpu, big, needs, way):  # noqa: F811
    """Tables that were allocated on the stream of the first call, read on another one: their memory is not given away before that."""
    say("attend_train: batch dropped behind slow work", needs, way)
    x, make = many(gpu, 5)
    want = train(*x, make())
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(a):
        segs = make()
        assert same(train(*x, segs), want)
    torch.cuda.synchronize()
    with torch.cuda.stream(b):
        slow(big)
        if needs:
            got = train(*x, segs)
        else:
            with torch.no_grad():
                got = [attend_train(*x[:3], segs, 0)]
    del segs
    with torch.cuda.stream(a):  # what takes the place of freed tables: zeros, which name no rows
        zeros = [torch.zeros(s, dtype=torch.uint8, device=gpu) for s in (256, 512, 1024, 2048, 4096, 8192, 16384, 32768, 65536) for _ in range(40)]
    torch.cuda.synchronize()
    assert same(got, want[:len(got)]) and all((z == 0).all() for z in zeros[::40])


# ---------------------------------------------------------------- captures
@ways
@pytest.mark.parametrize("kept", [True, False])
@pytest.mark.parametrize("needs", [True, False])
def test_a_refused_capture_leaves_nothing_behind(gpu, needs, kept, way):  # noqa: F811
    """A batch whose very first call is in a capture: refused before a table is made, since one made there would be kept on the batch
    and never filled. What the message asks for then works."""
    say("attend_train: first call of a new batch in a capture", needs, kept, way)
    x, make = many(gpu, 6, 3)
    want = train(*x, make())
    segs = make() if kept else list(make())
    leaves = [t.detach().requires_grad_(needs) for t in x[:3]]
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="before a capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=torch.cuda.Stream()):
            attend_train(*leaves, segs, 0)
    torch.cuda.synchronize()
    assert getattr(segs, "tile_plan", None) is None
    assert same(train(*x, segs), want)


@ways
@pytest.mark.parametrize("count,other,allowed", [(3, False, True), (3, True, False), (12, False, False)])
def test_another_layers_first_call_in_a_capture(gpu, count, other, allowed, way):  # noqa: F811
    """A layer that the warm-up left out is captured where that uploads and copies nothing, and refused otherwise; in either
    case an eager call of it is right afterwards, before any replay, and so is each replay."""
    say("attend_train: first call of a layer in a capture", count, other, way)
    x, make = many(gpu, 7, count, other)
    want = [train(*x, make(), layer) for layer in range(2)]
    segs = make()
    assert same(train(*x, segs, 0), want[0])
    leaves = [t.detach().requires_grad_() for t in x[:3]]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    if allowed:
        with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
            out = attend_train(*leaves, segs, 1)
            got = [out.detach(), *torch.autograd.grad(out, leaves, x[3])]
    else:
        with pytest.raises(RuntimeError, match="before a capture"):
            with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
                attend_train(*leaves, segs, 1)
    torch.cuda.synchronize()
    assert same(train(*x, segs, 1), want[1])
    if allowed:
        for _ in range(3):
            for t in got:
                t.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert same(got, want[1]) and same(train(*x, segs, 1), want[1])


# ---------------------------------------------------------------- prefix-cache entries
LENGTHS = [(40, [5, 9]), (0, [3, 4]), (7, [2])]


@ways
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("change", ["entry", "dict", "swap", "longer", "copy"])
def test_prefix_entries_replaced_between_calls(gpu, change, dtype, way):  # noqa: F811
    """A batch that is run again behind other prefixes (as when each step of a training loop makes them anew) reads those."""
    say("attend_train, prefix replaced:", change, dtype, way)
    other = change == "copy"
    dicts = [{0: entry(gpu, 1, 12, dtype, other=other)}, None, {0: entry(gpu, 2, 12, dtype, other=other)}]
    segs, n = batch(gpu, LENGTHS, dicts)
    g = torch.Generator().manual_seed(3)
    q, k, v, grad = (torch.randn(h, n, 64, generator=g).to(dtype).to(gpu) for h in (4, 2, 2, 4))
    first = test_gpu_attend_train.train(q, k, v, grad, segs)
    if change == "entry":
        segs[0].past[0] = entry(gpu, 5, 12, dtype)
    elif change == "dict":
        segs[0].past = {0: entry(gpu, 5, 12, dtype)}
    elif change == "swap":
        segs[0].past, segs[2].past = segs[2].past, segs[0].past
    elif change == "longer":
        segs[0].past, segs[0].past_len = {0: entry(gpu, 5, 33, dtype)}, 33
    else:
        segs[0].past[0][0].mul_(0.5)
        segs[2].past[0][1].add_(1)
    fresh, _ = batch(gpu, LENGTHS, [s.past for s in segs])
    want = test_gpu_attend_train.train(q, k, v, grad, fresh)
    assert not torch.equal(want[0], first[0])
    for _ in range(2):
        assert same(test_gpu_attend_train.train(q, k, v, grad, segs), want)
        with torch.no_grad():
            assert torch.equal(attend_train(q, k, v, segs, 0), want[0])
    test_gpu_attend_train.check(want, oracle.attend(q, k, v, segs, 0, grad=grad), dtype)


@ways
def test_an_entry_that_the_batch_itself_saves(gpu, way):  # noqa: F811
    """A segment behind another one's saved rows: each call reads the rows that it has saved, not an earlier call's, in each layer."""
    say("attend_train, a prefix that the batch saves", way)

    def make():
        segs, n = batch(gpu, [(20, [5]), (9, [4, 3])], [None, None])
        segs[0].save = 13
        segs[1].past, segs[1].past_len = segs[0].saved, 13
        return segs, n

    segs, n = make()
    g = torch.Generator().manual_seed(3)
    sets = [[torch.randn(h, n, 64, generator=g).to(BF16).to(gpu) for h in (4, 2, 2, 4)] for _ in range(3)]
    want = [train(*x, make()[0], 0) for x in sets]
    for _ in range(2):
        for layer in (0, 1):
            for x, w in zip(sets, want):
                assert same(train(*x, segs, layer), w)
    for x, w in zip(sets, want):
        assert torch.equal(attend_train(*x[:3], segs, 0), w[0])


@pytest.mark.parametrize("change", ["dict", "grown"])
def test_a_batch_changed_before_another_layers_first_call(gpu, change):
    say("attend_train, batch changed before another layer:", change)
    dicts = [{i: entry(gpu, 1 + i, 12) for i in range(2)}, None, None]
    segs, n = batch(gpu, LENGTHS[:2], dicts)
    g = torch.Generator().manual_seed(3)
    x = [torch.randn(h, n + 9, 64, generator=g).to(BF16).to(gpu) for h in (4, 2, 2, 4)]
    train(*x, segs, 0)
    if change == "dict":
        segs[0].past, segs[0].past_len = {i: entry(gpu, 5 + i, 20) for i in range(2)}, 20
    else:
        segs.append(segment(n, workloads.branch_ids(*LENGTHS[2]), None, 0, 0, str(gpu)))
    for layer in (1, 0):
        want = train(*x, Batch(segs), layer)
        assert same(train(*x, segs, layer), want) and torch.equal(attend_train(*x[:3], segs, layer), want[0])


def test_captured_without_a_gradient(gpu):
    """Behind attend's plan, rows of no segment among the others; a second layer of the same batch."""
    say("attend_train, captured without a gradient")
    segs, n = batch(gpu, LENGTHS, [{i: entry(gpu, 1 + i, 12) for i in range(2)}, None, None])
    g = torch.Generator().manual_seed(3)
    x = [torch.randn(h, n + 7, 64, generator=g).to(BF16).to(gpu) for h in (4, 2, 2, 4)]
    want = [train(*x, Batch(segs), layer)[0] for layer in range(2)]
    attend(*x[:3], segs, 0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        got = [attend_train(*x[:3], segs, layer) for layer in range(2)]
    for _ in range(3):
        for t in got:
            t.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        assert same(got, want)
        assert torch.equal(train(*x, segs, 1)[0], want[1])
    many_x, make = many(gpu, 9)
    segs = make()
    attend(*many_x[:3], segs, 0)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="before a capture"):  # (another layer's table would be uploaded)
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=torch.cuda.Stream()):
            attend_train(*many_x[:3], segs, 1)
    torch.cuda.synchronize()
    assert torch.equal(attend_train(*many_x[:3], segs, 1), train(*many_x, make(), 1)[0])


def test_a_captured_step_keeps_its_entries(gpu):
    """A call behind replaced entries leaves the tables alone that a captured step reads."""
    say("attend_train, captured behind entries that are replaced")
    segs, n = batch(gpu, LENGTHS, [{0: entry(gpu, 1, 12)}, None, {0: entry(gpu, 2, 12)}])
    g = torch.Generator().manual_seed(3)
    x = [torch.randn(h, n, 64, generator=g).to(BF16).to(gpu) for h in (4, 2, 2, 4)]
    want = train(*x, segs)
    leaves = [t.detach().requires_grad_() for t in x[:3]]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        out = attend_train(*leaves, segs, 0)
        got = [out.detach(), *torch.autograd.grad(out, leaves, x[3])]
    kept = segs[0].past[0]
    for i in range(3):
        segs[0].past[0] = entry(gpu, 10 + i, 12)
        other = train(*x, segs)
        assert not torch.equal(other[0], want[0])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert same(got, want)
    segs[0].past[0] = kept
    assert same(train(*x, segs), want)


@pytest.mark.parametrize("needs", [True, False])
def test_compiled_over_gaps_and_replaced_entries(gpu, needs):
    """torch.compile leaves the call to eager execution, with everything that it looks at on the host."""
    say("attend_train under torch.compile, eager backend", needs)
    segs, n = batch(gpu, LENGTHS, [{0: entry(gpu, 1, 12)}, None, {0: entry(gpu, 2, 12)}])
    g = torch.Generator().manual_seed(3)
    x = [torch.randn(h, n + 5, 64, generator=g).to(BF16).to(gpu) for h in (4, 2, 2, 4)]
    torch._dynamo.reset()
    f = torch.compile(lambda q, k, v: attend_train(q * 1, k * 1, v * 1, segs, 0) * 1, backend="eager")
    for seed in (1, 1, 7, 8):  # (the first call makes the batch's tables)
        segs[0].past[0] = entry(gpu, seed, 12)
        want = train(*x, Batch(segs))
        poison(want[0])
        leaves = [t.detach().requires_grad_(needs) for t in x[:3]]
        out = f(*leaves)
        assert torch.equal(out, want[0]) and (out[:, n:] == 0).all()
        if needs:
            assert same(torch.autograd.grad(out, leaves, x[3]), want[1:])
