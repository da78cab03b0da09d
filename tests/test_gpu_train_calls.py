"""add_norm, adapt and attend_train as a user's program calls them: layouts in memory, frozen inputs, streams, captured
graphs, what a second derivative and a changed input raise, and repeated runs.

Results are compared bit for bit where the same kernels run on the same values, and with the fp64 oracle elsewhere
(test_gpu_norm, test_gpu_adapt and test_gpu_attend_train derive the tolerances)."""
import threading

import pytest
import torch
import torch.utils.checkpoint

import test_gpu_adapt
import test_gpu_attend_train
import test_gpu_norm
from dan_amd import _layer
from dan_amd.adapters import adapt
from dan_amd.attention import attend, attend_train
from dan_amd.norm import add_norm
from oracle import training as oracle

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
TREE = [(40, [5, 9, 1]), (0, [3, 4]), (70, [33, 2])]


def say(*a):
    print("[gpu-case]", *a, flush=True)


class Case:
    """One operator with its inputs: ``call(*leaves)`` gives the outputs of which ``grads`` are the gradients."""

    def __init__(self, name, gpu, dtype=BF16):
        self.name, self.dtype = name, dtype
        if name == "norm":
            x, r, w = test_gpu_norm.make(gpu, 37, 264, dtype)
            g = torch.Generator().manual_seed(2)
            self.leaves = [x, r, w]
            self.grads = [torch.randn(37, 264, generator=g).to(dtype).to(gpu) for _ in range(2)]
        elif name == "adapt":
            y, x, a, b, index, scale, grad = test_gpu_adapt.make(gpu, 45, 136, 200, 24, 5, dtype)
            self.leaves, self.index, self.scale, self.grads = [y, x, a, b], index, scale, [grad]
        else:
            q, k, v, grad, self.segs = test_gpu_attend_train.make(gpu, TREE, 4, 2, 64, dtype, pasts=[12, 0, 0])
            self.leaves, self.grads = [q, k, v], [grad]

    def call(self, *leaves):
        if self.name == "norm":
            r = add_norm(*leaves)
            return [r.out, r.stream]
        if self.name == "adapt":
            return [adapt(*leaves, self.index, self.scale)]
        return [attend_train(*leaves, self.segs, 0)]

    def fresh(self, needs=None):
        return [x.detach().clone(memory_format=torch.preserve_format).requires_grad_(needs is None or i in needs) for i, x in enumerate(self.leaves)]

    def run(self, leaves=None, grads=None):
        leaves = self.fresh() if leaves is None else leaves
        out = self.call(*leaves)
        return [x.detach() for x in out] + list(torch.autograd.grad(out, [x for x in leaves if x.requires_grad], grads or self.grads))


class _Rest:
    """Stands for the host module: makes no call, so that the Python functions make every one."""

    add_norm = adapt = attend = staticmethod(lambda *args: None)


NAMES = ["norm", "adapt", "attend"]


@pytest.fixture
def way(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(_layer, "calls", lambda: _Rest)
    return request.param


ways = pytest.mark.parametrize("way", ["module", "python"], indirect=True)


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b, strict=True))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("name", NAMES)
def test_both_ways_and_repeated_runs_give_the_same_bits(gpu, name, dtype, monkeypatch):
    say(name, dtype, "repeated, and through Python")
    c = Case(name, gpu, dtype)
    want = c.run()
    assert all(x.isfinite().all() for x in want)
    for _ in range(3):
        assert same(c.run(), want)
    monkeypatch.setattr(_layer, "calls", lambda: _Rest)
    assert same(c.run(), want)


@ways
@pytest.mark.parametrize("name", NAMES)
def test_without_gradients_the_output_is_the_same(gpu, name, way):
    say(name, way, "under no_grad, and with inputs that need no gradient")
    c = Case(name, gpu)
    want = [x.detach() for x in c.call(*c.fresh())]
    with torch.no_grad():
        assert same(c.call(*c.fresh()), want)
    got = c.call(*c.leaves)
    assert same(got, want) and not any(x.requires_grad for x in got)


def test_attend_train_is_attend_bit_for_bit_and_saves_as_it_does(gpu):
    say("attend_train beside attend, with saves")
    for dtype in (BF16, FP16):
        c = Case("attend", gpu, dtype)
        q, k, v = c.leaves
        for s in c.segs:
            s.save = min(7, s.trunk)
        want = attend(q, k, v, c.segs, 0)
        saved = [s.saved[0] for s in c.segs if s.save]
        for s in c.segs:
            s.saved = {}
        leaves = c.fresh()
        out = attend_train(*leaves, c.segs, 0)
        assert torch.equal(out, want) and out.requires_grad
        for (a, b), s in zip(saved, [s for s in c.segs if s.save], strict=True):
            k2, v2 = s.saved[0]
            assert torch.equal(a, k2) and torch.equal(b, v2) and not k2.requires_grad
            assert k2.untyped_storage().data_ptr() != leaves[1].untyped_storage().data_ptr()


LAYOUTS = {
    "wide": lambda x: torch.nn.functional.pad(x, (0, 24))[..., :-24],  # rows of a larger tensor
    "shifted": lambda x: torch.nn.functional.pad(x, (3, 5))[..., 3:-5],  # not 16-byte aligned
    "odd": lambda x: torch.nn.functional.pad(x, (0, 1))[..., :-1],  # rows of odd strides
    "turned": lambda x: x.transpose(-1, -2).contiguous().transpose(-1, -2),  # no unit stride
    "dense": lambda x: x.contiguous().clone(),
}


@ways
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("name", NAMES)
def test_layouts_in_memory(gpu, name, layout, way):
    say(name, way, layout)
    c = Case(name, gpu)
    want = c.run()
    leaves = [(LAYOUTS[layout](x) if x.dim() > 1 else x).detach().requires_grad_() for x in c.leaves]
    grads = [LAYOUTS[layout](x) for x in c.grads]
    assert same(c.run(leaves, grads), want)


@ways
@pytest.mark.parametrize("name", NAMES)
def test_an_expanded_gradient(gpu, name, way):
    say(name, way, "gradient of a sum")
    c = Case(name, gpu)
    leaves = c.fresh()
    out = c.call(*leaves)
    got = torch.autograd.grad(sum(x.sum() for x in out), leaves)
    assert same(got, c.run(grads=[torch.ones_like(x) for x in out])[len(out):])


@ways
@pytest.mark.parametrize("name", NAMES)
def test_frozen_inputs(gpu, name, way):
    say(name, way, "one input at a time needs a gradient")
    c = Case(name, gpu)
    want = c.run()
    count = len(c.leaves)
    for i in range(count):
        out = c.call(*(leaves := c.fresh({i})))
        got = torch.autograd.grad(out[0], leaves[i], c.grads[0], retain_graph=True)[0]
        if len(out) == 1:
            assert torch.equal(got, want[len(out) + i])
        for j in range(count):
            assert j == i or leaves[j].grad is None


@ways
@pytest.mark.parametrize("part", [0, 1])
def test_one_of_the_norms_outputs_alone(gpu, part, way):
    say("norm", way, "gradient of", ("out", "stream")[part], "alone")
    c = Case("norm", gpu)
    leaves = c.fresh()
    out = c.call(*leaves)
    got = torch.autograd.grad(out[part], leaves[:2] if part else leaves, c.grads[part])
    if part:
        assert torch.equal(got[0], c.grads[1]) and torch.equal(got[1], c.grads[1])
    else:
        ref = oracle.add_norm(*c.leaves, grad=c.grads[0])
        u = torch.finfo(c.dtype).eps / 2
        test_gpu_norm.close("ds", got[0], ref["ds"], (3 * u + 2 ** -17) * ref["abs_ds"] + torch.finfo(c.dtype).tiny)
        assert torch.equal(got[0], got[1])


@ways
@pytest.mark.parametrize("name", NAMES)
def test_a_second_derivative_raises(gpu, name, way):
    say(name, way, "second derivative")
    c = Case(name, gpu)
    leaves = c.fresh()
    d = torch.autograd.grad(c.call(*leaves)[0], leaves[-1], c.grads[0], create_graph=True)[0]
    with pytest.raises(RuntimeError, match="once"):
        d.float().sum().backward()


@ways
@pytest.mark.parametrize("name", NAMES)
def test_an_input_changed_in_place_raises(gpu, name, way):
    say(name, way, "changed in place")
    c = Case(name, gpu)
    leaves = c.fresh()
    out = c.call(*leaves)[0]
    with torch.no_grad():
        leaves[-1].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward(c.grads[0])


@ways
def test_a_prefix_entry_changed_in_place_raises(gpu, way):
    say("attend", way, "prefix changed in place")
    c = Case("attend", gpu)
    out = c.call(*c.fresh())[0]
    c.segs[0].past[0][1].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward(c.grads[0])


@ways
@pytest.mark.parametrize("name", NAMES)
def test_a_graph_that_was_used_raises(gpu, name, way):
    say(name, way, "backward twice")
    c = Case(name, gpu)
    out = c.call(*c.fresh())[0]
    out.backward(c.grads[0])
    with pytest.raises(RuntimeError, match="second time"):
        out.backward(c.grads[0])


@ways
@pytest.mark.parametrize("name", NAMES)
def test_on_another_stream(gpu, name, way):
    say(name, way, "on another stream, behind slow work")
    c = Case(name, gpu)
    want = c.run()
    side = torch.cuda.Stream()
    big = torch.randn(4096, 4096, device=gpu)
    leaves = [torch.zeros_like(x).requires_grad_() for x in c.leaves]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(4):
            big = big @ big * 1e-2
        with torch.no_grad():
            for x, y in zip(leaves, c.leaves):
                x.copy_(y)
        got = c.run(leaves)
    side.synchronize()
    assert same(got, want)


@ways
@pytest.mark.parametrize("name", NAMES)
def test_a_captured_step_replays(gpu, name, way):
    say(name, way, "captured forward and backward")
    c = Case(name, gpu)
    c.run()  # (tables are uploaded before the capture)
    leaves = c.fresh()
    grads = [x.clone() for x in c.grads]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = c.run(leaves, grads)
    gen = torch.Generator(device=gpu).manual_seed(1)
    for i in range(3):
        with torch.no_grad():
            for x in leaves + grads:
                x.copy_(torch.randn(x.shape, device=gpu, generator=gen).to(x.dtype))
        graph.replay()
        torch.cuda.synchronize()
        have = [x.clone() for x in got]
        want = c.run([x.detach().requires_grad_() for x in leaves], grads)
        torch.cuda.synchronize()
        assert same(have, want), i


@ways
@pytest.mark.parametrize("name", NAMES)
def test_a_capture_that_an_eager_graph_would_join_is_refused(gpu, name, way):
    say(name, way, "captured backward beside an eager graph of the same leaves")
    c = Case(name, gpu)
    want = c.run()
    leaves = c.fresh()
    eager = c.call(*leaves)  # alive, with its graph
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured backward"):
        with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
            torch.autograd.grad(c.call(*leaves), leaves, c.grads)
    torch.cuda.synchronize()
    assert same(torch.autograd.grad(eager, leaves, c.grads), want[len(eager):])


def test_a_batchs_first_call_in_a_capture_is_refused(gpu):
    say("attend: first call of a batch in a capture")
    warm = Case("attend", gpu)
    warm.run()
    c = Case("attend", gpu)
    leaves = c.fresh()
    attend(*c.leaves, c.segs, 0)  # (the plan is there, the backward pass's tables are not)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before a capture"):
        with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
            c.call(*leaves)
    torch.cuda.synchronize()
    assert same(c.run(), warm.run())


def test_two_calls_before_either_backward(gpu):
    """Two results alive at once, of different sizes, backward in the other order: nothing is shared between calls."""
    for name in NAMES:
        say(name, "two calls, backward in the other order")
        c = Case(name, gpu)
        want = c.run()
        first, second = c.fresh(), [x.detach().mul(0.5).requires_grad_() for x in c.leaves]
        a, b = c.call(*first), c.call(*second)
        other = torch.autograd.grad(b, second, c.grads)
        assert same(torch.autograd.grad(a, first, c.grads), want[len(a):])
        assert same(other, c.run(second)[len(a):])


@ways
def test_the_same_leaf_twice(gpu, way):
    """k as v, and x as its own residual: autograd adds the two gradients up."""
    say("attend and norm", way, "the same leaf as two inputs")
    c = Case("attend", gpu)
    q, k, _ = c.leaves
    k = k.detach().requires_grad_()
    got = torch.autograd.grad(attend_train(q, k, k, c.segs, 0), k, c.grads[0])[0]
    two = [k.detach().requires_grad_() for _ in range(2)]
    dk, dv = torch.autograd.grad(attend_train(q, *two, c.segs, 0), two, c.grads[0])
    assert torch.equal(got, dk + dv)
    n = Case("norm", gpu)
    x = n.leaves[0].detach().requires_grad_()
    w = n.leaves[2]
    got = torch.autograd.grad(add_norm(x, x, w).out, x, n.grads[0])[0]
    two = [x.detach().requires_grad_() for _ in range(2)]
    da, db = torch.autograd.grad(add_norm(*two, w).out, two, n.grads[0])
    assert torch.equal(got, da + db)


def test_compiled_functions_break_the_graph_and_agree(gpu):
    """torch.compile leaves the calls to eager execution (no fake kernels are registered for them)."""
    for name in NAMES:
        say(name, "under torch.compile, eager backend")
        c = Case(name, gpu)
        want = c.run()
        torch._dynamo.reset()
        f = torch.compile(lambda *xs: [x * 1 for x in c.call(*xs)], backend="eager")
        leaves = c.fresh()
        out = f(*leaves)
        got = [x.detach() for x in out] + list(torch.autograd.grad(out, leaves, c.grads))
        assert same(got, want)


@ways
@pytest.mark.parametrize("name", NAMES)
def test_a_kept_graph_twice(gpu, name, way):
    say(name, way, "backward twice through a kept graph")
    c = Case(name, gpu)
    want = c.run()
    leaves = c.fresh()
    out = c.call(*leaves)
    for _ in range(2):
        assert same(torch.autograd.grad(out, leaves, c.grads, retain_graph=True), want[len(out):])


@ways
@pytest.mark.parametrize("name", NAMES)
def test_saved_tensors_that_leave_the_gpu(gpu, name, way):
    """What a call saves passes through torch's hooks: kept on the CPU, and made again by a checkpoint."""
    say(name, way, "saved on the CPU, and checkpointed")
    c = Case(name, gpu)
    want = c.run()
    leaves = c.fresh()
    with torch.autograd.graph.save_on_cpu():
        out = c.call(*leaves)
    assert same(torch.autograd.grad(out, leaves, c.grads), want[len(out):])
    for reentrant in (False, True):
        leaves = c.fresh()
        out = torch.utils.checkpoint.checkpoint(lambda *xs: tuple(c.call(*xs)), *leaves, use_reentrant=reentrant)
        torch.autograd.backward(out, c.grads)
        assert same([x.grad for x in leaves], want[len(out):])


@ways
def test_a_list_of_segments(gpu, way):
    say("attend", way, "a plain list instead of a Batch")
    c = Case("attend", gpu)
    want = c.run()
    c.segs = list(c.segs)
    for _ in range(2):
        assert same(c.run(), want)


@pytest.mark.parametrize("name", NAMES)
def test_two_threads_on_two_streams(gpu, name):
    """Two programs in one process: each thread its own inputs and stream; the batch (its tables) is shared."""
    say(name, "two threads")
    c = Case(name, gpu)
    want = [c.run(), c.run([x.detach().mul(0.5).requires_grad_() for x in c.leaves])]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    got = c.run([x.detach().mul(0.5 if i else 1.0).requires_grad_() for x in c.leaves])
                    torch.cuda.current_stream().synchronize()
                    if not same(got, want[i]):
                        bad.append(i)
        except Exception as e:  # noqa: BLE001  -- (shown by the assertion below)
            bad.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, bad


def derivative(call, oracle_call, leaves, grads, weights, dtype, step):
    """The kernel's directional derivative by differences against its gradient: what the outputs' rounding can move
    the difference by, and what the difference itself is off by (taken from the oracle), both computed."""
    at = [x.detach().double() for x in leaves]
    along = [d.double() / d.double().norm() for d in grads]
    moved = [[(x + s * step * u).to(dtype) for x, u in zip(at, along)] for s in (1, -1)]
    real = [(a.double() - b.double()) for a, b in zip(*moved)]  # the step as it is, rounded
    f = [sum((o.double() * w.double()).sum().item() for o, w in zip(call(*m), weights)) for m in moved]
    f64 = [sum((o * w.double().cpu()).sum().item() for o, w in zip(oracle_call(*m), weights)) for m in moved]
    outs = call(*moved[0])
    u = torch.finfo(dtype).eps / 2
    noise = 2 * 4 * u * sum((o.double() * w.double()).abs().sum().item() for o, w in zip(outs, weights))
    got = sum((g.double() * r).sum().item() for g, r in zip(grads, real))
    truncation = abs(f64[0] - f64[1] - got)
    say(f"  difference {f[0] - f[1]:.5g}, gradient {got:.5g}, oracle's difference {f64[0] - f64[1]:.5g}, rounding {noise:.3g}")
    assert abs(f[0] - f[1] - got) <= noise + truncation
    assert truncation <= 0.05 * abs(got) and noise <= 0.25 * abs(got)  # (or it would say nothing)


@pytest.mark.parametrize("name", NAMES)
def test_gradients_against_differences(gpu, name):
    say(name, "against differences")
    c = Case(name, gpu, FP16)
    # (a few outputs: fewer roundings beside the same change of each)
    weights = [g * (torch.arange(g.numel(), device=gpu).reshape(g.shape) % 97 == 0) if i == 0 else torch.zeros_like(g) for i, g in enumerate(c.grads)]
    leaves = c.fresh()
    grads = torch.autograd.grad(c.call(*leaves), leaves, weights)

    def reference(*xs):
        if name == "norm":
            r = oracle.add_norm(*xs)
            return [r["out"], r["stream"]]
        if name == "adapt":
            return [oracle.adapt(*xs, c.index.tolist(), c.scale)["out"]]
        return [oracle.attend(*xs, c.segs, 0)["out"]]

    derivative(c.call, reference, c.leaves, grads, weights, FP16, {"norm": 1.0, "adapt": 1.0, "attend": 2.0}[name])
