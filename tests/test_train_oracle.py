"""The oracle of what adapters are trained and served with, against torch's autograd in fp64 and against differences.

fp64: sums of some hundred terms near 1 agree to 1e-12; a central difference of step 1e-4 is off by the third
derivative's 1e-8 / 6 and by 1e-16 / 1e-4 of values of some hundreds: 1e-6 covers both."""
import math

import pytest
import torch

from dan_amd import workloads
from dan_amd.attention import Batch, segment
from oracle import training as oracle

F64 = torch.float64


def randn(g, *shape):
    return torch.randn(*shape, generator=g, dtype=F64)


def near(a, b, tol=1e-12):
    assert a.shape == b.shape and (a - b).abs().max().item() <= tol * max(1.0, b.abs().max().item())


def differences(f, x, grad, tol=1e-6, count=12):
    """The gradient of f at x against central differences along its first coordinates in a fixed, mixed order."""
    flat = x.flatten()
    for i in torch.randperm(flat.numel(), generator=torch.Generator().manual_seed(5))[:count].tolist():
        at = flat[i].item()
        flat[i] = at + 1e-4
        up = f()
        flat[i] = at - 1e-4
        down = f()
        flat[i] = at
        assert abs((up - down).item() / 2e-4 - grad.flatten()[i].item()) <= tol * max(1.0, grad.abs().max().item())


def tree(past):
    g = torch.Generator().manual_seed(3)
    segs, at = Batch(), 0
    for i, (t, ls) in enumerate([(5, [3, 1]), (0, [2, 4]), (3, [])]):
        ids = workloads.branch_ids(t, ls)
        entry = {0: (randn(g, 2, past, 8), randn(g, 2, past, 8))} if past and i != 1 else None
        segs.append(segment(at, ids, entry, 0, past if entry else 0, "cpu"))
        at += len(ids)
    return segs, at, g


@pytest.mark.parametrize("past", [0, 4])
def test_attend(past):
    segs, n, g = tree(past)
    q, k, v, grad = randn(g, 4, n, 8), randn(g, 2, n, 8), randn(g, 2, n, 8), randn(g, 4, n, 8)
    ref = oracle.attend(q, k, v, segs, 0, grad=grad)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    out = torch.zeros(4, n, 8, dtype=F64)
    for s in segs:
        m = s.end - s.start
        kk, vv = (x[:, s.start:s.end].repeat_interleave(2, 0) for x in leaves[1:])
        see = torch.zeros(m, m, dtype=torch.bool)
        see[:, :s.trunk] = True
        for a, b in s.branches:
            see[a - s.start:b - s.start, a - s.start:b - s.start] = True
        see &= torch.ones(m, m, dtype=torch.bool).tril()
        if s.past:
            pk, pv = (x.repeat_interleave(2, 0) for x in s.past[0])
            kk, vv, see = torch.cat((pk, kk), 1), torch.cat((pv, vv), 1), torch.cat((torch.ones(m, past, dtype=torch.bool), see), 1)
        x = (leaves[0][:, s.start:s.end] @ kk.transpose(1, 2) / math.sqrt(8)).masked_fill(~see, -math.inf)
        near(ref["lse"][:, s.start:s.end], x.detach().logsumexp(2))
        out = out.index_copy(1, torch.arange(s.start, s.end), x.softmax(2) @ vv)
    near(ref["out"], out.detach())
    for name, x in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, grad)):
        near(ref[name], x)
    for name, x in (("dq", q), ("dk", k), ("dv", v)):
        differences(lambda: (oracle.attend(q, k, v, segs, 0)["out"] * grad).sum(), x, ref[name])


def test_adapt():
    g = torch.Generator().manual_seed(4)
    y, x, a, b, grad = randn(g, 7, 6), randn(g, 7, 5), randn(g, 3, 2, 5), randn(g, 3, 6, 2), randn(g, 7, 6)
    index, scale = [0, 2, -1, 2, 0, -4, 2], torch.tensor([0.5, 2.0, -1.5])
    ref = oracle.adapt(y, x, a, b, index, scale, grad)
    leaves = [t.clone().requires_grad_() for t in (x, a, b)]
    out = torch.stack([y[n] + (0 if i < 0 else scale[i].double() * (leaves[2][i] @ (leaves[1][i] @ leaves[0][n]))) for n, i in enumerate(index)])
    near(ref["out"], out.detach())
    for name, d in zip(("dx", "da", "db"), torch.autograd.grad(out, leaves, grad, allow_unused=True)):
        near(ref[name], d)
    for name, t in (("dx", x), ("da", a), ("db", b)):
        differences(lambda: (oracle.adapt(y, x, a, b, index, scale)["out"] * grad).sum(), t, ref[name])
    far = oracle.adapt(y, x, a, b, [0, 3, 1, 9, 0, 0, 0], scale, grad)
    assert far["out"][1].isnan().all() and far["out"][3].isnan().all() and far["out"][[0, 2, 4, 5, 6]].isfinite().all()
    assert far["dx"][1].isnan().all() and far["dx"][3].isnan().all() and far["dx"][[0, 2]].isfinite().all() and far["da"].isfinite().all()


@pytest.mark.parametrize("norm", ["rms", "zero_centered"])
@pytest.mark.parametrize("residual", [True, False])
def test_add_norm(norm, residual):
    g = torch.Generator().manual_seed(5)
    x, r, w, go, gs = randn(g, 4, 6), randn(g, 4, 6), randn(g, 6), randn(g, 4, 6), randn(g, 4, 6)
    ref = oracle.add_norm(x, r if residual else None, w, norm=norm, grad=go, grad_stream=gs)
    leaves = [t.clone().requires_grad_() for t in (x, w)]
    s = leaves[0] + r if residual else leaves[0] * 1
    out = torch.nn.functional.rms_norm(s, (6,), leaves[1] + (norm == "zero_centered"), 1e-6)
    near(ref["stream"], s.detach())
    near(ref["out"], out.detach())
    for name, d in zip(("ds", "dw"), torch.autograd.grad((out, s), leaves, (go, gs))):
        near(ref[name], d)

    def loss():
        o = oracle.add_norm(x, r if residual else None, w, norm=norm)
        return (o["out"] * go).sum() + (o["stream"] * gs).sum()

    differences(loss, x, ref["ds"])
    differences(loss, w, ref["dw"])
