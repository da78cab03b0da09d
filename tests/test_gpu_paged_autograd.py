"""append_paged and attend_paged beside torch's autograd: caches that a graph has saved, inputs that require grad. Each through
the host module and through the Python functions alone."""
import pytest
import torch

from dan_amd import _decode
from dan_amd.paged import append_paged, attend_paged

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
H, HKV, D, PAGE = 4, 2, 64, 16


def say(msg):
    print(f"[gpu-case] {msg}", flush=True)


class _Rest:
    """Stands for the host module: makes no call, so that the Python functions make every one."""

    append = attend = logprobs = staticmethod(lambda *args: None)


@pytest.fixture(params=["host module", "python"])
def path(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(_decode, "calls", lambda: _Rest)
    return request.param


def inputs(gpu, n=2):
    q, k, v = (torch.ones(n, h, D, dtype=BF16, device=gpu) for h in (H, HKV, HKV))
    caches = [torch.zeros(3, HKV, PAGE, D, dtype=BF16, device=gpu) for _ in range(2)]
    table = torch.tensor([[0], [2]], dtype=torch.int32, device=gpu)
    places = torch.tensor([3, 0], dtype=torch.int32, device=gpu)
    return q, k, v, *caches, table, places


def append(q, k, v, kc, vc, table, places, **kw):
    kw.setdefault("norm", None)
    cos, sin = kw.pop("cos", None), kw.pop("sin", None)
    return append_paged(q, k, v, cos, sin, kc, vc, table, places, **kw)


@pytest.mark.parametrize("which", ["k", "v", "a view", "without q"])
def test_a_backward_that_saved_a_cache_raises_after_an_append(gpu, path, which):
    say(f"append: a saved cache, {which}, {path}")
    q, k, v, kc, vc, table, places = inputs(gpu)
    leaf = torch.ones(D, device=gpu, dtype=BF16, requires_grad=True)
    saved = {"k": kc, "v": vc, "a view": kc[1], "without q": vc}[which]
    loss = (saved * leaf).sum()
    versions = kc._version, vc._version
    append(None if which == "without q" else q, k, v, kc, vc, table, places)
    assert kc._version > versions[0] and vc._version > versions[1]
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()


def test_no_rows_and_reads_leave_the_versions(gpu, path):
    say(f"append: no rows, {path}")
    q, k, v, kc, vc, table, places = inputs(gpu)
    append(q[:0], k[:0], v[:0], kc, vc, table, places[:0])
    attend_paged(q.transpose(0, 1), kc, vc, table, places)
    assert kc._version == vc._version == 0


def test_inference_tensors_are_written(gpu, path):
    say(f"append: inference tensors, {path}")
    with torch.inference_mode():
        q, k, v, kc, vc, table, places = inputs(gpu)
        append(q, k, v, kc, vc, table, places)
        torch.cuda.synchronize()
        assert kc.is_inference() and (kc == 1).sum() == 2 * HKV * D
    q, k, v, kc, vc, table, places = inputs(gpu)
    with torch.inference_mode():
        append(q, k, v, kc, vc, table, places)  # caches made outside
    assert kc._version == 1 and (vc == 1).sum() == 2 * HKV * D
