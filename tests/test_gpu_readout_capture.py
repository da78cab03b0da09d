"""token_logprobs' backward inside a stream capture, where its calls go on in Python (no host module): the same refusal and the same replays."""
import pytest
import torch

from dan_amd import _decode
from dan_amd.readout import token_logprobs

pytestmark = pytest.mark.gpu


class _Rest:
    """Stands for the host module: makes no call, so that the Python functions make every one."""

    append = attend = logprobs = staticmethod(lambda *args: None)


def test_a_capture_that_an_eager_graph_would_join_is_refused_in_python_too(gpu, monkeypatch):
    print("[gpu-case] readout: captured gradient beside an eager graph, through Python", flush=True)
    monkeypatch.setattr(_decode, "calls", lambda: _Rest)
    x = torch.randn(4, 300, device=gpu, requires_grad=True)
    t = torch.tensor([1, 2, 3, -1], device=gpu)

    def grad(r):
        return torch.autograd.grad(r.logprobs, x, torch.ones_like(r.logprobs), retain_graph=True)[0]

    side = torch.cuda.Stream()
    eager = token_logprobs(x, t)  # alive, with its graph
    want = grad(eager)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured backward"):
        with torch.cuda.graph(graph, stream=side):
            grad(token_logprobs(x, t))
    torch.cuda.synchronize()
    assert torch.equal(grad(eager), want)
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = grad(token_logprobs(x, t))
    for _ in range(3):
        with torch.no_grad():
            x.add_(0.25)
        graph.replay()
        torch.cuda.synchronize()
        have = got.clone()
        assert torch.equal(have, grad(token_logprobs(x, t)))
