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


def test_every_input_that_wants_a_derivative_is_refused(gpu, path):
    """Both are forward-only: no input loses its gradient or tangent without a word, the norm's weights, tables and scales among them. Without grad
    mode, and where the call does not use them, they pass."""
    say(f"paged: inputs that require grad, {path}")
    q, k, v, kc, vc, table, places = inputs(gpu)
    one, cs = torch.ones(D, dtype=BF16, device=gpu), torch.ones(2, D, device=gpu)
    e4m3, scale = torch.zeros(3, HKV, PAGE, D, device=gpu).to(torch.float8_e4m3fn), torch.ones(1, device=gpu)
    plain = dict(q=q, k=k, v=v, kc=kc, vc=vc, table=table, places=places, norm="rms", q_norm_weight=one, k_norm_weight=one, cos=cs, sin=cs)
    coded = dict(plain, kc=e4m3, vc=e4m3.clone(), k_scale=scale, v_scale=scale)
    dual = torch.autograd.forward_ad
    for base, names in ((plain, ("q", "k", "v", "kc", "vc", "q_norm_weight", "k_norm_weight", "cos", "sin")), (coded, ("k_scale", "v_scale"))):
        append(**base)
        for name in names:
            wants = dict(base, **{name: base[name].clone().requires_grad_()})
            with pytest.raises(NotImplementedError):
                append(**wants)
            with torch.no_grad():
                append(**wants)
            with dual.dual_level(), pytest.raises(NotImplementedError):
                append(**dict(base, **{name: dual.make_dual(base[name], torch.ones_like(base[name]))}))
    append(**dict(plain, norm=None, q_norm_weight=one.clone().requires_grad_()))  # not used
    heads, lens = q.transpose(0, 1), torch.tensor([1, 1], dtype=torch.int32, device=gpu)
    for cache, scales in ((kc, {}), (e4m3, dict(k_scale=scale, v_scale=scale))):
        attend_paged(heads, cache, cache, table, lens, **scales)
        for name in scales:
            with pytest.raises(NotImplementedError):
                attend_paged(heads, cache, cache, table, lens, **dict(scales, **{name: scale.clone().requires_grad_()}))
            with dual.dual_level(), pytest.raises(NotImplementedError):
                attend_paged(heads, cache, cache, table, lens, **dict(scales, **{name: dual.make_dual(scale, scale)}))
