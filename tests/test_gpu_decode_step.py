"""The decode step's operators together: append_paged, attend_paged, token_logprobs, as a serving loop calls
them token by token, captured into a graph and replayed, and on another stream."""
import math

import pytest
import torch

from dan_amd.paged import append_paged, attend_paged
from dan_amd.readout import token_logprobs
from oracle import paged as OP
from oracle import readout as OR

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
H, HKV, D, PAGE, VOCAB = 8, 2, 128, 16, 1003


def say(msg):
    print(f"[gpu-case] {msg}", flush=True)


class Layer:
    """Random weights of one attention layer and a head, and a cache of `seqs` sequences of up to `most` tokens."""

    def __init__(self, gpu, seqs, most, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.gpu, self.seqs = gpu, seqs
        width = -(-most // PAGE)
        self.table = torch.randperm(seqs * width, generator=g).int().view(seqs, width).to(gpu)
        self.kc, self.vc = (torch.full((seqs * width, HKV, PAGE, D), math.nan, dtype=BF16, device=gpu) for _ in range(2))
        inv = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
        angle = torch.cat((torch.arange(most)[:, None] * inv,) * 2, 1)
        self.cos, self.sin = angle.cos().float().to(gpu), angle.sin().float().to(gpu)
        self.wq, self.wk = ((torch.randn(D, generator=g) * 0.2 + 1).to(BF16).to(gpu) for _ in range(2))
        self.head = (torch.randn(VOCAB, H * D, generator=g) * 0.2).to(BF16).to(gpu)

    def step(self, qkv, places, lens, tokens, seqs=None):
        n = qkv.shape[0]
        q, k, v = qkv.view(n, H + 2 * HKV, D).split([H, HKV, HKV], 1)
        q = append_paged(q, k, v, self.cos, self.sin, self.kc, self.vc, self.table, places, seqs=seqs, rope_rows=places,
                         q_norm_weight=self.wq, k_norm_weight=self.wk)
        if seqs is not None:
            return q
        o = attend_paged(q, self.kc, self.vc, self.table, lens)
        logits = o.transpose(0, 1).reshape(n, H * D) @ self.head.t()
        return (o, logits) + tuple(token_logprobs(logits, tokens, top=5, entropy=True))


def ids(x, gpu):
    return torch.tensor(x, dtype=torch.int32, device=gpu)


def test_decode_loop_matches_the_oracle(gpu):
    """Three prompts of unequal length, then six tokens of each. The cache's own rows (rounded, as any cache holds
    them) feed the oracle, so each step's output is within one rounding (2^-8) and its weights' fp32 error, far below that."""
    say("decode loop: prompts, then six steps")
    lens = [19, 1, 40]
    m = Layer(gpu, 3, 64)
    g = torch.Generator().manual_seed(7)
    rows = sum(lens)
    prompt = torch.randn(rows, (H + 2 * HKV) * D, generator=g).to(BF16).to(gpu)
    m.step(prompt, ids([t for n in lens for t in range(n)], gpu), None, None, seqs=ids([s for s, n in enumerate(lens) for _ in range(n)], gpu))
    for step in range(6):
        qkv = torch.randn(3, (H + 2 * HKV) * D, generator=g).to(BF16).to(gpu)
        tokens = torch.randint(0, VOCAB, (3, 2), generator=g)
        places = [n + step for n in lens]
        now = [p + 1 for p in places]
        o, logits, lp, lse, ent, tlp, tid = m.step(qkv, ids(places, gpu), ids(now, gpu), tokens.to(gpu))
        torch.cuda.synchronize()
        x = qkv.cpu().view(3, H + 2 * HKV, D)
        c, s = m.cos.cpu()[places], m.sin.cpu()[places]
        q = OP.rotate_norm(x[:, :H], m.wq.cpu(), "rms", c, s)
        k = OP.rotate_norm(x[:, H:H + HKV], m.wk.cpu(), "rms", c, s)
        table = m.table.cpu()
        for i, p in enumerate(places):
            row = m.kc.cpu()[int(table[i, p // PAGE]), :, p % PAGE].double()
            assert ((row - k[i]).abs() <= k[i].abs() * 2.0 ** -8 + 2.0 ** -18 * 16).all()
            assert torch.equal(m.vc.cpu()[int(table[i, p // PAGE]), :, p % PAGE], x[i, H + HKV:])
        ref, _, mag, big = OP.attend(q.to(BF16).transpose(0, 1), m.kc.cpu().double().nan_to_num(), m.vc.cpu().double().nan_to_num(), table, now)
        # q's own rounding may fall the other way where its fp32 value lies next to a border: 2^-8 of it, in every score
        tol = 2.0 ** -8 * ref.abs() + (2.0 ** -14 + 2 * 2.0 ** -7 * 2.0 ** -6 * big[..., None] / math.sqrt(D)) * mag
        assert ((o.cpu().double() - ref).abs() <= tol).all()
        rlp, rlse, rent, rtlp, rid = OR.token_logprobs(logits.cpu(), tokens, 5)
        assert torch.equal(tid.cpu(), rid)
        for got, want in ((lp, rlp), (lse, rlse), (ent, rent), (tlp, rtlp)):
            assert (got.cpu().double() - want).abs().max() < 2.0 ** -14


def test_captured_step_replays_with_changing_lengths(gpu):
    """One captured step serves every later one: places, lengths, values and tokens change between replays, a row turns
    idle, and eager work runs in between. Two graphs share nothing: the second is replayed between the first's replays."""
    say("decode step: two graphs, replayed in turn")
    places, lens, tokens = ids([300, 5, 77], gpu), ids([301, 6, 78], gpu), torch.zeros(3, 2, dtype=torch.long, device=gpu)
    qkv = torch.zeros(3, (H + 2 * HKV) * D, dtype=BF16, device=gpu)
    g = torch.Generator().manual_seed(3)
    layers = [Layer(gpu, 3, 512, seed=s) for s in (1, 2)]
    for m in layers:
        m.kc.normal_()
        m.vc.normal_()
    copies = [(m.kc.clone(), m.vc.clone()) for m in layers]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for m in layers:
            m.step(qkv, places, lens, tokens)
    torch.cuda.current_stream().wait_stream(side)
    for m in layers:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(m.step(qkv, places, lens, tokens))
        graphs.append(graph)
    for m, (kc, vc) in zip(layers, copies):
        m.kc.copy_(kc)
        m.vc.copy_(vc)
    for step in range(4):
        at = [300 + 13 * step, 5 + step, 77 + step]
        n = [p + 1 for p in at]
        if step == 2:
            at[1], n[1] = -1, 0  # idle
        places.copy_(ids(at, gpu))
        lens.copy_(ids(n, gpu))
        qkv.copy_(torch.randn(qkv.shape, generator=g).to(BF16))
        tokens.copy_(torch.randint(-1, VOCAB, tokens.shape, generator=g))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in o] + [m.kc.clone(), m.vc.clone()] for o, m in zip(outs, layers)]
        for m, have in zip(layers, got):
            want = list(m.step(qkv, places, lens, tokens)) + [m.kc, m.vc]  # writes the same rows again
            torch.cuda.synchronize()
            assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(have, want))
            if step == 2:
                assert (have[0][:, 1] == 0).all()


def test_another_stream(gpu):
    """Everything on a stream of its own, tensors made on it; the default stream works meanwhile."""
    say("decode step: another stream")
    m = Layer(gpu, 2, 256)
    m.kc.normal_()
    m.vc.normal_()
    g = torch.Generator().manual_seed(4)
    qkv = torch.randn(2, (H + 2 * HKV) * D, generator=g).to(BF16).to(gpu)
    tokens = torch.tensor([3, 4], device=gpu)
    want = [t.clone() for t in m.step(qkv, ids([200, 9], gpu), ids([201, 10], gpu), tokens)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(side):
            got = m.step(qkv, ids([200, 9], gpu), ids([201, 10], gpu), tokens)
        noise = torch.randn(1 << 20, device=gpu).sum()
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.isfinite(noise)


def test_gradient_replays(gpu):
    """Forward and backward of the readout in one captured graph, replayed on changed logits."""
    say("readout: captured gradient")
    x = torch.randn(5, 777, device=gpu, requires_grad=True)
    t = torch.randint(0, 777, (5,), device=gpu)
    w = torch.randn(5, device=gpu)

    def grad():
        r = token_logprobs(x, t, entropy=True)
        return torch.autograd.grad([r.logprobs, r.entropy], x, [w, w])[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grad()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = grad()
    for _ in range(3):
        with torch.no_grad():
            x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        have = out.clone()
        assert torch.equal(have, grad())


class _Rest:
    """Stands for the host module: makes no call, so that the Python functions make every one."""

    append = attend = logprobs = staticmethod(lambda *args: None)


def test_both_host_paths_make_the_same_calls(gpu, monkeypatch):
    """Plain calls go through the host module, all others through Python: here the same calls through either."""
    say("decode step: host module and Python")
    from dan_amd import _decode

    g = torch.Generator().manual_seed(5)
    qkv = torch.randn(3, (H + 2 * HKV) * D, generator=g).to(BF16).to(gpu)
    tokens = torch.randint(-1, VOCAB, (3, 2), generator=g).to(gpu)
    x = torch.randn(4, VOCAB, generator=g).to(gpu).requires_grad_()

    def run():
        m = Layer(gpu, 3, 700, seed=3)
        m.kc.zero_()
        m.vc.zero_()
        out = list(m.step(qkv, ids([650, 0, -1], gpu), ids([651, 1, 0], gpu), tokens)) + [m.kc, m.vc]
        cache8 = m.kc.to(torch.float8_e4m3fn)
        scale = torch.full((1,), 0.5, device=gpu)
        out += attend_paged(out[0], cache8, cache8, m.table, ids([651, 1, 0], gpu), 0.1, k_scale=scale, v_scale=scale, max_len=660, return_lse=True)
        r = token_logprobs(x, torch.arange(4, device=gpu), top=3, entropy=True)
        out += list(r) + [torch.autograd.grad([r.logprobs, r.logsumexp, r.entropy, r.top_logprobs], x, [torch.ones_like(t) for t in (r.logprobs, r.logsumexp, r.entropy, r.top_logprobs)])[0]]
        torch.cuda.synchronize()
        return out

    made = []
    real = _decode.calls()

    class Watch:
        append, attend, logprobs = (staticmethod(lambda *a, f=f: made.append(f(*a)) or made[-1]) for f in (real.append, real.attend, real.logprobs))

    monkeypatch.setattr(_decode, "calls", lambda: Watch)
    first = run()
    assert len(made) == 5 and all(m is not None for m in made)
    monkeypatch.setattr(_decode, "calls", lambda: _Rest)
    for a, b in zip(first, run(), strict=True):
        assert a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride() and torch.equal(a, b)


def test_what_is_not_plain_is_left_to_python(gpu):
    """The host module makes no call on other types, layouts, sizes, or where a gradient or tangent is to be refused."""
    say("host module: calls it leaves")
    from dan_amd import _decode

    c = _decode.calls()
    m = Layer(gpu, 2, 64)
    q, k = torch.zeros(2, H, D, dtype=BF16, device=gpu), torch.zeros(2, HKV, D, dtype=BF16, device=gpu)
    places, lens, norm = ids([0, 1], gpu), ids([1, 2], gpu), 0
    a = lambda **w: c.append(*{**dict(q=q, k=k, v=k, cos=None, sin=None, kc=m.kc, vc=m.vc, t=m.table, p=places, s=None, r=None, qw=None, kw=None, e=1e-6,
                                      n=norm, ks=None, vs=None), **w}.values())
    t = lambda **w: c.attend(*{**dict(q=q.transpose(0, 1), kc=m.kc, vc=m.vc, t=m.table, l=lens, s=None, ks=None, vs=None, m=None, r=False), **w}.values())
    x, tok = torch.zeros(2, 50, device=gpu), torch.zeros(2, dtype=torch.long, device=gpu)
    r = lambda **w: c.logprobs(*{**dict(x=x, t=tok, top=1, e=False), **w}.values())
    assert a() is not None and t() is not None and r() is not None
    odd = torch.zeros(2 * HKV * D + 1, dtype=BF16, device=gpu)[1:].view(2, HKV, D)
    dual = torch.autograd.forward_ad
    for w in (dict(q=None), dict(k=odd), dict(q=q.cpu()), dict(k=k.clone().requires_grad_()), dict(p=places.long()), dict(n=1), dict(n=-1), dict(n=3),
              dict(t=m.table.t()), dict(kc=m.kc[:, :, :, :64]), dict(kc=m.kc[:1].expand(m.kc.shape)), dict(ks=x[:1, 0]), dict(cos=x), dict(sin=x), dict(e=1),
              dict(q=5), dict(s=places[:1]), dict(vc=m.vc.half()), dict(p=m.table[:, 0].cpu())):
        assert a(**w) is None, w
    for w in (dict(q=q), dict(m=10 ** 30), dict(m=-1), dict(m=65), dict(s=0.0), dict(s=math.nan), dict(s=1), dict(l=lens.long()), dict(q=q.float().transpose(0, 1)),
              dict(q=q.transpose(0, 1)[:7]), dict(t=m.table[:1]), dict(kc=None), dict(q=q.transpose(0, 1).clone().requires_grad_())):
        assert t(**w) is None, w
    for w in (dict(top=33), dict(top=-1), dict(top=10 ** 30), dict(t=tok.int()), dict(x=x.double()), dict(x=x.t()[:, :0]), dict(x=x[0]), dict(t=None), dict(top=None), dict(x=x.cpu())):
        assert r(**w) is None, w
    with dual.dual_level():
        assert r(x=dual.make_dual(x, x)) is None and t(q=dual.make_dual(q, q).transpose(0, 1)) is None
    assert c.append() is None and c.attend(1) is None and c.logprobs() is None


def test_without_keys_no_table_is_read(gpu):
    """max_len 0 needs no cache and no table, whatever width is given for one."""
    say("attend: no table")
    from dan_amd import _decode

    q, lens = torch.ones(2, H, D, dtype=BF16, device=gpu), ids([0, 1], gpu)
    out, lse = torch.ones_like(q), torch.ones(2, H, device=gpu)
    fields = dict(abi_version=_decode.PAGED_ABI_VERSION, num_seqs=2, num_heads=H, num_kv_heads=HKV, head_dim=D, page_size=16, num_pages=4, table_width=4,
                  scale=1.0, q=q.data_ptr(), q_stride_seq=H * D, q_stride_head=D, out=out.data_ptr(), o_stride_seq=H * D, o_stride_head=D,
                  lse=lse.data_ptr(), kc_stride_tok=D, vc_stride_tok=D, table_stride=4, lens=lens.data_ptr())
    _decode.call_paged_attn(torch.cuda.current_stream().cuda_stream, *(fields.get(n, 0) for n, _ in _decode.DanPagedAttnArgs._fields_))
    torch.cuda.synchronize()
    assert not out[0].any() and (lse[0] == -math.inf).all() and out[1].isnan().all() and lse[1].isnan().all()


def test_inference_mode_and_two_threads(gpu):
    """The same step from two threads at once, each on a stream of its own, in inference mode."""
    say("decode step: two threads in inference mode")
    import threading

    g = torch.Generator().manual_seed(6)
    qkv = torch.randn(2, (H + 2 * HKV) * D, generator=g).to(BF16).to(gpu)
    tokens = torch.tensor([3, 4], device=gpu)
    got, wrong = {}, []

    def run(i):
        try:
            with torch.inference_mode(), torch.cuda.stream(torch.cuda.Stream()):
                m = Layer(gpu, 2, 256, seed=2)
                m.kc.fill_(0.25)
                m.vc.fill_(0.5)
                for _ in range(20):
                    out = m.step(qkv, ids([200, 9], gpu), ids([201, 10], gpu), tokens)
                torch.cuda.current_stream().synchronize()
                got[i] = [t.clone() for t in out]
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # shown by the test's own thread
            wrong.append(e)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and all(torch.equal(a, b) and a.is_inference() for a, b in zip(got[0], got[1], strict=True))


def test_compiled_step(gpu):
    """A compiled function that calls the operators gives what the plain one does."""
    say("decode step: torch.compile")
    m = Layer(gpu, 2, 256, seed=2)
    m.kc.fill_(0.25)
    m.vc.fill_(0.5)
    qkv = torch.randn(2, (H + 2 * HKV) * D, generator=torch.Generator().manual_seed(6)).to(BF16).to(gpu)
    args = qkv, ids([200, 9], gpu), ids([201, 10], gpu), torch.tensor([3, 4], device=gpu)
    with torch.no_grad():
        want = m.step(*args)
        got = torch.compile(m.step, backend="eager")(*args)
    assert all(torch.equal(a, b) for a, b in zip(got, want, strict=True))


def test_an_appended_copy_on_write_cache_leaves_its_source(gpu):
    say("append: copy on write")
    m = Layer(gpu, 2, 64)
    m.kc.zero_()
    m.vc.zero_()
    kc, vc = m.kc, m.vc
    m.kc, m.vc = torch._lazy_clone(kc), torch._lazy_clone(vc)
    qkv = torch.ones(2, (H + 2 * HKV) * D, dtype=BF16, device=gpu)
    m.step(qkv, ids([0, 1], gpu), ids([1, 2], gpu), torch.tensor([3, 4], device=gpu))
    assert not kc.any() and not vc.any() and m.kc.any() and (m.vc == 1).sum() == 2 * HKV * D


@pytest.mark.parametrize("tokens", [torch.int64, torch.int32])
def test_a_capture_that_an_eager_graph_would_join_is_refused(gpu, tokens):
    """While an eager result holds the graph of a leaf, a captured backward to the same leaf raises, and both go on."""
    say(f"readout: captured gradient beside an eager graph, {tokens}")
    x = torch.randn(4, 300, device=gpu, requires_grad=True)
    t = torch.tensor([1, 2, 3, -1], device=gpu, dtype=tokens)

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
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
