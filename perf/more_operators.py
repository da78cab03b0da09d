"""The operators of adapter training and serving as measurable cases: their plain forms in
elementary torch operations, and the calls that a user makes of the framework's own.

Three operators, what a decoder layer runs where its own weights stay as they are and
adapters are trained beside them, or served:

- ``attend``: tree attention of packed reads with its gradient, the output and the gradients of
  q, k and v (``dan_amd.attention.attend_train``);
- ``adapt``: the low-rank adapters of many requests added to a shared projection's output
  (``dan_amd.adapters.adapt``), and with ``grad`` the gradients of the input and of the adapters too;
- ``norm``: the residual's addition and the root-mean-square norm in front of a projection, its
  result in 16 bits or in 8 bits with a scale for each row (``dan_amd.norm.add_norm``), and with
  ``grad`` the gradients of the addends and of the weight too.

``own`` selects: false, the plain forms (fp32 whatever the inputs' type, rounded once at
the end); true, the framework's calls. Values come from the seed given to ``prepare``, the
packing of the reads from the case's own ``shape``.
"""
import math
import random
from types import SimpleNamespace

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
LAYOUTS = ((32, 8, 128), (32, 8, 128), (16, 2, 256), (8, 2, 64), (32, 32, 128))  # q heads, kv heads, head_dim
LLAMA3_8B_LINEARS = ((6144, 4096), (4096, 4096), (28672, 4096), (4096, 14336))  # qkv, o, gate_up, down: (out, in)
E4M3_MAX = 448.0
BUDGET = 8192  # packed tokens of a full serving batch


def _heads(heads, kv_heads, head_dim):
    return dict(heads=heads, kv_heads=kv_heads, head_dim=head_dim)


def _tree(shape, tokens, requests, branches, length, past=0):
    return dict(shape=shape, tokens=tokens, requests=requests, fewest=branches[0], most=branches[1], shortest=length[0], longest=length[1],
                past=past)


def listed():
    return [
        # The smallest step: one short request with three questions, of a small model's heads.
        dict(name="attend_request", kind="attend", dtype="bf16", **_heads(8, 2, 64), **_tree(1, 55, 1, (3, 3), (1, 9))),
        # A few requests of mixed lengths in half precision.
        dict(name="attend_requests_fp16", kind="attend", dtype="fp16", **_heads(32, 8, 128), **_tree(2, 3413, 4, (3, 6), (16, 64))),
        # Hybrid models' gated layers (head_dim 256) behind a shared, cached prompt, which has no gradient.
        dict(name="attend_prefix_d256", kind="attend", dtype="bf16", **_heads(16, 2, 256), **_tree(3, 4099, 5, (3, 12), (16, 96), 1024)),
        # A training step of one long document with 32 questions, a full budget.
        dict(name="attend_document", kind="attend", dtype="bf16", **_heads(32, 8, 128), **_tree(5, BUDGET, 1, (32, 32), (16, 16))),
        # One user's next token: a single row beside the fused qkv projection, where latency counts.
        dict(name="adapt_token", kind="adapt", dtype="bf16", rows=1, n_in=4096, n_out=6144, rank=16, adapters=1, mixed=True, grad=False),
        # The next tokens of a batch whose requests have adapters of their own, or none.
        dict(name="adapt_batch", kind="adapt", dtype="bf16", rows=64, n_in=4096, n_out=4096, rank=16, adapters=24, mixed=True, grad=False),
        # The packed prompts of a full budget, each request with its adapter.
        dict(name="adapt_prompts", kind="adapt", dtype="bf16", rows=BUDGET, n_in=4096, n_out=6144, rank=16, adapters=7, mixed=False,
             grad=False),
        # Several adapters of high rank trained at once on packed requests, half precision.
        dict(name="adapt_train_fp16", kind="adapt", dtype="fp16", rows=1037, n_in=4096, n_out=4096, rank=64, adapters=5, mixed=False,
             grad=True),
        # A training step of a full budget beside the widest projection.
        dict(name="adapt_train_budget", kind="adapt", dtype="bf16", rows=BUDGET, n_in=4096, n_out=28672, rank=16, adapters=1, mixed=False,
             grad=True),
        # The next tokens of a few users, in 8 bits for the quantised projection behind.
        dict(name="norm_batch_e4m3", kind="norm", dtype="bf16", rows=7, cols=4096, norm="rms", codes=True, grad=False),
        # A full budget of prompts, in 8 bits.
        dict(name="norm_prompts_e4m3", kind="norm", dtype="bf16", rows=BUDGET, cols=4096, norm="rms", codes=True, grad=False),
        # A training step's norm of a hybrid model (zero-centered weights), half precision.
        dict(name="norm_train_fp16", kind="norm", dtype="fp16", rows=4099, cols=2048, norm="zero_centered", codes=False, grad=True),
    ]


def _log(rng, lo, hi):
    """An integer in [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    kind = rng.choice(("attend", "attend", "adapt", "adapt", "norm"))
    if kind == "norm":
        codes = rng.random() < 0.5
        return dict(kind=kind, dtype=dtype, rows=_log(rng, 1, BUDGET), cols=rng.choice((1024, 2048, 4096, 14336, 16 * rng.randint(4, 384))),
                    norm=rng.choice(("rms", "zero_centered")), codes=codes, grad=not codes and rng.random() < 0.6)
    if kind == "attend":
        h, hkv, d = rng.choice(LAYOUTS)
        tokens = _log(rng, 16, BUDGET)
        requests = rng.randint(1, 8) if tokens >= 512 else rng.randint(1, 2)
        most = rng.randint(0, 12)
        past = rng.choice((0, 0, _log(rng, 1, 1024))) if tokens <= 6144 else 0
        return dict(kind="attend", dtype=dtype, **_heads(h, hkv, d),
                    **_tree(rng.randrange(1 << 30), tokens, requests, (most // 2, most), (1, rng.choice((16, 96))), past))
    n_out, n_in = rng.choice(LLAMA3_8B_LINEARS + ((8 * rng.randint(8, 768), 8 * rng.randint(8, 768)),) * 3)
    grad = rng.random() < 0.5
    rows = _log(rng, 1, BUDGET)
    return dict(kind="adapt", dtype=dtype, rows=rows, n_in=n_in, n_out=n_out, rank=rng.choice((1, 4, 8, 16, 16, 24, 32, 64)),
                adapters=_log(rng, 1, 8 if grad or rows > 512 else 32), mixed=rng.random() < 0.5, grad=grad)


def _structure(case):
    """[(trunk, [branch lengths])] of the packed requests, ``tokens`` together."""
    r = random.Random(case["shape"])
    share = [r.uniform(0.4, 1.6) for _ in range(case["requests"])]
    cuts = [0]
    for s in share:
        cuts.append(cuts[-1] + s)
    cuts = [round(c / cuts[-1] * case["tokens"]) for c in cuts]
    out = []
    for a, b in zip(cuts, cuts[1:]):
        lens = []
        for _ in range(r.randint(case["fewest"], case["most"])):
            n = r.randint(case["shortest"], case["longest"])
            if sum(lens) + n < b - a:  # the trunk keeps a token
                lens.append(n)
        if b > a:
            out.append((b - a - sum(lens), lens))
    return out


def _spans(case):
    """(start, end, each row's branch: 0 for the trunk) of each request."""
    at = 0
    for trunk, lens in _structure(case):
        ids = [0] * trunk + [j for j, n in enumerate(lens, 1) for _ in range(n)]
        yield at, at + len(ids), ids
        at += len(ids)


# ------------------------------------------------------------------ inputs, from the seed alone


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def _prepare_attend(case, seed):
    g = _gen(seed)
    n, h, hkv, d = (case[f] for f in ("tokens", "heads", "kv_heads", "head_dim"))
    dt = DTYPES[case["dtype"]]
    # q, k, v as an attention layer hands them over: views of the fused projection's rows.
    rows = _randn(g, n, h + 2 * hkv, d, dtype=dt)
    q, k, v = (rows[:, a:b].transpose(0, 1).detach().requires_grad_() for a, b in ((0, h), (h, h + hkv), (h + hkv, h + 2 * hkv)))
    past = tuple(_randn(g, hkv, case["past"], d, dtype=dt) for _ in range(2)) if case["past"] else None
    s = dict(q=q, k=k, v=v, past=past, g=_randn(g, n, h, d, dtype=dt).transpose(0, 1), spans=list(_spans(case)))
    if own:
        from dan_amd.attention import Batch, segment

        s["segments"] = Batch(segment(a, ids, past and {0: past}, 0, case["past"], "cuda") for a, _, ids in s["spans"])
    return s


def _prepare_adapt(case, seed):
    g = _gen(seed)
    n, n_in, n_out, r, count = (case[f] for f in ("rows", "n_in", "n_out", "rank", "adapters"))
    dt = DTYPES[case["dtype"]]
    a, b = _randn(g, count, r, n_in, std=n_in ** -0.5, dtype=dt), _randn(g, count, n_out, r, std=0.1, dtype=dt)
    if case["mixed"]:  # a batch's rows in any order, about one in nine without an adapter
        index = torch.randint(0, count, (n,), generator=g, device="cuda")
        index[4::9] = -1
    else:  # packed requests, one after the other
        index = torch.arange(n, device="cuda") * count // n
    scale = torch.rand(count, generator=g, device="cuda") * 1.5 + 0.5
    s = dict(x=_randn(g, n, n_in, dtype=dt), y=_randn(g, n, n_out, dtype=dt), a=a, b=b, index=index.to(torch.int32), scale=scale)
    if case["grad"]:
        for f in ("x", "a", "b"):
            s[f].requires_grad_()
        s["g"] = _randn(g, n, n_out, dtype=dt)
    return s


def _prepare_norm(case, seed):
    g = _gen(seed)
    n, cols = case["rows"], case["cols"]
    dt = DTYPES[case["dtype"]]
    s = dict(x=_randn(g, n, cols, dtype=dt), stream=_randn(g, n, cols, std=3.0, dtype=dt), norm=case["norm"], codes=case["codes"],
             w=(_randn(g, cols, std=0.2) + (case["norm"] == "rms")).to(dt))
    if case["grad"]:
        for f in ("x", "stream", "w"):
            s[f].requires_grad_()
        s["g"], s["gs"] = _randn(g, n, cols, dtype=dt), _randn(g, n, cols, dtype=dt)
    return s


def prepare(case, seed):
    make = {"attend": _prepare_attend, "adapt": _prepare_adapt, "norm": _prepare_norm}[case["kind"]]
    return SimpleNamespace(kind=case["kind"], grad=case.get("grad", True), **make(case, seed))


# ------------------------------------------------------------------ the plain forms


def _hidden(ids, past, device):
    """[n, past + n]: the keys that a row does not see (later ones, and those of other branches)."""
    ids = torch.tensor(ids, device=device)
    at = torch.arange(len(ids), device=device)
    seen = (at[None] <= at[:, None]) & ((ids[None] == 0) | (ids[None] == ids[:, None]))
    return torch.cat((torch.zeros(len(ids), past, dtype=torch.bool, device=device), ~seen), 1)


def _t(x):
    return x.transpose(-1, -2).contiguous()


def _plain_attend(s):
    h, n, d = s.q.shape
    hkv = s.k.shape[0]
    scale = d ** -0.5
    q, k, v, g = (x.detach().float() for x in (s.q, s.k, s.v, s.g))
    out, dq, dk, dv = (torch.empty(n, x.shape[0], d, device=x.device).transpose(0, 1) for x in (q, q, k, v))
    for a, b, ids in s.spans:
        past = s.past[0].shape[1] if s.past else 0
        keys, values = (torch.cat((c.float(), x[:, a:b]), 1) if past else x[:, a:b].contiguous()
                        for c, x in zip(s.past or (None, None), (k, v)))
        qs, gs = (x[:, a:b].reshape(hkv, -1, d) for x in (q, g))  # the heads of a kv head, one after the other
        p = torch.matmul(qs, _t(keys)) * scale
        p.view(h, b - a, -1).masked_fill_(_hidden(ids, past, p.device), -math.inf)
        p = torch.exp(p - p.amax(-1, keepdim=True))
        p /= p.sum(-1, keepdim=True)
        out[:, a:b] = torch.matmul(p, values).view(h, b - a, d)
        dv[:, a:b] = torch.matmul(_t(p), gs)[:, past:]
        ds = torch.matmul(gs, _t(values))
        ds -= (ds * p).sum(-1, keepdim=True)
        ds *= p
        ds *= scale
        dq[:, a:b] = torch.matmul(ds, keys).view(h, b - a, d)
        dk[:, a:b] = torch.matmul(_t(ds), qs)[:, past:]
    return tuple(x.to(s.q.dtype) for x in (out, dq, dk, dv))


def _plain_adapt(s):
    """All adapters' products at once, each row keeping those of its own."""
    count, r, n_in = s.a.shape
    n, n_out = s.y.shape
    x, a, b = s.x.detach().float(), s.a.detach().float(), s.b.detach().float()
    mine = (s.index[:, None] == torch.arange(count, device=x.device)) * s.scale  # [N, R], scaled
    b_all = b.transpose(1, 2).reshape(count * r, n_out)
    h = (torch.matmul(x, _t(a.view(-1, n_in))).view(n, count, r) * mine[..., None]).view(n, -1)
    out = (s.y.float() + torch.matmul(h, b_all)).to(s.y.dtype)
    if not s.grad:
        return out
    g = s.g.float()
    dh = (torch.matmul(g, _t(b_all)).view(n, count, r) * mine[..., None]).view(n, -1)
    da, db = torch.matmul(_t(dh), x), torch.matmul(_t(h), g)
    return (out, torch.matmul(dh, a.view(-1, n_in)).to(s.x.dtype), da.view(s.a.shape).to(s.a.dtype),
            db.view(count, r, n_out).transpose(1, 2).to(s.b.dtype))


def _plain_norm(s, eps=1e-6):
    dt = s.x.dtype
    t = s.x.detach().float() + s.stream.detach().float()
    w = s.w.detach().float() + (s.norm == "zero_centered")
    r = torch.rsqrt(t.square().mean(1, keepdim=True) + eps)
    hat = t * r
    y = hat * w
    if s.codes:
        scale = y.abs().amax(1, keepdim=True).clamp(min=1e-12) / E4M3_MAX
        return t.to(dt), (y / scale).to(torch.float8_e4m3fn), scale
    if not s.grad:
        return t.to(dt), y.to(dt)
    g = s.g.float()
    dw = (g * hat).sum(0)
    g = g * w
    dt_ = r * (g - hat * (g * hat).mean(1, keepdim=True)) + s.gs.float()  # of both addends
    return t.to(dt), y.to(dt), dt_.to(dt), dw.to(dt)


# ------------------------------------------------------------------ one pass


def run(s):
    if not own:
        return {"attend": _plain_attend, "adapt": _plain_adapt, "norm": _plain_norm}[s.kind](s)
    if s.kind == "norm":
        from dan_amd.norm import add_norm

        r = add_norm(s.x, s.stream, s.w, norm=s.norm, fp8="rows" if s.codes else None)
        if s.codes:
            return r.stream, r.codes, r.scale
        if not s.grad:
            return r.stream, r.out
        dx, dw = torch.autograd.grad((r.out, r.stream), (s.x, s.w), (s.g, s.gs))
        return r.stream.detach(), r.out.detach(), dx, dw
    if s.kind == "attend":
        from dan_amd.attention import attend_train

        out = attend_train(s.q, s.k, s.v, s.segments, 0)
        return (out.detach(), *torch.autograd.grad(out, (s.q, s.k, s.v), s.g))
    from dan_amd.adapters import adapt

    out = adapt(s.y, s.x, s.a, s.b, s.index, s.scale)
    return (out.detach(), *torch.autograd.grad(out, (s.x, s.a, s.b), s.g)) if s.grad else out


# ------------------------------------------------------------------ what a pass cannot do without


def _pairs(case):
    """(query, key) pairs that see each other: among the packed rows, and with the prefix."""
    pairs = 0
    for trunk, lens in _structure(case):
        pairs += trunk * (trunk + 1) // 2 + sum(n * trunk + n * (n + 1) // 2 for n in lens)
    return pairs, case["tokens"] * case["past"]


def work(case):
    if case["kind"] == "attend":
        n, h, hkv, d = (case[f] for f in ("tokens", "heads", "kv_heads", "head_dim"))
        pairs, past = _pairs(case)
        # Forward: scores and output. Backward: scores again, the probabilities' gradient, dq, dk and dv (no dk, dv of a prefix).
        return {"bytes": 2 * d * (n * (4 * h + 4 * hkv) + 2 * hkv * case["past"]), "flops": 2 * d * h * (7 * pairs + 5 * past)}
    if case["kind"] == "norm":
        n, cols = case["rows"], case["cols"]
        if case["grad"]:  # the addends, the two gradients; the sum, the norm, the addends' gradient
            return {"bytes": 2 * cols * (7 * n + 2), "flops": 15 * n * cols}
        return {"bytes": 2 * cols * (3 * n + 1) + n * (cols + 4 if case["codes"] else 2 * cols), "flops": n * cols * (7 if case["codes"] else 5)}
    n, n_in, n_out, r = (case[f] for f in ("rows", "n_in", "n_out", "rank"))
    used = min(n, case["adapters"])
    rows = n - (len(range(4, n, 9)) if case["mixed"] else 0)
    weights = r * (n_in + n_out)
    if not case["grad"]:
        return {"bytes": 2 * (n * (n_in + 2 * n_out) + used * weights) + 4 * n, "flops": 2 * rows * weights}
    return {"bytes": 2 * (n * (2 * n_in + 3 * n_out) + (used + case["adapters"]) * weights) + 4 * n, "flops": 6 * rows * weights}


# ------------------------------------------------------------------ the definitions in 64 bits


def _exact_attend(s):
    h, n, d = s.q.shape
    rep = h // s.k.shape[0]
    out, dq = (torch.zeros(h, n, d, dtype=torch.float64, device="cuda") for _ in range(2))
    dk, dv = (torch.zeros(s.k.shape, dtype=torch.float64, device="cuda") for _ in range(2))
    for a, b, ids in s.spans:
        branch = torch.tensor(ids, device="cuda")
        seen = torch.tril((branch[None] == 0) | (branch[None] == branch[:, None]))
        p0 = s.past[0].shape[1] if s.past else 0
        for i in range(h):
            j = i // rep
            kk, vv = s.k[j, a:b].detach().double(), s.v[j, a:b].detach().double()
            if p0:
                kk, vv = torch.cat((s.past[0][j].double(), kk)), torch.cat((s.past[1][j].double(), vv))
            qq, gg = s.q[i, a:b].detach().double(), s.g[i, a:b].double()
            score = (qq @ kk.T) / math.sqrt(d)
            score[:, p0:][~seen] = -math.inf
            w = torch.softmax(score, 1)
            o = w @ vv
            out[i, a:b] = o
            e = w * (gg @ vv.T - (gg * o).sum(1, keepdim=True)) / math.sqrt(d)
            dq[i, a:b] = e @ kk
            dk[j, a:b] += (e.T @ qq)[p0:]
            dv[j, a:b] += (w.T @ gg)[p0:]
    return out, dq, dk, dv


def _exact_adapt(s):
    x, a, b = s.x.detach().double(), s.a.detach().double(), s.b.detach().double()
    out = s.y.double()
    if s.grad:
        g = s.g.double()
        dx, da, db = torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b)
    for i, c in enumerate(s.scale.double().tolist()):
        rows = torch.nonzero(s.index == i)[:, 0]
        down = x[rows] @ a[i].T
        out[rows] += c * (down @ b[i].T)
        if s.grad:
            up = c * (g[rows] @ b[i])
            dx[rows] = up @ a[i]
            da[i] = up.T @ x[rows]
            db[i] = c * (g[rows].T @ down)
    return (out, dx, da, db) if s.grad else out


def _exact_norm(s):
    t = s.x.detach().double() + s.stream.detach().double()
    w = s.w.detach().double()
    if s.norm == "zero_centered":
        w = 1.0 + w
    rms = torch.sqrt((t * t).sum(1) / t.shape[1] + 1e-6)[:, None]
    y = t / rms * w
    if s.codes:
        scale = torch.clip(y.abs().max(1, keepdim=True).values, min=1e-12) / E4M3_MAX
        return t, y / scale, scale
    if not s.grad:
        return t, y
    g = s.g.double()
    dt = g * w / rms - t * ((g * w * t).sum(1, keepdim=True) / (t.shape[1] * rms ** 3)) + s.gs.double()
    return t, y, dt, (g * t / rms).sum(0)


def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "adapt": _exact_adapt, "norm": _exact_norm}[s.kind](s)
