"""The operators of a decode step as measurable cases: their plain forms in elementary
torch operations, and the calls that a user makes of the framework's own.

Three operators, used one after the other for every new token:

- ``append``: the q/k norm and rotation of new tokens, q returned, k and v written into a
  paged cache (``dan_amd.paged.append_paged``);
- ``attend``: one new token of each sequence over that cache (``dan_amd.paged.attend_paged``);
- ``logprobs``: log probabilities of given tokens with the logsumexp, the entropy and the top
  alternatives (``dan_amd.readout.token_logprobs``), and with ``grad`` the gradient of the logits too.

``own`` selects: false, the plain forms (fp32 whatever the inputs' type, rounded once at
the end); true, the framework's calls. Values come from the seed given to ``prepare``,
structures (sequence lengths, the order of pages) from it, too, within the case's sizes.
"""
import math
from types import SimpleNamespace

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1}
E4M3_MAX = 448.0


def _heads(heads, kv_heads, head_dim):
    return dict(heads=heads, kv_heads=kv_heads, head_dim=head_dim)


def listed():
    return [
        # The smallest call: the one new token of a single user's sequence.
        dict(name="append_token", kind="append", dtype="bf16", cache="bf16", tokens=1, seqs=1, page=16, norm="none",
             rotary=128, gated=False, padded=False, decode=True, **_heads(32, 8, 128)),
        # A decode batch of the hybrid models' gated layers (partial rotary) on an e4m3 cache, padded to a fixed size.
        dict(name="append_batch_e4m3", kind="append", dtype="bf16", cache="e4m3", tokens=237, seqs=237, page=64,
             norm="zero_centered", rotary=64, gated=True, padded=True, decode=True, **_heads(16, 2, 256)),
        # The prompts of a full serving budget written into the cache.
        dict(name="append_prompts", kind="append", dtype="bf16", cache="bf16", tokens=8192, seqs=7, page=16, norm="rms",
             rotary=128, gated=False, padded=False, decode=False, **_heads(32, 8, 128)),
        # One user's next token behind a short prompt: latency counts.
        dict(name="attend_short", kind="attend", dtype="bf16", cache="bf16", seqs=1, longest=277, page=16, idle=False,
             **_heads(32, 8, 128)),
        # A serving batch of 64 sequences of mixed lengths.
        dict(name="attend_batch", kind="attend", dtype="bf16", cache="bf16", seqs=64, longest=8192, page=16, idle=False,
             **_heads(32, 8, 128)),
        # One long document: few rows, the work split over the length.
        dict(name="attend_document", kind="attend", dtype="bf16", cache="bf16", seqs=1, longest=131072, page=64, idle=False,
             **_heads(32, 8, 128)),
        # The hybrid models' layout (head_dim 256) on an e4m3 cache, some rows of the batch idle.
        dict(name="attend_batch_e4m3", kind="attend", dtype="bf16", cache="e4m3", seqs=37, longest=4099, page=32, idle=True,
             **_heads(16, 2, 256)),
        # As many kv heads as q heads, many short sequences.
        dict(name="attend_mha_fp16", kind="attend", dtype="fp16", cache="fp16", seqs=100, longest=1000, page=16, idle=False,
             **_heads(32, 32, 128)),
        # The next token of one sequence with its 20 best alternatives.
        dict(name="logprobs_token", kind="logprobs", dtype="bf16", rows=1, vocab=128256, labels=1, top=20, entropy=True,
             masked=False, grad=False),
        # Decision reads: each row's label tokens, under a grammar mask, at an odd vocabulary in fp32.
        dict(name="logprobs_labels_fp32", kind="logprobs", dtype="fp32", rows=45, vocab=50257, labels=12, top=5, entropy=False,
             masked=True, grad=False),
        # Scoring a prompt: every token's log probability, entropy and best alternatives.
        dict(name="logprobs_prompt", kind="logprobs", dtype="bf16", rows=2039, vocab=128256, labels=1, top=5, entropy=True,
             masked=False, grad=False),
        # A training step's loss: log probabilities and entropies of a batch, and the logits' gradient.
        dict(name="logprobs_train", kind="logprobs", dtype="bf16", rows=4096, vocab=128256, labels=1, top=0, entropy=True,
             masked=False, grad=True),
    ]


def _log(rng, lo, hi):
    """An integer in [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("append", "attend", "attend", "logprobs", "logprobs"))
    h, hkv, d = rng.choice(((32, 8, 128), (32, 8, 128), (16, 2, 256), (8, 2, 64), (32, 32, 128), (14, 2, 128)))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    cache = rng.choice((dtype, dtype, "e4m3"))
    page = rng.choice((16, 16, 32, 64, 128))
    if kind == "append":
        decode = rng.random() < 0.4
        tokens = _log(rng, 1, 512 if decode else 8192)
        return dict(kind=kind, dtype=dtype, cache=cache, tokens=tokens, seqs=tokens if decode else rng.randint(1, min(tokens, 16)),
                    page=page, norm=rng.choice(("none", "rms", "zero_centered")), rotary=rng.choice((d, d, d // 2, d // 4)),
                    gated=rng.random() < 0.3, padded=rng.random() < 0.3, decode=decode, **_heads(h, hkv, d))
    if kind == "attend":
        longest = _log(rng, 1, 131072 if hkv <= 8 else 16384)
        most = (1 << 29) // (2 * longest * hkv * d * BYTES[cache])
        return dict(kind=kind, dtype=dtype, cache=cache, seqs=_log(rng, 1, max(1, min(256, most))), longest=longest, page=page,
                    idle=rng.random() < 0.3, **_heads(h, hkv, d))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    grad = rng.random() < 0.4
    vocab = rng.choice((128256, 151936, 50257, _log(rng, 500, 262144)))
    return dict(kind=kind, dtype=dtype, rows=_log(rng, 1, max(2, min(4096, (1 << 29) // (vocab * BYTES[dtype] * (1 + grad))))),
                vocab=vocab, labels=rng.choice((1, 1, rng.randint(2, 24))), top=rng.choice((0, 1, 5, 20)),
                entropy=rng.random() < 0.6, masked=not grad and rng.random() < 0.3, grad=grad)


# ------------------------------------------------------------------ inputs, from the seed alone


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def _lengths(g, case):
    """The sequences' lengths: one of the longest, the others even up to it; a fifth of an idle batch is empty."""
    n = torch.randint(1, case["longest"] + 1, (case["seqs"],), generator=g, device="cuda")
    n[0] = case["longest"]
    if case["idle"] and case["seqs"] > 1:
        n[1::5] = 0
    return n


def _pages(g, lengths, page, width, pages=None):
    """A page table [sequences, width] of pages in random order (-1 where a sequence has none) and the cache's
    pages: a few more than the sequences need, if not given."""
    need = (lengths + page - 1) // page
    pages = pages or int(need.sum()) + 3
    first = need.cumsum(0) - need
    at = torch.arange(width, device="cuda")
    order = torch.randperm(pages, generator=g, device="cuda")
    table = torch.where(at < need[:, None], order[(first[:, None] + at).clamp(max=pages - 1)], -1)
    return table.to(torch.int32), pages


def _cache(g, case, pages):
    shape = (pages, case["kv_heads"], case["page"], case["head_dim"])
    ks = vs = None
    k, v = _randn(g, *shape), _randn(g, *shape)
    if case["cache"] == "e4m3":
        ks, vs = (torch.full((1,), s / E4M3_MAX, device="cuda") for s in (6.5, 6.0))
        k, v = (k / ks).clamp(-E4M3_MAX, E4M3_MAX), (v / vs).clamp(-E4M3_MAX, E4M3_MAX)
    dt = DTYPES[case["cache"]]
    return k.to(dt), v.to(dt), ks, vs


def _prepare_append(case, seed):
    g = _gen(seed)
    n, h, hkv, d, r, page = (case[f] for f in ("tokens", "heads", "kv_heads", "head_dim", "rotary", "page"))
    dt = DTYPES[case["dtype"]]
    # The fused projection's rows: q (with its gate behind each head, where it has one), then k, then v.
    qd = h * d * (2 if case["gated"] else 1)
    rows = _randn(g, n, qd + 2 * hkv * d, dtype=dt)
    q, k, v = rows[:, :qd].reshape(n, h, -1)[..., :d], rows[:, qd:qd + hkv * d].view(n, hkv, d), rows[:, qd + hkv * d:].view(n, hkv, d)
    if case["decode"]:  # each sequence's next token
        longest = 256
        seqs, places = None, torch.randint(0, longest, (n,), generator=g, device="cuda")
        lengths = places + 1
    else:  # whole prompts, one after the other
        longest = -(-n // case["seqs"])
        seqs = torch.arange(n, device="cuda") // longest
        places = torch.arange(n, device="cuda") % longest
        lengths = torch.bincount(seqs, minlength=case["seqs"])
    width = -(-longest // page)
    table, pages = _pages(g, lengths, page, width, case["seqs"] * width)
    # Rotary tables of the tokens, as a model makes them once for its layers (angles in 64 bits).
    inv = 500000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64, device="cuda") / r)
    angle = torch.cat((places.double()[:, None] * inv,) * 2, 1)
    if case["padded"]:  # rows without a token
        places[n // 2::7] = -1
    w = None if case["norm"] == "none" else [_randn(g, d, std=0.2, dtype=dt) + (case["norm"] == "rms") for _ in range(2)]
    kc, vc, ks, vs = _cache(g, case, pages)
    return dict(q=q, k=k, v=v, cos=angle.cos().to(dt), sin=angle.sin().to(dt), places=places.to(torch.int32), table=table,
                seqs=None if seqs is None else seqs.to(torch.int32), kc=kc, vc=vc, ks=ks, vs=vs,
                norm=None if case["norm"] == "none" else case["norm"], qw=w and w[0], kw=w and w[1], page=page)


def _prepare_attend(case, seed):
    g = _gen(seed)
    lengths = _lengths(g, case)
    table, pages = _pages(g, lengths, case["page"], -(-case["longest"] // case["page"]))
    kc, vc, ks, vs = _cache(g, case, pages)
    q = _randn(g, case["seqs"], case["heads"], case["head_dim"], std=1.5, dtype=DTYPES[case["dtype"]]).transpose(0, 1)
    return dict(q=q, kc=kc, vc=vc, ks=ks, vs=vs, table=table, lens=lengths.to(torch.int32), longest=case["longest"])


def _prepare_logprobs(case, seed):
    g = _gen(seed)
    n, vocab, labels = case["rows"], case["vocab"], case["labels"]
    x = _randn(g, n, vocab, std=2.5, dtype=DTYPES[case["dtype"]])
    tokens = torch.randint(0, vocab, (n, labels), generator=g, device="cuda")
    if labels > 1:  # lists of unequal length
        tokens[torch.arange(labels, device="cuda") >= torch.randint(1, labels + 1, (n, 1), generator=g, device="cuda")] = -1
    if case["masked"]:  # every other row allows one token in 50 (its labels among them)
        allowed = torch.rand(n, vocab, generator=g, device="cuda") < 0.02
        allowed[::2] = True
        allowed.scatter_(1, tokens.clamp(min=0), True)
        x.masked_fill_(~allowed, -math.inf)
    s = dict(tokens=tokens[:, 0].contiguous() if labels == 1 else tokens, top=case["top"], entropy=case["entropy"])
    if case["grad"]:
        x.requires_grad_()
        s["g"] = _randn(g, *s["tokens"].shape)
        s["ge"] = _randn(g, n, std=0.1) if case["entropy"] else None
        s["gt"] = _randn(g, n, case["top"]) if case["top"] else None
    return dict(x=x, **s)


def prepare(case, seed):
    make = {"append": _prepare_append, "attend": _prepare_attend, "logprobs": _prepare_logprobs}[case["kind"]]
    return SimpleNamespace(kind=case["kind"], grad=case.get("grad", False), **make(case, seed))


# ------------------------------------------------------------------ the plain forms


def _plain_norm_rope(x, weight, norm, cos, sin, eps=1e-6):
    """fp32 [N, heads, D] of a head row's norm and rotation."""
    x = x.float()
    if norm is not None:
        w = weight.float()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * (w if norm == "rms" else 1 + w)
    r = cos.shape[1]
    a, b = x[..., :r // 2], x[..., r // 2:r]
    c, s = cos.float()[:, None], sin.float()[:, None]
    return torch.cat((x[..., :r] * c + torch.cat((-b, a), -1) * s, x[..., r:]), -1)


def _plain_store(cache, x, scale, page, slot):
    """x [N, Hkv, D] into the cache's rows."""
    if scale is not None:
        x = (x / scale).clamp(-E4M3_MAX, E4M3_MAX)
    x = x.to(cache.dtype)
    if scale is not None:  # 8-bit values move as bytes
        cache, x = cache.view(torch.uint8), x.view(torch.uint8)
    cache[page, :, slot] = x


def _plain_append(s):
    q = _plain_norm_rope(s.q, s.qw, s.norm, s.cos, s.sin).to(s.q.dtype)
    k = _plain_norm_rope(s.k, s.kw, s.norm, s.cos, s.sin)
    token = torch.nonzero(s.places >= 0)[:, 0]
    place = s.places[token].long()
    page = s.table[token if s.seqs is None else s.seqs[token].long(), place // s.page].long()
    _plain_store(s.kc, k[token], s.ks, page, place % s.page)
    _plain_store(s.vc, s.v[token].float(), s.vs, page, place % s.page)
    return q.transpose(0, 1)


def _plain_rows(cache, scale, table):
    """The sequences' rows [B, Hkv, width * page, D] in fp32."""
    b, width = table.shape
    x = cache.view(torch.uint8)[table.clamp(min=0).long()].view(cache.dtype) if scale is not None else cache[table.clamp(min=0).long()]
    _, _, hkv, page, d = x.shape
    x = x.permute(0, 2, 1, 3, 4).reshape(b, hkv, width * page, d).float()
    return x if scale is None else x * scale


def _plain_attend(s):
    h, b, d = s.q.shape
    hkv = s.kc.shape[1]
    q = s.q.transpose(0, 1).reshape(b, hkv, h // hkv, d).float()
    k, v = _plain_rows(s.kc, s.ks, s.table), _plain_rows(s.vc, s.vs, s.table)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) * d ** -0.5
    hidden = torch.arange(k.shape[2], device=q.device) >= s.lens[:, None]
    score = score.masked_fill(hidden[:, None, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30))
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return o.reshape(b, h, d).to(s.q.dtype).transpose(0, 1)


def _plain_top(x, top):
    """The ``top`` largest of each row, ties to the lowest index: keys of the value's order, then the index."""
    bits = (x + 0.0).view(torch.int32).long()
    key = (torch.where(bits < 0, -2147483648 - bits, bits) << 20) - torch.arange(x.shape[1], device=x.device)
    at = torch.topk(key, top, dim=1, sorted=True).indices
    return x.gather(1, at), at


def _plain_logprobs(s):
    tokens = s.tokens if s.tokens.dim() == 2 else s.tokens[:, None]
    x = s.x.detach().float()
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(1, keepdim=True)
    lse = m + torch.log(z)
    given = tokens >= 0
    at = tokens.clamp(min=0)
    out = dict(logprobs=torch.where(given, x.gather(1, at) - lse, 0.0).reshape(s.tokens.shape), logsumexp=lse[:, 0])
    if s.entropy:
        entropy = torch.log(z) - (e * (x - m).clamp(min=-1e30)).sum(1, keepdim=True) / z
        out["entropy"] = entropy[:, 0]
    if s.top:
        value, out["top_ids"] = _plain_top(x, s.top)
        out["top_logprobs"] = value - lse
    if s.grad:
        p = e / z
        g = torch.where(given, s.g.reshape(tokens.shape), 0.0)
        grad = p * -(g.sum(1, keepdim=True) + (s.gt.sum(1, keepdim=True) if s.top else 0))
        if s.entropy:
            grad -= s.ge[:, None] * p * (x - lse + entropy)
        grad.scatter_add_(1, at, g)
        if s.top:
            grad.scatter_add_(1, out["top_ids"], s.gt)
        out["grad"] = grad.to(s.x.dtype)
    return out


# ------------------------------------------------------------------ one pass


def _own_logprobs(s):
    from dan_amd.readout import token_logprobs

    r = token_logprobs(s.x, s.tokens, top=s.top, entropy=s.entropy)
    out = dict(logprobs=r.logprobs, logsumexp=r.logsumexp)
    if s.entropy:
        out["entropy"] = r.entropy
    if s.top:
        out["top_ids"], out["top_logprobs"] = r.top_ids, r.top_logprobs
    if s.grad:
        parts = [(r.logprobs, s.g), (r.entropy, s.ge), (r.top_logprobs, s.gt)]
        parts = [p for p in parts if p[1] is not None]
        out["grad"] = torch.autograd.grad([p[0] for p in parts], s.x, [p[1] for p in parts])[0]
        out = {f: t.detach() for f, t in out.items()}
    return out


def run(s):
    if s.kind == "append":
        if own:
            from dan_amd.paged import append_paged

            q = append_paged(s.q, s.k, s.v, s.cos, s.sin, s.kc, s.vc, s.table, s.places, seqs=s.seqs, q_norm_weight=s.qw,
                             k_norm_weight=s.kw, norm=s.norm, k_scale=s.ks, v_scale=s.vs)
        else:
            q = _plain_append(s)
        return q, s.kc, s.vc
    if s.kind == "attend":
        if own:
            from dan_amd.paged import attend_paged

            return attend_paged(s.q, s.kc, s.vc, s.table, s.lens, k_scale=s.ks, v_scale=s.vs, max_len=s.longest)
        return _plain_attend(s)
    return _own_logprobs(s) if own else _plain_logprobs(s)


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    if case["kind"] == "append":
        n, h, hkv, d, r = (case[f] for f in ("tokens", "heads", "kv_heads", "head_dim", "rotary"))
        es, ec = BYTES[case["dtype"]], BYTES[case["cache"]]
        stored = n - (len(range(n // 2, n, 7)) if case["padded"] else 0)
        return {"bytes": n * ((2 * h + hkv) * d + 2 * r) * es + stored * hkv * d * (es + 2 * ec),
                "flops": n * (h + hkv) * (3 * r + (0 if case["norm"] == "none" else 4 * d))}
    if case["kind"] == "attend":
        b, h, hkv, d = (case[f] for f in ("seqs", "heads", "kv_heads", "head_dim"))
        idle = len(range(1, b, 5)) if case["idle"] and b > 1 else 0
        keys = case["longest"] + (b - 1 - idle) * (case["longest"] + 1) / 2
        return {"bytes": 2 * keys * hkv * d * BYTES[case["cache"]] + 2 * b * h * d * BYTES[case["dtype"]],
                "flops": 4 * keys * h * d}
    n, vocab = case["rows"], case["vocab"]
    moved = n * vocab * BYTES[case["dtype"]]
    out = n * (12 * case["labels"] + 4 + 4 * case["entropy"] + 12 * case["top"])
    return {"bytes": moved * (2 if case["grad"] else 1) + out, "flops": n * vocab * (4 + 2 * case["entropy"]) * (2 if case["grad"] else 1)}


# ------------------------------------------------------------------ the definitions in 64 bits


def _exact_head(x, w, norm, cos, sin):
    """[heads, D] of one token's rows, from the definition."""
    x = x.double()
    if norm is not None:
        gain = w.double() + (1.0 if norm == "zero_centered" else 0.0)
        x = gain * x / torch.sqrt((x * x).sum(2, keepdim=True) / x.shape[2] + 1e-6)
    r = cos.shape[1]
    y = x.clone()
    for i, sign in ((0, -1.0), (r // 2, 1.0)):
        j = r // 2 - i
        y[..., i:i + r // 2] = (x[..., i:i + r // 2] * cos.double()[:, None, i:i + r // 2]
                                + sign * x[..., j:j + r // 2] * sin.double()[:, None, i:i + r // 2])
    return y


def _exact_append(s):
    q, k, v = _exact_head(s.q, s.qw, s.norm, s.cos, s.sin), _exact_head(s.k, s.kw, s.norm, s.cos, s.sin), s.v.double()
    if s.ks is not None:
        k, v = (torch.clip(x / c.double(), -E4M3_MAX, E4M3_MAX) for x, c in ((k, s.ks), (v, s.vs)))
    kc, vc = s.kc.double(), s.vc.double()
    kept = s.places >= 0
    seq = torch.arange(len(kept), device=kept.device) if s.seqs is None else s.seqs
    place = s.places[kept].long()
    flat = s.table[seq[kept].long(), torch.div(place, s.page, rounding_mode="floor")].long() * s.page + place % s.page
    for cache, x in ((kc, k), (vc, v)):
        rows = cache.transpose(1, 2).reshape(-1, *x.shape[1:])
        rows[flat] = x[kept]
        cache.copy_(rows.view(cache.shape[0], s.page, *x.shape[1:]).transpose(1, 2))
    return q.transpose(0, 1), kc, vc


def _exact_attend(s):
    h, b, d = s.q.shape
    hkv = s.kc.shape[1]
    out = torch.zeros(b, h, d, dtype=torch.float64, device=s.q.device)
    for i, n in enumerate(s.lens.tolist()):
        if not n:
            continue
        pages = s.table[i, :-(-n // s.kc.shape[2])].long()
        k, v = (c.view(torch.uint8)[pages].view(c.dtype) if s.ks is not None else c[pages] for c in (s.kc, s.vc))
        k, v = (x.double().transpose(0, 1).reshape(hkv, -1, d)[:, :n] for x in (k, v))
        if s.ks is not None:
            k, v = k * s.ks.double(), v * s.vs.double()
        score = (k @ s.q[:, i].double().view(hkv, h // hkv, d).transpose(1, 2).contiguous()) / math.sqrt(d)
        w = torch.softmax(score, 1)
        out[i] = (w.transpose(1, 2).contiguous() @ v).reshape(h, d)
    return out.transpose(0, 1)


def _exact_logprobs(s):
    tokens = s.tokens.view(len(s.tokens), -1)
    rows = max(1, (1 << 27) // s.x.shape[1])
    parts = []
    for i in range(0, len(tokens), rows):
        x, t = s.x[i:i + rows].detach().double(), tokens[i:i + rows]
        logp = torch.log_softmax(x, 1)
        given = t >= 0
        o = dict(logprobs=torch.where(given, logp.gather(1, t.clamp(min=0)), 0.0), logsumexp=torch.logsumexp(x, 1))
        p = logp.exp()
        entropy = -torch.where(p > 0, p * logp, 0.0).sum(1)
        if s.entropy:
            o["entropy"] = entropy
        if s.top:
            o["top_logprobs"] = torch.topk(logp, s.top, 1).values
        if s.grad:
            g = torch.where(given, s.g.view(tokens.shape)[i:i + rows].double(), 0.0)
            grad = torch.zeros_like(logp).scatter_add_(1, t.clamp(min=0), g) - p * g.sum(1, keepdim=True)
            if s.top:
                gt, at = s.gt[i:i + rows].double(), torch.sort(x, stable=True, dim=1, descending=True).indices[:, :s.top]
                grad = grad.scatter_add_(1, at, gt) - p * gt.sum(1, keepdim=True)
            if s.entropy:
                grad -= s.ge[i:i + rows, None].double() * p * (logp + entropy[:, None])
            o["grad"] = grad
        parts.append(o)
    out = {f: torch.cat([o[f] for o in parts]) for f in parts[0]}
    out["logprobs"] = out["logprobs"].view(s.tokens.shape)
    return dict(out, top_ids=None)


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "logprobs": _exact_logprobs}[s.kind](s)
