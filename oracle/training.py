"""CPU oracle of the operators that train and serve adapters -- TEST INFRASTRUCTURE ONLY.

fp64 restatements from the definitions:

- ``attend``: tree attention and its gradient, one query row at a time: the visible keys of
  a row are listed from the segment's trunk and branches (dan/attention.py:54-59), so that a
  hidden key takes no part in any sum;
- ``adapt``: low-rank adapters beside a shared projection, one row at a time.

Where a result was made by adding up terms, its bound (what a test multiplies by a
rounding's size) is the same sum over the terms' magnitudes: ``abs_`` results.
"""
import math

import torch


def attend(q, k, v, segments, layer, scale=None, grad=None):
    """q [H, N, D], k, v [Hkv, N, D] (any dtype) -> dict of fp64 tensors: out [H, N, D], lse [H, N] (natural), and with
    ``grad`` [H, N, D] dq, dk, dv, and their bounds abs_out, abs_dq, abs_dk, abs_dv: what they would be if every
    product of a row's P, dS, K, Q, V or G had its magnitude (dS's own: P (|dP| + |delta|))."""
    q, k, v = (x.detach().double().cpu() for x in (q, k, v))
    h, n, d = q.shape
    rep = h // k.shape[0]
    scale = d ** -0.5 if scale is None else scale
    r = dict(out=torch.zeros_like(q), lse=torch.full((h, n), -math.inf, dtype=torch.float64), abs_out=torch.zeros_like(q))
    if grad is not None:
        grad = grad.detach().double().cpu()
        r.update({f: torch.zeros_like(x) for f, x in (("dq", q), ("dk", k), ("dv", v), ("abs_dq", q), ("abs_dk", k), ("abs_dv", v))})
    for s in segments:
        pk = pv = None
        if s.past:
            pk, pv = (x.detach().double().cpu() for x in s.past[layer][:2])
        spans = [(s.start, s.start + s.trunk)] + list(s.branches)
        for j, (a, b) in enumerate(spans):
            for i in range(a, b):
                own = list(range(s.start, (i if j == 0 else s.start + s.trunk - 1) + 1)) + (list(range(a, i + 1)) if j else [])
                kk, vv = k[:, own], v[:, own]
                if pk is not None:
                    kk, vv = torch.cat((pk, kk), 1), torch.cat((pv, vv), 1)
                kk, vv = kk.repeat_interleave(rep, 0), vv.repeat_interleave(rep, 0)  # [H, keys, D]
                x = scale * (kk @ q[:, i, :, None])[..., 0]
                m = x.amax(1, keepdim=True)
                e = (x - m).exp()
                z = e.sum(1, keepdim=True)
                p = e / z
                r["lse"][:, i] = (m + z.log())[:, 0]
                r["out"][:, i] = (p[:, None] @ vv)[:, 0]
                r["abs_out"][:, i] = (p[:, None] @ vv.abs())[:, 0]
                if grad is None:
                    continue
                g = grad[:, i]
                dp = (vv @ g[..., None])[..., 0]
                delta = (p * dp).sum(1, keepdim=True)
                ds = p * (dp - delta)
                ads = p * (dp.abs() + (vv.abs() @ g.abs()[..., None])[..., 0].mul(p).sum(1, keepdim=True))
                first = 0 if pk is None else pk.shape[1]
                r["dq"][:, i] = scale * (ds[:, None] @ kk)[:, 0]
                r["abs_dq"][:, i] = scale * (ads[:, None] @ kk.abs())[:, 0]
                idx = torch.tensor(own)
                for f, w, y in (("dk", scale * ds, q[:, i]), ("dv", p, g), ("abs_dk", scale * ads, q[:, i].abs()), ("abs_dv", p, g.abs())):
                    term = w[:, first:, None] * y[:, None]  # [H, own keys, D]
                    r[f].index_add_(1, idx, term.view(-1, rep, len(own), d).sum(1))
    return r


def adapt(y, x, a, b, index, scale, grad=None):
    """Row by row, fp64: dict of out and abs_out, and with ``grad`` dx, da, db and their abs_ bounds. index: a list; negative:
    no adapter, past the last: NaN (in dx, too; no part of da and db)."""
    y, x, a, b = (t.detach().double().cpu() for t in (y, x, a, b))
    scale = scale.double().cpu().tolist() if isinstance(scale, torch.Tensor) else [scale] * len(a)
    r = dict(out=y.clone(), abs_out=y.abs())
    if grad is not None:
        grad = grad.detach().double().cpu()
        r.update({f: torch.zeros_like(t) for f, t in (("dx", x), ("da", a), ("db", b), ("abs_dx", x), ("abs_da", a), ("abs_db", b))})
    for n, i in enumerate(index):
        if i < 0:
            continue
        if i >= len(a):
            r["out"][n] = math.nan
            if grad is not None:
                r["dx"][n] = math.nan
            continue
        c, h, ah = scale[i], a[i] @ x[n], a[i].abs() @ x[n].abs()
        r["out"][n] += c * (b[i] @ h)
        r["abs_out"][n] += abs(c) * (b[i].abs() @ ah)
        if grad is not None:
            g, ag = grad[n] @ b[i], grad[n].abs() @ b[i].abs()
            r["dx"][n] = c * (g @ a[i])
            r["abs_dx"][n] = abs(c) * (ag @ a[i].abs())
            r["da"][i] += c * torch.outer(g, x[n])
            r["abs_da"][i] += abs(c) * torch.outer(ag, x[n].abs())
            r["db"][i] += c * torch.outer(grad[n], h)
            r["abs_db"][i] += abs(c) * torch.outer(grad[n].abs(), ah)
    return r


def add_norm(x, residual, weight, eps=1e-6, norm="rms", grad=None, grad_stream=None):
    """fp64: dict of stream, out, scale (of e4m3 codes), and with ``grad`` ds, dw and their abs_ bounds."""
    s = x.detach().double().cpu()
    if residual is not None:
        s = s + residual.detach().double().cpu()
    w = weight.detach().double().cpu() + (1.0 if norm == "zero_centered" else 0.0)
    rs = 1.0 / ((s * s).mean(1, keepdim=True) + eps).sqrt()
    hat = s * rs
    out = hat * w
    r = dict(stream=s, out=out, scale=out.abs().amax(1, keepdim=True).clamp(min=1e-12) / 448.0)
    if grad is not None:
        g = grad.detach().double().cpu()
        gs = torch.zeros_like(s) if grad_stream is None else grad_stream.detach().double().cpu()
        r["ds"] = rs * (w * g - hat * (w * g * hat).mean(1, keepdim=True)) + gs
        r["abs_ds"] = rs * ((w * g).abs() + hat.abs() * (w * g * hat).abs().mean(1, keepdim=True)) + gs.abs()
        r["dw"], r["abs_dw"] = (g * hat).sum(0), (g * hat).abs().sum(0)
    return r
