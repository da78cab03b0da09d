"""CPU oracle of the paged cache -- TEST INFRASTRUCTURE ONLY, in float64.

``append`` restates the norm and rotation of the front end (oracle/front.py
``front_bruteforce``'s formulas) without any intermediate rounding and writes
k and v to their pages; ``attend`` is softmax attention of one token per
sequence over the keys its table names. Both loop over tokens.
"""
import math

import torch


def rotate_norm(x, weight, norm, cos, sin, eps=1e-6):
    """float64 [N, heads, D]."""
    x = x.double()
    if norm is not None:
        gain = weight.double() + (1.0 if norm == "zero_centered" else 0.0)
        x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * gain
    if cos is None:
        return x
    r = cos.shape[-1]
    a, b = x[..., :r // 2], x[..., r // 2:r]
    c, s = cos.double()[:, None], sin.double()[:, None]
    return torch.cat((a * c[..., :r // 2] - b * s[..., :r // 2], b * c[..., r // 2:] + a * s[..., r // 2:], x[..., r:]), -1)


def place_of(table, seq, place, page, pages):
    """(page, row) of a place, or None where there is none."""
    if place < 0 or not 0 <= seq < table.shape[0] or place // page >= table.shape[1]:
        return None
    p = int(table[seq, place // page])
    return (p, place % page) if 0 <= p < pages else None


def append(k, v, k_cache, v_cache, table, places, seqs=None):
    """Writes float64 k, v [N, Hkv, D] to float64 caches; returns the (page, row) of each token."""
    pages, _, page, _ = k_cache.shape
    at = [place_of(table, i if seqs is None else int(seqs[i]), int(t), page, pages) for i, t in enumerate(places)]
    for i, w in enumerate(at):
        if w is not None:
            k_cache[w[0], :, w[1]] = k[i]
            v_cache[w[0], :, w[1]] = v[i]
    return at


def attend(q, k_cache, v_cache, table, lens, scale=None):
    """q [H, B, D], caches [pages, Hkv, page, D] of the values they stand for (float64). Returns out
    [H, B, D], lse [H, B], sum p |v| [H, B, D] and max_j sum_d |q_d k_jd| [H, B]; NaN where a
    length or a page is none."""
    h, b, d = q.shape
    pages, hkv, page, _ = k_cache.shape
    scale = 1 / math.sqrt(d) if scale is None else scale
    out, mag = torch.zeros(h, b, d, dtype=torch.float64), torch.zeros(h, b, d, dtype=torch.float64)
    lse, big = torch.full((h, b), -math.inf, dtype=torch.float64), torch.zeros(h, b, dtype=torch.float64)
    for i in range(b):
        n = int(lens[i])
        at = [place_of(table, i, t, page, pages) for t in range(0, max(n, 0), page)]
        if n < 0 or n > table.shape[1] * page or any(w is None for w in at):
            out[:, i], lse[:, i] = math.nan, math.nan
            continue
        if n == 0:
            continue
        rows = torch.tensor([w[0] for w in at])
        k = k_cache[rows].transpose(0, 1).reshape(hkv, -1, d)[:, :n].repeat_interleave(h // hkv, 0)
        v = v_cache[rows].transpose(0, 1).reshape(hkv, -1, d)[:, :n].repeat_interleave(h // hkv, 0)
        s = (k @ q[:, i].double()[..., None])[..., 0] * scale
        p = torch.softmax(s, -1)
        out[:, i], mag[:, i] = (p[:, None] @ v)[:, 0], (p[:, None] @ v.abs())[:, 0]
        lse[:, i] = torch.logsumexp(s, -1)
        big[:, i] = (k.abs() @ q[:, i].double().abs()[..., None])[..., 0].amax(-1)
    return out, lse, mag, big
