"""A paged key-value cache on gfx950: appending new tokens, and attention of one
new token per sequence over what is there.

The reference reads prompts and generates nothing (dan/runner.py:66-82); its
prefix cache keeps whole ``[Hkv, P, D]`` entries (dan/cache.py:11-39). A
sequence that goes on token by token keeps its keys and values in pages instead:

- ``k_cache``, ``v_cache``: ``[pages, Hkv, page_size, D]`` (any page, head and
  token strides: a layer's slice of one allocation will do), bf16 or fp16, or
  e4m3 with one fp32 scale each (``x ~ xq * scale``, as ``attend`` takes it);
- ``table``: int32 ``[sequences, width]``; the key at place ``t`` of a sequence lies
  in page ``table[sequence, t // page_size]``, row ``t % page_size``. Entries
  behind a sequence's last page are not read.

``append_paged`` stands beside ``dan_amd.front.qkv_front`` (norm and rotary of q
and k, dan/models/llama.py:78-86, with the cache as the destination) and
``attend_paged`` beside ``dan_amd.attend``. Both launch on the current stream of the
tensors' device, can be captured into a HIP graph, and read lengths, places and
pages from the device alone: a captured call serves every later step.

There is no CPU path: CPU tensors raise (oracle/paged.py is the test oracle).
"""
import math

import torch

from . import _decode, _native
from .attention import _DTYPES, E4M3, has_tangent
from .front import NORMS, _row_ok, _view


def _check_cache(k_cache, v_cache, k_scale, v_scale, table, dtype, device):
    """Refuses a cache or table that the kernels cannot read; returns
    (pages, Hkv, page size, D) and the scales' addresses."""
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape:
        raise ValueError(f"k_cache {tuple(k_cache.shape)} and v_cache {tuple(v_cache.shape)} must both be [pages, Hkv, page, D]")
    if k_cache.dtype != v_cache.dtype or (k_cache.dtype != dtype and k_cache.dtype != E4M3):
        raise ValueError(f"k_cache and v_cache must share q's {dtype} or {E4M3}; got {k_cache.dtype}, {v_cache.dtype}")
    if not (k_cache.device == v_cache.device == table.device == device):
        raise ValueError(f"k_cache, v_cache and table must be on {device}")
    if not (_row_ok(k_cache) and _row_ok(v_cache)):
        raise ValueError("the cache's rows must have unit stride and be 16-byte aligned (they are written and read in place)")
    if table.dim() != 2 or table.dtype != torch.int32 or (table.shape[1] > 1 and table.stride(1) != 1):
        raise ValueError(f"table must be int32 [sequences, width] with unit stride; got {table.dtype} {tuple(table.shape)}")
    if k_cache.dtype != E4M3:
        if k_scale is not None or v_scale is not None:
            raise ValueError("k_scale and v_scale belong to an e4m3 cache")
        return k_cache.shape, 0, 0
    for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
        if not (isinstance(t, torch.Tensor) and t.numel() == 1 and t.dtype == torch.float32 and t.device == device):
            raise ValueError(f"an e4m3 cache needs {name}: a one-element fp32 tensor on {device}")
    return k_cache.shape, k_scale.data_ptr(), v_scale.data_ptr()


def _check_index(t, name, count, device):
    if t.dtype != torch.int32 or t.shape != (count,) or t.device != device or (count > 1 and t.stride(0) != 1):
        raise ValueError(f"{name} must be a contiguous int32 [{count}] on {device}; got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def append_paged(q, k, v, cos, sin, k_cache, v_cache, table, places, *, seqs=None, rope_rows=None, q_norm_weight=None,
                 k_norm_weight=None, eps=1e-6, norm="rms", k_scale=None, v_scale=None):
    """Writes new tokens' keys and values into their pages, k after its norm and
    rotation, v as it is, and returns q after the same norm and rotation.

    q: [N, H, D]; k, v: [N, Hkv, D] (views of the projection output: any strides
    with a unit-stride head_dim), bf16 or fp16; q may be None (a prefix moved
    into the cache: pass its k with ``norm=None`` and no cos and sin).
    ``norm``, ``q_norm_weight``, ``k_norm_weight``, ``eps``: as in ``qkv_front``.
    cos, sin: [N, R] or None, in the model dtype or fp32 (R: rotary dims, a
    multiple of 16 up to D); with ``rope_rows`` (int32 [N]) token n takes row
    ``rope_rows[n]`` of tables of any length instead (``rope_rows=places`` where a
    token's position is its place), and a row that does not exist makes its
    rotated values NaN.

    ``places`` (int32 [N]): each token's place in its sequence; a negative one
    marks a row without a token (a batch padded to a fixed size), whose k and v are not
    stored. ``seqs`` (int32 [N]): its row of ``table``; None: token n belongs to
    sequence n (a decode step). Tokens whose page the table does not name (past its width,
    or outside the cache) are not stored either. No two tokens may share a place.

    Returns q [H, N, D], a view of a new token-major [N, H, D] tensor (None
    without q). All arithmetic is fp32, rounded once at each store (an e4m3
    cache: ``x / scale`` clamped to +-448), where ``qkv_front`` rounds after each of the
    reference's eager ops; the two differ by up to two roundings of the dtype."""
    dev = k.device
    if not k.is_cuda:
        raise RuntimeError(f"dan_amd.append_paged runs on a gfx950 GPU only; got tensors on {dev}")
    if dev.index != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            return append_paged(q, k, v, cos, sin, k_cache, v_cache, table, places, seqs=seqs, rope_rows=rope_rows,
                                q_norm_weight=q_norm_weight, k_norm_weight=k_norm_weight, eps=eps, norm=norm, k_scale=k_scale,
                                v_scale=v_scale)
    inputs = [t for t in (q, k, v, k_cache, v_cache) if t is not None]
    if (torch.is_grad_enabled() and any(t.requires_grad for t in inputs)) or has_tangent(*inputs):
        raise NotImplementedError("append_paged is forward-only")
    if k.dim() != 3 or v.shape != k.shape:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must both be [N, Hkv, D]")
    n, hkv, d = k.shape
    h = 0
    if q is not None:
        if q.dim() != 3 or q.shape[0] != n or q.shape[2] != d or q.dtype != k.dtype or q.device != dev:
            raise ValueError(f"q {tuple(q.shape)} {q.dtype} must be [{n}, H, {d}] {k.dtype} on {dev}")
        h = q.shape[1]
    if k.dtype not in (torch.bfloat16, torch.float16) or v.dtype != k.dtype or v.device != dev:
        raise ValueError(f"q, k, v must share bf16 or fp16 on {dev}; got {k.dtype}, {v.dtype} on {v.device}")
    if norm not in NORMS:
        raise ValueError(f"norm {norm!r}: one of {list(NORMS)}")
    (pages, chkv, page, cd), ks, vs = _check_cache(k_cache, v_cache, k_scale, v_scale, table, k.dtype, dev)
    if (chkv, cd) != (hkv, d):
        raise ValueError(f"a cache of {chkv} heads x {cd} for k of {hkv} x {d}")
    if any(s == 0 and c > 1 for t in (k_cache, v_cache) for s, c in zip(t.stride(), t.shape)):
        raise ValueError("an expanded cache cannot be written")
    place_p = _check_index(places, "places", n, dev)
    seq_p = 0 if seqs is None else _check_index(seqs, "seqs", n, dev)
    rope_p = 0 if rope_rows is None else _check_index(rope_rows, "rope_rows", n, dev)
    if seqs is None and table.shape[0] < n:
        raise ValueError(f"{n} tokens without seqs need a table of as many rows; got {table.shape[0]}")
    r = 0 if cos is None else cos.shape[-1]
    if r:
        rows = cos.shape[0]
        if cos.dim() != 2 or sin is None or sin.shape != cos.shape or (rows != n and rope_rows is None):
            raise ValueError(f"cos and sin must both be [{n}, R] ([any, R] with rope_rows)")
        if cos.dtype not in (k.dtype, torch.float32) or sin.dtype != cos.dtype or not (cos.device == sin.device == dev):
            raise ValueError(f"cos and sin must share {k.dtype} or fp32 on {dev}; got {cos.dtype}, {sin.dtype}")
        if cos.stride() != sin.stride() or not (_row_ok(cos) and _row_ok(sin)) or cos.stride(0) < r:
            cos, sin = (torch.empty_like(t, memory_format=torch.contiguous_format).copy_(t) for t in (cos, sin))
        elif rows == 1:
            cos, sin = cos.contiguous(), sin.contiguous()
    elif sin is not None and sin.shape[-1]:
        raise ValueError("sin without cos")
    qw = kw = None
    if norm is not None:
        for name, w in (("q_norm_weight", q_norm_weight), ("k_norm_weight", k_norm_weight)):
            if (name[0] == "k" or q is not None) and not (isinstance(w, torch.Tensor) and w.shape == (d,) and w.device == dev):
                raise ValueError(f"norm {norm!r} needs {name}: a [{d}] tensor on {dev}")
        qw, kw = (None if w is None else _view(w.detach().to(k.dtype)) for w in (q_norm_weight if q is not None else None, k_norm_weight))
    q_in, k_in, v_in = None if q is None else _view(q), _view(k), _view(v)
    q_out = None if q is None else torch.empty((n, h, d), dtype=k.dtype, device=dev)
    _decode.call_append(
        _native.stream(dev), _decode.PAGED_ABI_VERSION, _DTYPES[k.dtype], _DTYPES[k_cache.dtype], _DTYPES[cos.dtype if r else k.dtype],
        n, h, hkv, d, r, NORMS[norm], page, pages, table.shape[1], table.shape[0], rows if r else 0, _native.f32(float(eps)),
        *((0, 0, 0) if q is None else (q_in.data_ptr(), *q_in.stride()[:2])), k_in.data_ptr(), *k_in.stride()[:2], v_in.data_ptr(),
        *v_in.stride()[:2], cos.data_ptr() if r else 0, sin.data_ptr() if r else 0, cos.stride(0) if r else 0,
        0 if qw is None else qw.data_ptr(), 0 if kw is None else kw.data_ptr(), *((0, 0, 0) if q is None else (q_out.data_ptr(), h * d, d)),
        k_cache.data_ptr(), *k_cache.stride()[:3], v_cache.data_ptr(), *v_cache.stride()[:3], ks, vs, table.data_ptr(), table.stride(0),
        place_p, seq_p, rope_p)
    return None if q is None else q_out.transpose(0, 1)


def attend_paged(q, k_cache, v_cache, table, lens, scale=None, *, k_scale=None, v_scale=None, max_len=None, return_lse=False):
    """Attention of one new token per sequence over the sequence's cached keys.

    q: [H, B, D] (rotary applied; what ``append_paged`` returns), bf16 or fp16,
    H a multiple of Hkv. ``lens`` (int32 [B]): how many keys each sequence has,
    the new token's own among them; places behind them are not read (they may hold
    anything). ``max_len``: the most that any entry of ``lens`` reaches while this
    call (or a graph that captured it) runs, by default all that the table can
    hold; the launch is sized for it, so a tight one saves time.

    Returns [H, B, D], a view of token-major [B, H, D] storage, in q's dtype;
    with ``return_lse`` also the fp32 [H, B] log of the sum of e^score (a merge with other
    keys' attention takes it, dan/fused.py:94-101). A sequence of no keys gives
    zeros and -inf. A length outside [0, max_len], or a page outside the
    cache, gives NaN for its sequence.

    The keys are split between work groups by B, Hkv and ``max_len`` alone, so a
    sequence's result does not depend on its neighbours' lengths."""
    dev = q.device
    if not q.is_cuda:
        raise RuntimeError(f"dan_amd.attend_paged runs on a gfx950 GPU only; got tensors on {dev}")
    if dev.index != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            return attend_paged(q, k_cache, v_cache, table, lens, scale, k_scale=k_scale, v_scale=v_scale, max_len=max_len,
                                return_lse=return_lse)
    if (torch.is_grad_enabled() and (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad)) or has_tangent(q, k_cache, v_cache):
        raise NotImplementedError("attend_paged is forward-only")
    if q.dim() != 3 or q.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"q must be [H, B, D] in bf16 or fp16; got {tuple(q.shape)} {q.dtype}")
    h, b, d = q.shape
    (pages, hkv, page, cd), ks, vs = _check_cache(k_cache, v_cache, k_scale, v_scale, table, q.dtype, dev)
    if cd != d or hkv == 0 or h == 0 or h % hkv:
        raise ValueError(f"q of {h} heads x {d} on a cache of {hkv} x {cd}: the heads must be a multiple, head_dim the same")
    if table.shape[0] != b:
        raise ValueError(f"a table of {table.shape[0]} sequences for {b} tokens")
    len_p = _check_index(lens, "lens", b, dev)
    most = table.shape[1] * page if max_len is None else int(max_len)
    if not 0 <= most <= table.shape[1] * page:
        raise ValueError(f"max_len {max_len}: the table holds {table.shape[1] * page} keys a sequence")
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    elif not (float(scale) > 0 and math.isfinite(float(scale))):
        raise ValueError(f"scale {scale}: the kernel needs a finite positive softmax scale")
    q = _view(q)
    out = torch.empty((b, h, d), dtype=q.dtype, device=dev)
    lse = torch.empty((b, h), dtype=torch.float32, device=dev) if return_lse else None
    need = _decode.paged_attn_workspace_size(dev.index, b, h, hkv, d, most)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need > 0 else None
    _decode.call_paged_attn(
        _native.stream(dev), _decode.PAGED_ABI_VERSION, _DTYPES[q.dtype], _DTYPES[k_cache.dtype], b, h, hkv, d, page, pages,
        table.shape[1], most, _native.f32(float(scale)), q.data_ptr(), q.stride(1), q.stride(0), out.data_ptr(), h * d, d,
        0 if lse is None else lse.data_ptr(), k_cache.data_ptr(), *k_cache.stride()[:3], v_cache.data_ptr(), *v_cache.stride()[:3],
        ks, vs, table.data_ptr(), table.stride(0), len_p, 0 if ws is None else ws.data_ptr(), max(need, 0))
    out = out.transpose(0, 1)
    return (out, lse.transpose(0, 1)) if return_lse else out
