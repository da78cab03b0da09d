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
  behind a sequence's last page may be loaded (the whole table has to be
  readable), but nothing follows from what they hold.

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
from .front import NORMS


def _rows(t):
    """t (16-bit, three-dimensional) or a fresh contiguous copy where its rows are not 16-byte aligned or of unit
    stride, with its address and its first two strides."""
    s0, s1, s2 = t.stride()
    at = t.data_ptr()
    if s2 != 1 or ((s0 | s1) * 2 | at) & 15:
        t = torch.empty_like(t, memory_format=torch.contiguous_format).copy_(t)
        (s0, s1, _), at = t.stride(), t.data_ptr()
    return t, at, s0, s1


def _cache_rows(t):
    """A cache's address and first three strides; its rows are written and read in place."""
    s0, s1, s2, s3 = t.stride()
    at = t.data_ptr()
    if s3 != 1 or ((s0 | s1 | s2) * t.element_size() | at) & 15:
        raise ValueError("the cache's rows must have unit stride and be 16-byte aligned (they are written and read in place)")
    return at, s0, s1, s2


def _check_cache(k_cache, v_cache, k_scale, v_scale, table, dtype, device):
    """Refuses a cache or table that the kernels cannot read; returns
    [pages, Hkv, page size, D] and the scales' addresses."""
    shape, kind = k_cache.shape, k_cache.dtype
    if len(shape) != 4 or shape != v_cache.shape:
        raise ValueError(f"k_cache {tuple(shape)} and v_cache {tuple(v_cache.shape)} must both be [pages, Hkv, page, D]")
    if kind != v_cache.dtype or (kind != dtype and kind != E4M3):
        raise ValueError(f"k_cache and v_cache must share q's {dtype} or {E4M3}; got {kind}, {v_cache.dtype}")
    if not (k_cache.device == v_cache.device == table.device == device):
        raise ValueError(f"k_cache, v_cache and table must be on {device}")
    if table.dim() != 2 or table.dtype != torch.int32 or (table.stride(1) != 1 and table.shape[1] > 1):
        raise ValueError(f"table must be int32 [sequences, width] with unit stride; got {table.dtype} {tuple(table.shape)}")
    if kind != E4M3:
        if k_scale is not None or v_scale is not None:
            raise ValueError("k_scale and v_scale belong to an e4m3 cache")
        return shape, 0, 0
    for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
        if not (isinstance(t, torch.Tensor) and t.numel() == 1 and t.dtype == torch.float32 and t.device == device):
            raise ValueError(f"an e4m3 cache needs {name}: a one-element fp32 tensor on {device}")
    return shape, k_scale.data_ptr(), v_scale.data_ptr()


def _forward_only(name, *inputs):
    """Refuses inputs that a derivative is wanted of."""
    inputs = [t for t in inputs if isinstance(t, torch.Tensor)]
    if (torch.is_grad_enabled() and any(t.requires_grad for t in inputs)) or has_tangent(*inputs):
        raise NotImplementedError(f"{name} is forward-only")


def _check_index(t, name, count, device):
    if t.dtype != torch.int32 or t.shape != (count,) or t.device != device or (t.stride(0) != 1 and count > 1):
        raise ValueError(f"{name} must be a contiguous int32 [{count}] on {device}; got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def append_paged(q, k, v, cos, sin, k_cache, v_cache, table, places, *, seqs=None, rope_rows=None, q_norm_weight=None,
                 k_norm_weight=None, eps=1e-6, norm="rms", k_scale=None, v_scale=None):
    """Writes new tokens' keys and values into their pages, k after its norm and
    rotation, v as it is, and returns q after the same norm and rotation.

    q: [N, H, D]; k, v: [N, Hkv, D] (views of the projection output: any strides
    with a unit-stride head_dim), bf16 or fp16; q may be None (keys that ``qkv_front`` has
    made for ``attend``, or a prefix, moved into the cache as they are: pass them with
    ``norm=None`` and no cos and sin).
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
    or outside the cache) are not stored either. No two tokens may share a place, and
    q, k and v may not lie in rows of the cache that the call writes. To autograd it is an in-place
    operation on both caches.

    Returns q [H, N, D], a view of a new token-major [N, H, D] tensor (None
    without q). All arithmetic is fp32, rounded once at each store (an e4m3
    cache: ``x / scale`` clamped to +-448), where ``qkv_front`` rounds after each of the
    reference's eager ops; the two differ by up to two roundings of the dtype."""
    out = _decode.calls().append(q, k, v, cos, sin, k_cache, v_cache, table, places, seqs, rope_rows, q_norm_weight, k_norm_weight,
                                 eps, NORMS.get(norm, -1), k_scale, v_scale)
    if out is not None:  # a plain call, made
        return out
    dev = k.device
    if not k.is_cuda:
        raise RuntimeError(f"dan_amd.append_paged runs on a gfx950 GPU only; got tensors on {dev}")
    if dev.index != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            return append_paged(q, k, v, cos, sin, k_cache, v_cache, table, places, seqs=seqs, rope_rows=rope_rows,
                                q_norm_weight=q_norm_weight, k_norm_weight=k_norm_weight, eps=eps, norm=norm, k_scale=k_scale,
                                v_scale=v_scale)
    _forward_only("append_paged", q, k, v, cos, sin, k_cache, v_cache, k_scale, v_scale, *((q_norm_weight, k_norm_weight) if norm is not None else ()))
    dtype, shape = k.dtype, k.shape
    if len(shape) != 3 or v.shape != shape:
        raise ValueError(f"k {tuple(shape)} and v {tuple(v.shape)} must both be [N, Hkv, D]")
    n, hkv, d = shape
    if (dtype != torch.bfloat16 and dtype != torch.float16) or v.dtype != dtype or v.device != dev:
        raise ValueError(f"q, k, v must share bf16 or fp16 on {dev}; got {dtype}, {v.dtype} on {v.device}")
    (pages, chkv, page, cd), ks, vs = _check_cache(k_cache, v_cache, k_scale, v_scale, table, dtype, dev)
    if chkv != hkv or cd != d:
        raise ValueError(f"a cache of {chkv} heads x {cd} for k of {hkv} x {d}")
    kc, vc = _cache_rows(k_cache), _cache_rows(v_cache)
    if (0 in kc or 0 in vc) and any(s == 0 and c > 1 for t in (k_cache, v_cache) for s, c in zip(t.stride(), t.shape)):
        raise ValueError("an expanded cache cannot be written")
    seqs_of_table, width = table.shape
    if seqs is None and seqs_of_table < n:
        raise ValueError(f"{n} tokens without seqs need a table of as many rows; got {seqs_of_table}")
    place_p = _check_index(places, "places", n, dev)
    seq_p = 0 if seqs is None else _check_index(seqs, "seqs", n, dev)
    rope_p = 0 if rope_rows is None else _check_index(rope_rows, "rope_rows", n, dev)

    r = rows = cs_p = sn_p = cs_st = 0
    cs_type = dtype
    if cos is not None and cos.shape[-1]:
        rows, r = cos.shape if cos.dim() == 2 else (0, 0)
        if not r or sin is None or sin.shape != cos.shape or (rows != n and rope_rows is None):
            raise ValueError(f"cos and sin must both be [{n}, R] ([any, R] with rope_rows)")
        cs_type = cos.dtype
        if (cs_type != dtype and cs_type != torch.float32) or sin.dtype != cs_type or not (cos.device == sin.device == dev):
            raise ValueError(f"cos and sin must share {dtype} or fp32 on {dev}; got {cs_type}, {sin.dtype}")
        cs_st, one = cos.stride()
        cs_p, sn_p = cos.data_ptr(), sin.data_ptr()
        if one != 1 or sin.stride() != (cs_st, one) or cs_st < r or (cs_st * cos.element_size() | cs_p | sn_p) & 15:
            cos, sin = (torch.empty_like(t, memory_format=torch.contiguous_format).copy_(t) for t in (cos, sin))
            cs_st, cs_p, sn_p = r, cos.data_ptr(), sin.data_ptr()
    elif sin is not None and sin.shape[-1]:
        raise ValueError("sin without cos")

    if norm not in NORMS:
        raise ValueError(f"norm {norm!r}: one of {list(NORMS)}")
    qw_p = kw_p = 0
    if norm is not None:
        qw, kw = (_weight(w, name, norm, dtype, d, dev) for w, name in ((k_norm_weight if q is None else q_norm_weight, "q_norm_weight"),
                                                                        (k_norm_weight, "k_norm_weight")))
        qw_p, kw_p = qw.data_ptr(), kw.data_ptr()
    h = q_p = q_st = q_sh = out_p = 0
    out = None
    if q is not None:
        if q.dim() != 3 or q.shape[0] != n or q.shape[2] != d or q.dtype != dtype or q.device != dev:
            raise ValueError(f"q {tuple(q.shape)} {q.dtype} must be [{n}, H, {d}] {dtype} on {dev}")
        h = q.shape[1]
        q, q_p, q_st, q_sh = _rows(q)
        out = torch.empty((n, h, d), dtype=dtype, device=dev)
        out_p = out.data_ptr()
    k, k_p, k_st, k_sh = _rows(k)
    v, v_p, v_st, v_sh = _rows(v)
    _decode.call_append(
        _native.stream(dev), _decode.PAGED_ABI_VERSION, _DTYPES[dtype], _DTYPES[k_cache.dtype], _DTYPES[cs_type], n, h, hkv, d, r, NORMS[norm],
        page, pages, width, seqs_of_table, rows, _native.f32(float(eps)), q_p, q_st, q_sh, k_p, k_st, k_sh, v_p, v_st, v_sh,
        cs_p, sn_p, cs_st, qw_p, kw_p, out_p, h * d, d, *kc, *vc, ks, vs, table.data_ptr(), table.stride(0), place_p, seq_p, rope_p)
    if n:  # a backward that has saved a cache must not take the new rows for the old
        torch.autograd.graph.increment_version([k_cache, v_cache])
    return None if out is None else out.transpose(0, 1)


def _weight(w, name, norm, dtype, d, device):
    """A norm weight in the model dtype, contiguous and 16-byte aligned."""
    if not (isinstance(w, torch.Tensor) and w.shape == (d,) and w.device == device):
        raise ValueError(f"norm {norm!r} needs {name}: a [{d}] tensor on {device}")
    if w.dtype == dtype and w.stride(0) == 1 and not w.data_ptr() & 15:
        return w
    return torch.empty(d, dtype=dtype, device=device).copy_(w.detach())


def attend_paged(q, k_cache, v_cache, table, lens, scale=None, *, k_scale=None, v_scale=None, max_len=None, return_lse=False):
    """Attention of one new token per sequence over the sequence's cached keys.

    q: [H, B, D] (rotary applied; what ``append_paged`` returns), bf16 or fp16,
    H a multiple of Hkv. ``lens`` (int32 [B]): how many keys each sequence has,
    the new token's own among them; rows behind them, and page 0, may be loaded, but
    whatever they hold changes no result. ``max_len``: the most that any entry of ``lens`` reaches while this
    call (or a graph that captured it) runs, by default all that the table can
    hold. The launch and its workspace are sized for it: up to about twice the longest length costs a short
    sequence a second launch and others nothing, far more does (64 sequences of up to 1000 keys: 33 us, 155 for a table of 131072).

    Returns [H, B, D], a view of token-major [B, H, D] storage, in q's dtype;
    with ``return_lse`` also the fp32 [H, B] log of the sum of e^score (a merge with other
    keys' attention takes it, dan/fused.py:94-101). A sequence of no keys gives
    zeros and -inf. ``scale``: positive, at most 2^127. A length outside [0, max_len], or a page outside the
    cache, gives NaN for its sequence. An infinite value among a sequence's own may give NaN where
    the sum would be infinite (weights are held in parts).

    How a sequence's keys are split between work groups follows from its own length,
    B, Hkv and ``max_len``: its result does not depend on its neighbours' lengths."""
    made = _decode.calls().attend(q, k_cache, v_cache, table, lens, scale, k_scale, v_scale, max_len, return_lse)
    if made is not None:  # a plain call
        return made
    dev = q.device
    if not q.is_cuda:
        raise RuntimeError(f"dan_amd.attend_paged runs on a gfx950 GPU only; got tensors on {dev}")
    if dev.index != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            return attend_paged(q, k_cache, v_cache, table, lens, scale, k_scale=k_scale, v_scale=v_scale, max_len=max_len,
                                return_lse=return_lse)
    _forward_only("attend_paged", q, k_cache, v_cache, k_scale, v_scale)
    dtype, shape = q.dtype, q.shape
    if len(shape) != 3 or (dtype != torch.bfloat16 and dtype != torch.float16):
        raise ValueError(f"q must be [H, B, D] in bf16 or fp16; got {tuple(shape)} {dtype}")
    h, b, d = shape
    (pages, hkv, page, cd), ks, vs = _check_cache(k_cache, v_cache, k_scale, v_scale, table, dtype, dev)
    if cd != d or hkv == 0 or h == 0 or h % hkv:
        raise ValueError(f"q of {h} heads x {d} on a cache of {hkv} x {cd}: the heads must be a multiple, head_dim the same")
    rows, width = table.shape
    if rows != b:
        raise ValueError(f"a table of {rows} sequences for {b} tokens")
    len_p = _check_index(lens, "lens", b, dev)
    most = width * page if max_len is None else int(max_len)
    if not 0 <= most <= width * page:
        raise ValueError(f"max_len {max_len}: the table holds {width * page} keys a sequence")
    if scale is None:
        scale = d ** -0.5
    elif not (float(scale) > 0 and math.isfinite(float(scale))):
        raise ValueError(f"scale {scale}: the kernel needs a finite positive softmax scale")
    q, q_p, q_sh, q_ss = _rows(q)
    out = torch.empty((b, h, d), dtype=dtype, device=dev)
    lse = torch.empty((b, h), dtype=torch.float32, device=dev) if return_lse else None
    kind = _DTYPES[k_cache.dtype]
    need = _decode.paged_attn_workspace_size(dev.index, kind, b, h, hkv, d, most)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need > 0 else None
    _decode.call_paged_attn(
        _native.stream(dev), _decode.PAGED_ABI_VERSION, _DTYPES[dtype], kind, b, h, hkv, d, page, pages, width, most,
        _native.f32(float(scale)), q_p, q_ss, q_sh, out.data_ptr(), h * d, d, 0 if lse is None else lse.data_ptr(),
        *_cache_rows(k_cache), *_cache_rows(v_cache), ks, vs, table.data_ptr(), table.stride(0), len_p,
        0 if ws is None else ws.data_ptr(), max(need, 0))
    out = out.transpose(0, 1)
    return (out, lse.transpose(0, 1)) if return_lse else out
