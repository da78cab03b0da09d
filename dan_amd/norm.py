"""The residual's addition and the root-mean-square norm in front of a
projection (include/dan_norm.h), in one pass, with the result in 16 bits, as
e4m3 codes for ``dan_amd.quant.fp8_gemm``, or both.

dan adds, normalises (dan/fused.py:35-48) and quantises (dan/fused.py:85-91) in
steps; ``add_norm`` reads both addends once, and has a gradient.

There is no CPU path: CPU tensors raise.
"""
from typing import NamedTuple, Optional

import torch

from . import _decode, _layer, _native
from .attention import _DTYPES, E4M3, has_tangent
from .quant import TiledE4M3, tiled_bytes

NORMS = {"rms": _layer.NORM_RMS, "zero_centered": _layer.NORM_ZERO_CENTERED}
LAYOUTS = {"rows": _native.FP8_LAYOUT_ROWS, "tiled": _native.FP8_LAYOUT_TILED}


class Normed(NamedTuple):
    """``add_norm``'s results; None where not asked for."""

    out: Optional[torch.Tensor]  # [N, K], x's dtype
    stream: torch.Tensor  # x + residual [N, K] (x itself without a residual)
    codes: object = None  # e4m3 [N, K], or a TiledE4M3
    scale: Optional[torch.Tensor] = None  # fp32 [N, 1]


def _forward(x, residual, weight, eps, norm, fp8, want_out, want_rstd):
    """(out, stream, codes, scale, rstd)."""
    n, k = x.shape
    dev = x.device
    x, weight = _layer.rows_of(x), _layer.dense(weight)
    stream = out = codes = scale = rstd = None
    if residual is not None:
        residual = _layer.rows_of(residual)
        stream = torch.empty((n, k), dtype=x.dtype, device=dev)
    if want_out:
        out = torch.empty((n, k), dtype=x.dtype, device=dev)
    if fp8 is not None:
        scale = torch.empty((n, 1), dtype=torch.float32, device=dev)
        codes = torch.empty((n, k), dtype=E4M3, device=dev) if fp8 == "rows" else torch.empty(tiled_bytes(n, k), dtype=torch.uint8, device=dev)
    if want_rstd:
        rstd = torch.empty(n, dtype=torch.float32, device=dev)
    if n:
        _layer.call_norm(
            _native.stream(dev), _layer.NORM_ABI_VERSION, _DTYPES[x.dtype], n, k, NORMS[norm], LAYOUTS[fp8 or "rows"], _native.f32(float(eps)), 0,
            x.data_ptr(), x.stride(0), 0 if residual is None else residual.data_ptr(), 0 if residual is None else residual.stride(0),
            weight.data_ptr(), 0 if stream is None else stream.data_ptr(), k, 0 if out is None else out.data_ptr(), k,
            0 if codes is None else codes.data_ptr(), 0 if scale is None else scale.data_ptr(), 0 if rstd is None else rstd.data_ptr())
    return out, stream, TiledE4M3(codes, n, k) if fp8 == "tiled" else codes, scale, rstd


class _AddNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps, norm):
        out, stream, _, _, rstd = _forward(x, residual, weight, eps, norm, None, True, True)
        ctx.save_for_backward(x if residual is None else stream, weight, rstd)
        ctx.norm, ctx.alone = norm, residual is None
        ctx.set_materialize_grads(False)
        return out if residual is None else (out, stream)

    @staticmethod
    @_layer.once("add_norm")
    def backward(ctx, g, g_stream=None):
        s, weight, rstd = ctx.saved_tensors
        _decode.check_capture(s.device.index, "add_norm")
        need_x, need_r, need_w = ctx.needs_input_grad[:3]
        if g is None:  # the sum alone was used
            return g_stream if need_x else None, g_stream if need_r else None, None, None, None
        with torch.cuda.device(s.device):  # (the engine's thread is on the gradient's device)
            ds, dw = _backward(s, weight, rstd, g, g_stream, ctx.norm, need_w)
        return ds if need_x else None, ds if need_r else None, dw, None, None


def _backward(s, weight, rstd, g, g_stream, norm, need_w):
    n, k = s.shape
    dev = s.device
    ds = torch.empty((n, k), dtype=s.dtype, device=dev)
    dw = torch.empty(k, dtype=s.dtype, device=dev) if need_w else None
    if not n:
        return ds, None if dw is None else dw.zero_()
    s, g, w = _layer.rows_of(s), _layer.rows_of(g), _layer.dense(weight)
    gs = None if g_stream is None else _layer.rows_of(g_stream)
    nbytes = _layer.norm_grad_workspace_size(n, k) if need_w else 0
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if need_w else None
    _layer.call_norm_grad(
        _native.stream(dev), _layer.NORM_ABI_VERSION, _DTYPES[s.dtype], n, k, NORMS[norm], 0, s.data_ptr(), s.stride(0), w.data_ptr(),
        rstd.data_ptr(), g.data_ptr(), g.stride(0), 0 if gs is None else gs.data_ptr(), 0 if gs is None else gs.stride(0), ds.data_ptr(), k,
        0 if dw is None else dw.data_ptr(), 0 if ws is None else ws.data_ptr(), nbytes)
    return ds, dw


def add_norm(x, residual, weight, *, eps=1e-6, norm="rms", fp8=None, out=None):
    """x, residual: [N, K] (bf16 or fp16; residual may be None), weight: [K] of
    the same dtype. Returns ``Normed``:

    - ``stream``: x + residual, rounded to x's dtype (x itself without a residual);
    - ``out``: the norm of the sum times the weight ("rms", dan/fused.py:35-40) or
      one plus the weight ("zero_centered", :44-48), in x's dtype;
    - with ``fp8`` "rows" or "tiled": ``codes``, the same norm as e4m3 codes [N, K],
      or as the GEMM's operand (``TiledE4M3``), and ``scale`` [N, 1], a row's largest
      magnitude over 448, as ``dan_amd.quant.fp8_quantize`` makes them.

    The norm is of the fp32 sum; ``out`` and the codes are each rounded once, from
    fp32. ``out`` defaults to whether ``fp8`` is None; True gives both, as a
    projection with adapters needs them. K: a multiple of 8 (16 with ``fp8``), at
    most 16384; fewer than 2^24 rows (with ``fp8`` "tiled" and
    more than 1024 columns at most 2^24 - 256).

    Without ``fp8`` the result is differentiable (once) in x, residual and weight;
    the gradient takes the sum as ``stream`` holds it. A backward pass that is
    captured into a HIP graph has its forward pass in the same capture, and no
    earlier, eager result that holds the graph of the same leaves is alive (where an
    input is such a leaf itself, that raises)."""
    want_out = fp8 is None if out is None else bool(out)
    made = _layer.calls().add_norm(x, residual, weight, eps, NORMS.get(norm), -1 if fp8 is None else LAYOUTS.get(fp8), want_out)
    if made is not None:  # a plain call
        out, stream, codes, scale = made
        return Normed(out, x if residual is None else stream, TiledE4M3(codes, *x.shape) if fp8 == "tiled" else codes, scale)
    if not x.is_cuda:
        raise RuntimeError(f"dan_amd.add_norm runs on a gfx950 GPU only; got tensors on {x.device}")
    if x.device.index != torch._C._cuda_getDevice():
        with torch.cuda.device(x.device):
            return add_norm(x, residual, weight, eps=eps, norm=norm, fp8=fp8, out=out)
    if norm not in NORMS:
        raise ValueError(f"norm {norm!r}: one of {list(NORMS)}")
    if fp8 is not None and fp8 not in LAYOUTS:
        raise ValueError(f"fp8 {fp8!r}: None or one of {list(LAYOUTS)}")
    if x.dim() != 2 or x.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"x must be [N, K] in bf16 or fp16; got {tuple(x.shape)} {x.dtype}")
    n, k = x.shape
    if k % (8 if fp8 is None else 16) or not 0 < k <= _layer.MAX_COLS:
        raise ValueError(f"K {k}: a multiple of {8 if fp8 is None else 16} up to {_layer.MAX_COLS}")
    if n >= 1 << 24 or fp8 == "tiled" and k > 1024 and n > (1 << 24) - 256:
        raise ValueError(f"{n} rows: fewer than 2^24, at most 2^24 - 256 with tiled codes of more than 1024 columns")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError(f"residual {tuple(residual.shape)} {residual.dtype} on {residual.device} must be as x")
    if weight.shape != (k,) or weight.dtype != x.dtype or weight.device != x.device:
        raise ValueError(f"weight must be [{k}] {x.dtype} on {x.device}; got {tuple(weight.shape)} {weight.dtype} on {weight.device}")
    if not 0 <= float(eps) < float("inf"):
        raise ValueError(f"eps {eps}: finite and not negative")
    if fp8 is None and not want_out:
        raise ValueError("out=False without fp8: nothing is left to compute")
    inputs = [t for t in (x, residual, weight) if t is not None]
    if has_tangent(*inputs):
        raise NotImplementedError("add_norm has no forward-mode derivative")
    if torch.is_grad_enabled() and any(t.requires_grad for t in inputs):
        if fp8 is not None:
            raise NotImplementedError("add_norm: e4m3 codes have no gradient")
        got = _AddNorm.apply(x, residual, weight, eps, norm)
        return Normed(got, x) if residual is None else Normed(*got)
    out, stream, codes, scale, _ = _forward(x, residual, weight, eps, norm, fp8, want_out, False)
    return Normed(out, x if residual is None else stream, codes, scale)
