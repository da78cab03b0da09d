"""Low-rank adapters beside a shared projection (include/dan_adapt.h).

dan trains one adapter and merges it into the model's weights (dan/lora.py,
dan/tuning.py:82-133). Here the projection is shared, in any form (``nn.Linear``,
``dan_amd.quant.FP8Linear``), and each row of a packed batch adds its own
request's adapter to the projection's output: ``adapt``, with its gradient.

There is no CPU path: CPU tensors raise.
"""
import math

import torch
from torch import nn

from . import _decode, _layer, _native
from .attention import _DTYPES, has_tangent
from .quant import FP8Linear


def _down_rank(r):
    return 16 if r <= 16 else 32 if r <= 32 else 64 if r <= 64 else 128


def _scale_args(scale):
    return (scale.data_ptr(), 0.0) if isinstance(scale, torch.Tensor) else (0, _native.f32(scale))


def _forward(y, x, a, b, index, scale, want_down):
    """(out, the rows' x A^T or None)."""
    (n, n_in), n_out = x.shape, y.shape[1]
    x, y = _layer.rows_of(x), _layer.rows_of(y)
    a, b = _layer.dense(a), _layer.dense(b)
    r = a.shape[1]
    out = torch.empty((n, n_out), dtype=x.dtype, device=x.device)
    down = torch.empty((n, _down_rank(r)), dtype=torch.float32, device=x.device) if want_down else None
    if n:
        nbytes = _layer.adapt_workspace_size(n, n_in, r, a.shape[0])
        ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        _layer.call_adapt(
            _native.stream(x.device), _layer.ADAPT_ABI_VERSION, _DTYPES[x.dtype], n, n_in, n_out, r, a.shape[0], 0,
            x.data_ptr(), x.stride(0), y.data_ptr(), y.stride(0), a.data_ptr(), b.data_ptr(), 0 if index is None else index.data_ptr(),
            *_scale_args(scale), out.data_ptr(), n_out, 0 if down is None else down.data_ptr(), ws.data_ptr(), nbytes)
    return out, down


class _Adapt(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, x, a, b, index, scale):
        out, down = _forward(y, x, a, b, index, scale, True)
        ctx.save_for_backward(x, a, b, down, *(t for t in (index, scale) if isinstance(t, torch.Tensor)))
        ctx.index, ctx.scale = index is not None, None if isinstance(scale, torch.Tensor) else scale
        return out

    @staticmethod
    @_layer.once("adapt")
    def backward(ctx, g):
        saved = list(ctx.saved_tensors)
        x, a, b, down = saved[:4]
        index = saved[4] if ctx.index else None
        scale = saved[-1] if ctx.scale is None else ctx.scale
        _decode.check_capture(x.device.index, "adapt")
        need_y, *need = ctx.needs_input_grad[:4]
        grads = (None, None, None)
        if any(need):
            with torch.cuda.device(x.device):  # (the engine's thread is on the gradient's device)
                grads = _backward(x, a, b, down, index, scale, g, need)
        return g if need_y else None, *grads, None, None


def _backward(x, a, b, down, index, scale, g, need):
    (n, n_in), n_out, rank = x.shape, b.shape[1], a.shape[1]
    dev = x.device
    a, b, count = _layer.dense(a), _layer.dense(b), a.shape[0]
    new = torch.empty if n else torch.zeros
    dx = new((n, n_in), dtype=x.dtype, device=dev) if need[0] else None
    da, db = (new(t.shape, dtype=x.dtype, device=dev) if want else None for t, want in ((a, need[1]), (b, need[2])))
    if n:
        x, g = _layer.rows_of(x), _layer.rows_of(g)
        nbytes = _layer.adapt_grad_workspace_size(n, n_in, n_out, rank, count)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        _layer.call_adapt_grad(
            _native.stream(dev), _layer.ADAPT_ABI_VERSION, _DTYPES[x.dtype], n, n_in, n_out, rank, count, 0,
            x.data_ptr(), x.stride(0), g.data_ptr(), g.stride(0), a.data_ptr(), b.data_ptr(), 0 if index is None else index.data_ptr(),
            *_scale_args(scale), down.data_ptr(), 0 if dx is None else dx.data_ptr(), n_in, 0 if da is None else da.data_ptr(),
            0 if db is None else db.data_ptr(), ws.data_ptr(), nbytes)
    return dx, da, db


def adapt(y, x, a, b, index=None, scale=1.0):
    """``y[n] + scale_i (x[n] a_i^T) b_i^T`` with i = ``index[n]``, as a new tensor.

    y: [N, n_out], a shared projection's output; x: [N, n_in], its input; a: [R,
    rank, n_in] and b: [R, n_out, rank], R adapters (all bf16 or all fp16); index:
    int32 or int64 [N], each row's adapter, in any order: negative for none (the row
    of y as it is), past the last one gives NaN, as x's gradient; None: the only adapter,
    for every row. scale: a number, or fp32 [R].

    Sums are fp32 in an order that the sizes alone fix; x a^T stays fp32, the result
    is rounded once. Rows of other adapters take no part in a row's sums, whatever
    they hold. An infinite x a^T (G b in the gradients) gives the formula's infinities;
    an infinity in b (and where the gradients multiply by them, in a, x or G)
    gives an infinity or NaN. Ranks 1 to 128, n_in and n_out multiples of 8
    up to 2^20, at most 2^20 rows and 65535 adapters; rows * max(n_in, n_out) below
    2^39, and for the gradient R * (n_in + n_out) below 2^30, that times rank below 2^35.

    Differentiable (once) in y, x, a and b. A backward pass that is captured into a HIP graph has
    its forward pass in the same capture, and no earlier, eager result that holds
    the graph of the same leaves is alive (where an input is such a leaf itself, that
    raises)."""
    made = _layer.calls().adapt(y, x, a, b, index, scale)
    if made is not None:  # a plain call
        return made
    if not x.is_cuda:
        raise RuntimeError(f"dan_amd.adapt runs on a gfx950 GPU only; got tensors on {x.device}")
    if x.device.index != torch._C._cuda_getDevice():
        with torch.cuda.device(x.device):
            return adapt(y, x, a, b, index, scale)
    dev, dt = x.device, x.dtype
    if x.dim() != 2 or y.dim() != 2 or x.shape[0] != y.shape[0] or dt not in (torch.bfloat16, torch.float16):
        raise ValueError(f"x must be [N, n_in] and y [N, n_out] in bf16 or fp16; got {tuple(x.shape)} {dt} and {tuple(y.shape)}")
    (n, n_in), n_out = x.shape, y.shape[1]
    if a.dim() != 3 or b.dim() != 3 or a.shape[2] != n_in or b.shape[1] != n_out or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2]:
        raise ValueError(f"a must be [R, rank, {n_in}] and b [R, {n_out}, rank]; got {tuple(a.shape)} and {tuple(b.shape)}")
    count, rank = a.shape[:2]
    if any(t.dtype != dt or t.device != dev for t in (y, a, b)):
        raise ValueError(f"y, a and b must be {dt} on {dev} as x; got {[(t.dtype, str(t.device)) for t in (y, a, b)]}")
    if n_in % 8 or n_out % 8 or not n_in or not n_out:
        raise ValueError(f"n_in {n_in} and n_out {n_out}: multiples of 8")
    if not 1 <= rank <= _layer.MAX_RANK or not count:
        raise ValueError(f"{count} adapters of rank {rank}: at least one, of rank 1 to {_layer.MAX_RANK}")
    if index is None:
        if count != 1:
            raise ValueError(f"{count} adapters need an index")
    elif index.shape != (n,) or index.dtype not in (torch.int32, torch.int64) or index.device != dev:
        raise ValueError(f"index must be int32 or int64 [{n}] on {dev}; got {index.dtype} {tuple(index.shape)} on {index.device}")
    else:
        if index.dtype == torch.int64:  # (a value past int32's stays past the last adapter, or negative)
            index = index.clamp(-1, count).int()
        index = index.contiguous()
    if isinstance(scale, torch.Tensor):
        if scale.shape != (count,) or scale.dtype != torch.float32 or scale.device != dev:
            raise ValueError(f"scale must be a number or fp32 [{count}] on {dev}; got {scale.dtype} {tuple(scale.shape)} on {scale.device}")
        scale = scale.contiguous()
    elif not math.isfinite(_native.f32(float(scale))):
        raise ValueError(f"scale {scale}: a finite number")
    else:
        scale = float(scale)
    inputs = [y, x, a, b] + ([scale] if isinstance(scale, torch.Tensor) else [])
    if has_tangent(*inputs):
        raise NotImplementedError("adapt has no forward-mode derivative")
    if torch.is_grad_enabled() and any(t.requires_grad for t in inputs):
        if isinstance(scale, torch.Tensor) and scale.requires_grad:
            raise NotImplementedError("adapt has no gradient of scale")
        return _Adapt.apply(y, x, a, b, index, scale)
    return _forward(y, x, a, b, index, scale, False)[0]


class AdaptedLinear(nn.Module):
    """A linear layer that many requests share, with ``adapters`` low-rank adapters
    beside it: ``forward(x, index)`` is ``adapt(base(x), x, a, b, index, scale)`` over
    x's rows. ``base``: an ``nn.Linear`` or an ``FP8Linear`` (which has no gradient of
    its input: with one, x that requires grad raises). The base's parameters are
    frozen; an adapter starts as nothing (b is zeros)."""

    def __init__(self, base, adapters, rank, scale=1.0):
        super().__init__()
        dtype = base.out_dtype if isinstance(base, FP8Linear) else base.weight.dtype
        new = dict(dtype=dtype, device=base.weight.device)
        self.base = base.requires_grad_(False)
        self.a = nn.Parameter(torch.randn(adapters, rank, base.in_features, **new) * base.in_features ** -0.5)
        self.b = nn.Parameter(torch.zeros(adapters, base.out_features, rank, **new))
        self.scale = float(scale)

    def forward(self, x, index=None):
        if isinstance(self.base, FP8Linear) and x.requires_grad and torch.is_grad_enabled():
            raise NotImplementedError("FP8Linear has no gradient of its input")
        rows = x.reshape(-1, x.shape[-1])
        return adapt(self.base(rows), rows, self.a, self.b, index, self.scale).view(*x.shape[:-1], self.base.out_features)
