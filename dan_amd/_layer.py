"""ctypes binding of include/dan_norm.h and include/dan_adapt.h: what a decoder
layer runs in front of and beside its projections, in the library that
``_native`` loads."""
import ctypes
import functools

from . import _decode, _native

_i32, _i64, _f32, _vp = ctypes.c_int32, ctypes.c_int64, ctypes.c_float, ctypes.c_void_p

NORM_ABI_VERSION = 1
MAX_COLS = 16384  # DAN_NORM_MAX_COLS
NORM_RMS, NORM_ZERO_CENTERED = 0, 1
ADAPT_ABI_VERSION = 1
MAX_RANK = 128  # DAN_ADAPT_MAX_RANK


class DanNormArgs(ctypes.Structure):
    _fields_ = [("abi_version", _i32), ("dtype", _i32), ("rows", _i32), ("cols", _i32), ("norm", _i32), ("layout", _i32),
                ("eps", _f32), ("reserved", _i32), ("x", _vp), ("x_stride", _i64), ("residual", _vp), ("residual_stride", _i64),
                ("weight", _vp), ("stream", _vp), ("stream_stride", _i64), ("out", _vp), ("out_stride", _i64),
                ("codes", _vp), ("scale", _vp), ("rstd", _vp)]


class DanNormGradArgs(ctypes.Structure):
    _fields_ = [("abi_version", _i32), ("dtype", _i32), ("rows", _i32), ("cols", _i32), ("norm", _i32), ("reserved", _i32),
                ("s", _vp), ("s_stride", _i64), ("weight", _vp), ("rstd", _vp), ("g", _vp), ("g_stride", _i64),
                ("g_stream", _vp), ("g_stream_stride", _i64), ("ds", _vp), ("ds_stride", _i64), ("dw", _vp),
                ("workspace", _vp), ("workspace_bytes", _i64)]


class DanAdaptArgs(ctypes.Structure):
    _fields_ = [("abi_version", _i32), ("dtype", _i32), ("rows", _i32), ("n_in", _i32), ("n_out", _i32), ("rank", _i32),
                ("adapters", _i32), ("reserved", _i32), ("x", _vp), ("x_stride", _i64), ("y", _vp), ("y_stride", _i64),
                ("a", _vp), ("b", _vp), ("index", _vp), ("scale", _vp), ("scale_value", _f32), ("out", _vp), ("out_stride", _i64),
                ("down", _vp), ("workspace", _vp), ("workspace_bytes", _i64)]


class DanAdaptGradArgs(ctypes.Structure):
    _fields_ = [("abi_version", _i32), ("dtype", _i32), ("rows", _i32), ("n_in", _i32), ("n_out", _i32), ("rank", _i32),
                ("adapters", _i32), ("reserved", _i32), ("x", _vp), ("x_stride", _i64), ("g", _vp), ("g_stride", _i64),
                ("a", _vp), ("b", _vp), ("index", _vp), ("scale", _vp), ("scale_value", _f32), ("down", _vp),
                ("dx", _vp), ("dx_stride", _i64), ("da", _vp), ("db", _vp), ("workspace", _vp), ("workspace_bytes", _i64)]


EXPORTS = ("dan_add_norm", "dan_add_norm_grad", "dan_norm_grad_workspace_size", "dan_norm_abi_version",
           "dan_adapt", "dan_adapt_grad", "dan_adapt_workspace_size", "dan_adapt_grad_workspace_size", "dan_adapt_abi_version")

call_norm = _native.Entry("dan_add_norm", DanNormArgs)
call_norm_grad = _native.Entry("dan_add_norm_grad", DanNormGradArgs)
call_adapt = _native.Entry("dan_adapt", DanAdaptArgs)
call_adapt_grad = _native.Entry("dan_adapt_grad", DanAdaptGradArgs)


@functools.lru_cache(maxsize=None)
def calls():
    """The host module of the plain calls (csrc/layer_calls.cpp), bound to the library. Like the
    library it has to be there: there is no fallback for a missing one."""
    return _decode.load_calls("_layer_calls", (
        "dan_add_norm", "dan_add_norm_grad", "dan_norm_grad_workspace_size", "dan_adapt", "dan_adapt_grad", "dan_adapt_workspace_size",
        "dan_adapt_grad_workspace_size", "dan_tree_attn_fwd_lse", "dan_tree_attn_bwd", "dan_fp8_tiled_bytes", "dan_tree_attn_last_error"))


def _sized(name, restype, count):
    fn = _native.load()[name]
    fn.argtypes, fn.restype = [_i32] * count, restype
    return fn


@functools.lru_cache(maxsize=1024)
def norm_grad_workspace_size(rows, cols):
    return _sized("dan_norm_grad_workspace_size", _i64, 2)(rows, cols)


@functools.lru_cache(maxsize=1024)
def adapt_workspace_size(rows, n_in, rank, adapters):
    return _sized("dan_adapt_workspace_size", _i64, 4)(rows, n_in, rank, adapters)


@functools.lru_cache(maxsize=1024)
def adapt_grad_workspace_size(rows, n_in, n_out, rank, adapters):
    return _sized("dan_adapt_grad_workspace_size", _i64, 5)(rows, n_in, n_out, rank, adapters)


def once(name):
    """Marks a backward as differentiable once, as the host module's are: where a second derivative is being recorded (by
    the gradients or by a saved input, which torch's own decorator does not look at), taking it raises."""
    def mark(backward):
        @functools.wraps(backward)
        def run(ctx, *grads):
            import torch

            again = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (*grads, *ctx.saved_tensors))
            with torch.no_grad():
                out = backward(ctx, *grads)
            if not again:
                return out
            new = [i for i, t in enumerate(out) if t is not None and all(t is not g for g in grads)]
            out = list(out)
            if new:
                late = torch._C._functions.DelayedError(f"{name} is differentiable once", len(new))
                for i, t in zip(new, late(*[out[i].detach().requires_grad_() for i in new])):
                    out[i] = t
            return tuple(out)
        return run
    return mark


def rows_of(t):
    """A 2-D tensor that the kernels read in place (unit stride, rows 16-byte aligned), or a new copy of it."""
    s0, s1 = t.stride()
    if (s1 == 1 or t.shape[1] == 1) and not (t.data_ptr() | s0 * t.element_size()) & 15:
        return t
    import torch

    return torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)


def dense(t):
    """A contiguous, 16-byte aligned tensor."""
    return t if t.is_contiguous() and not t.data_ptr() & 15 else t.clone(memory_format=_contiguous())


def _contiguous():
    import torch

    return torch.contiguous_format
