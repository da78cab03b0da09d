"""The gradient of tree attention (include/dan_tree_grad.h): its argument
structure, its tables, and the autograd function behind
``dan_amd.attention.attend_train``."""
import ctypes
import functools

import numpy as np
import torch

from . import _decode, _layer, _native

_i32, _i64, _f32, _vp = ctypes.c_int32, ctypes.c_int64, ctypes.c_float, ctypes.c_void_p

GRAD_ABI_VERSION = 1
TILE = 32  # rows or keys of one step


class DanTreeGradArgs(ctypes.Structure):
    _fields_ = [("abi_version", _i32), ("dtype", _i32), ("num_heads", _i32), ("num_kv_heads", _i32), ("head_dim", _i32),
                ("num_tokens", _i32), ("scale", _f32), ("key_rows", _i32),
                ("q", _vp), ("q_stride_tok", _i64), ("q_stride_head", _i64),
                ("k", _vp), ("k_stride_tok", _i64), ("k_stride_head", _i64),
                ("v", _vp), ("v_stride_tok", _i64), ("v_stride_head", _i64),
                ("out", _vp), ("o_stride_tok", _i64), ("o_stride_head", _i64),
                ("grad", _vp), ("g_stride_tok", _i64), ("g_stride_head", _i64),
                ("lse", _vp),
                ("dq", _vp), ("dq_stride_tok", _i64), ("dq_stride_head", _i64),
                ("dk", _vp), ("dk_stride_tok", _i64), ("dk_stride_head", _i64),
                ("dv", _vp), ("dv_stride_tok", _i64), ("dv_stride_head", _i64),
                ("key_units", _vp), ("num_key_units", _i32), ("query_units", _vp), ("num_query_units", _i32),
                ("row_lo", _vp), ("row_end", _vp), ("pasts", _vp), ("num_pasts", _i32),
                ("workspace", _vp), ("workspace_bytes", _i64), ("key_splits", _i32), ("reserved", _i32)]


EXPORTS = ("dan_tree_attn_fwd_lse", "dan_tree_attn_bwd", "dan_tree_grad_key_rows", "dan_tree_grad_query_rows",
           "dan_tree_grad_workspace_size", "dan_tree_grad_abi_version")

call_backward = _native.Entry("dan_tree_attn_bwd", DanTreeGradArgs)


def templates(segments, q, k, v, layer, scale, plan_args):
    """What the host module's ``attend`` takes beside q, k and v: the two argument structures as bytes, their workspaces' sizes, whether a row
    is in no segment, and the tensors that they point to."""
    from . import attention as A

    args, pasts_host, plan = plan_args
    (h, n, d), hkv = q.shape, k.shape[0]
    t = tables(segments, plan, h, hkv, d, A._num_cus(q.device))
    code, nbytes, back = A._DTYPES[q.dtype], _native.workspace_size(hkv, d, plan.vt_cols) if plan.num_work else 0, workspace_size(h, hkv, d, n, t.key_splits)
    past = plan.past_tables[layer][0]
    device_tables = args[3]
    units, sched_off = (device_tables[5].data_ptr(), device_tables[6].data_ptr()) if plan.num_work else (0, 0)
    num_segments, num_pasts, num_work, tile_q, vt_cols, slots = args[5][:6]
    forward = call_forward_lse.pack(
        _native.ABI_VERSION, code, code, code, h, hkv, d, n, _native.f32(args[6]), *[0] * 12, 0, 0, 0, device_tables[0].data_ptr(), num_segments,
        past.data_ptr(), num_pasts, device_tables[1].data_ptr(), num_work, device_tables[2].data_ptr(), tile_q, vt_cols, device_tables[3].data_ptr(),
        0, 0, _native.PHASES_ALL, units, sched_off, slots, 0, 0 if pasts_host is None else pasts_host.data_ptr(), A._layout(h, hkv, d)[0] // tile_q, 0, 0, 0)
    backward = call_backward.pack(
        GRAD_ABI_VERSION, code, h, hkv, d, n, _native.f32(args[6]), t.key_rows, *[0] * 15, 0, *[0] * 9, t.keys, t.num_keys, t.queries, t.num_queries,
        t.row_lo, t.row_end, past.data_ptr(), num_pasts, 0, 0, t.key_splits, 0)
    pasts = tuple(x for entry in plan.past_dicts for x in entry[layer][:2])
    # (the prefix's rows as the kernels read them, where they had to be copied, are behind past_tables)
    refs = tuple(x for x in plan.past_tables[layer][1][0] if isinstance(x, torch.Tensor))
    return (forward, nbytes, backward, back, not t.covered, (t.blob, past, *device_tables, *refs), pasts), (t, pasts_host)


class _ForwardLse(_native.Entry):
    """``dan_tree_attn_fwd_lse``: the forward entry with one more argument."""

    def __call__(self, lse, stream, *fields):
        if self.fn is None:
            fn = _native.load()[self.name]
            fn.argtypes, fn.restype = [ctypes.c_char_p, _vp, _vp], ctypes.c_int
            self.fn = fn
        rc = self.fn(self.pack(*fields), lse, stream)
        if rc != _native.OK:
            raise RuntimeError(f"{self.name} failed (status {rc}): {_native.last_error(_native.load())}")


call_forward_lse = _ForwardLse("dan_tree_attn_fwd_lse", _native.DanTreeAttnArgs)


@functools.lru_cache(maxsize=None)
def _rows(h, hkv, d, small):
    """(keys of a key unit, rows of a query unit) of a head layout."""
    lib = _native.load()
    return lib["dan_tree_grad_key_rows"](d, int(small)), lib["dan_tree_grad_query_rows"](h, hkv, d)


@functools.lru_cache(maxsize=256)
def workspace_size(h, hkv, d, n, splits=1):
    fn = _native.load()["dan_tree_grad_workspace_size"]
    fn.argtypes, fn.restype = [_i32] * 5, _i64
    return fn(h, hkv, d, n, splits)


def choose_units(lengths, h, hkv, d, num_cus):
    """(keys of a key unit, parts of a kv head's heads) of segments of `lengths` rows.

    Larger units read less of Q and G, smaller ones and parts of the heads fill the chip, with the units of dQ behind them in
    the same launch: of a number of parts that divides the heads evenly and gives up to one work group a compute unit, while
    the longest unit keeps 16 steps (the parts are written and read again in fp32). Forward and backward pass, us: 8192 rows,
    32/8 heads x 128, units of 128 / 64 keys 2264 / 2293, 3413 rows in four requests 251 / 239; 2000 rows, 16/2 heads x 128, units of 64
    keys in 1 / 2 / 4 / 8 parts 260 / 175 / 170 / 205; 4000 rows, 16/4 x 128, 1 / 2 parts 355 / 414; 4099 rows in five requests, 16/2 x 256,
    1 / 2 / 4 parts 371 / 372 / 409."""
    whole, small = (int((-(-lengths // _rows(h, hkv, d, x)[0])).sum()) * hkv for x in (False, True))
    if whole >= num_cus or not small:
        return _rows(h, hkv, d, False)[0], 1
    rep, at_once = h // hkv, 2 if d == 256 else 4  # tiles of a step
    tiles = -(-int(lengths.max()) // TILE) * rep
    parts = [s for s in range(1, rep + 1) if rep % s == 0 and small * s <= num_cus and (s == 1 or tiles >= 16 * at_once * s)]
    return _rows(h, hkv, d, True)[0], max(parts, default=1)


def build_units(segs, spans, num_tokens, key_rows, query_rows):
    """The backward pass's tables: (key units int32 [K, 8], query units int32
    [Q, 8], row_lo int32 [N], row_end int32 [N]) as DanTreeGradArgs takes them.
    ``segs``: rows whose first fields are (start, n, trunk, past_len, past
    index); ``spans``: each segment's branches (a, b) in packed rows. Units are
    sorted by the steps they take, longest first: the hardware starts work
    groups in order."""
    row_lo, row_end = np.zeros(num_tokens, np.int32), np.zeros(num_tokens, np.int32)
    taken = np.zeros(num_tokens, bool)
    keys, queries = [], []
    for seg, branches in zip(segs, spans):
        start, n, trunk, past, pidx = (int(x) for x in seg[:5])
        if taken[start:start + n].any():
            raise ValueError(f"segment at row {start}: its rows belong to another segment, too")
        taken[start:start + n] = True
        row_end[start:start + trunk] = n
        for a, b in branches:
            row_lo[a:b], row_end[a:b] = a - start, b - start
        at = np.arange(0, n, key_rows)
        end = np.minimum(at + key_rows, n)
        q_end = np.array([row_end[start + a:start + b].max() for a, b in zip(at, end)])
        u = np.zeros((len(at), 9), np.int64)
        u[:, 0], u[:, 1], u[:, 2], u[:, 3], u[:, 4], u[:, 5] = start, n, trunk, at, end - at, q_end
        u[:, 8] = -(-(q_end - at) // TILE)
        keys.append(u)
        at = np.arange(0, n, query_rows)
        end = np.minimum(at + query_rows, n)
        mixed = end > trunk  # holds branch rows
        b0 = np.where(mixed, row_lo[start + np.minimum(np.maximum(at, trunk), n - 1)], 0)
        u = np.zeros((len(at), 9), np.int64)
        u[:, 0], u[:, 1], u[:, 2], u[:, 3], u[:, 4], u[:, 5], u[:, 6], u[:, 7] = start, n, trunk, at, end - at, past, pidx, b0
        u[:, 8] = -(-past // TILE) + -(-np.minimum(trunk, end) // TILE) + np.where(mixed, -(-(end - b0) // TILE), 0)
        queries.append(u)
    out = []
    for units in (keys, queries):
        u = np.concatenate(units) if units else np.zeros((0, 9), np.int64)
        out.append(u[np.argsort(-u[:, 8], kind="stable"), :8].astype(np.int32))
    return (*out, row_lo, row_end, bool(taken.all()))


class Tables:
    """Device copy of ``build_units``' arrays for one head layout."""

    def __init__(self, segments, plan, h, hkv, d, num_cus):
        from .plan import _upload

        self.device, n = plan.device, plan.num_tokens
        spans = [s.branches for s in segments]
        rows = _rows(h, hkv, d, False)[1]
        self.key_rows, self.key_splits = choose_units(plan.segs[:, 1], h, hkv, d, num_cus)
        keys, queries, row_lo, row_end, self.covered = build_units(plan.segs, spans, n, self.key_rows, rows)
        self.num_keys, self.num_queries = len(keys), len(queries)
        self.blob = _upload(np.concatenate([keys.ravel(), queries.ravel(), row_lo, row_end]), self.device)
        at = self.blob.data_ptr()
        self.keys, self.queries = at, at + keys.nbytes
        self.row_lo = self.queries + queries.nbytes
        self.row_end = self.row_lo + row_lo.nbytes
        plan.make_spare(ctypes.sizeof(_native.DanPastDesc) * max(len(plan.past_dicts), 1))
        plan.fills()


def tables(segments, plan, h, hkv, d, num_cus):
    """The batch's tables, kept on its plan with the forward pass's."""
    if (h, hkv, d) not in plan.grad_tables:
        plan.grad_tables[h, hkv, d] = Tables(segments, plan, h, hkv, d, num_cus)
    return plan.grad_tables[h, hkv, d]


BEFORE_CAPTURE = "attend_train: run the batch once before a capture (its tables are uploaded then)"


def planned(plan, layer):
    """Whether a first call of ``layer`` finds the forward pass's tables on the device. What a capture uploads or copies is there only
    once the graph has run: tables kept from it would be read before."""
    from . import attention as A

    if plan is None:
        return False
    if layer in plan.past_tables:
        return plan.past_hosts[layer] is not None or layer in plan.past_uploaded
    return len(plan.past_dicts) <= _native.INLINE_PASTS and all(A._in_place(x) for entry in plan.past_dicts for x in entry[layer][:2])


def capturable(plan, layer, layout):
    """Whether a first training call of ``layer`` and a head layout (heads, kv heads, head_dim) does, and finds the backward pass's, and a
    prefix table that shares no memory with the graph's other calls."""
    return (planned(plan, layer) and layout in plan.grad_tables
            and (not plan.past_dicts or layer in plan.past_tables or layer in plan.spare))


def attend(q, k, v, segments, layer, scale):
    """The differentiable call: through the host module where q, k and v are read in place."""
    from . import attention as A

    plan = getattr(segments, "tile_plan", None)
    if plan is None or plan.num_tokens != q.shape[1] or plan.device != q.device:
        plan = None
    key = (layer, *q.shape[::2], k.shape[0], q.dtype, scale)
    made = None if plan is None else plan.train_calls.get(key)
    if made is None:
        if q.is_cuda and torch.cuda.is_current_stream_capturing() and not capturable(plan, layer, (q.shape[0], k.shape[0], q.shape[-1])):
            raise RuntimeError(BEFORE_CAPTURE)
        with torch.no_grad():
            plan_args = A._call_args(q, k, v, segments, layer, scale, None, _native.PHASES_ALL, False, upload=False)
        made, plan = templates(segments, q, k, v, layer, scale, plan_args), plan_args[2]
        plan.train_calls[key] = made
    call, _ = made
    plan.order(q.device)  # (behind what was uploaded on any stream: for an earlier call, another layer, or by ``attend``)
    out = _layer.calls().attend(q, k, v, *call)
    return TreeAttention.apply(q, k, v, segments, layer, scale) if out is None else out


class TreeAttention(torch.autograd.Function):
    """Tree attention with its gradient: q [H, N, D], k and v [Hkv, N, D] -> [H, N, D]."""

    @staticmethod
    def forward(ctx, q, k, v, segments, layer, scale):
        from . import attention as A

        args, pasts_host, plan = A._call_args(q, k, v, segments, layer, scale, None, _native.PHASES_ALL, False, upload=False)
        (h, n, d), hkv = q.shape, k.shape[0]
        t = tables(segments, plan, h, hkv, d, A._num_cus(q.device))
        lse = torch.empty((h, n), dtype=torch.float32, device=q.device)
        out = A._launch_tree_attn(*args, None, pasts_host, launch=functools.partial(call_forward_lse, lse.data_ptr()), zero=not t.covered)
        # The prefix's own tensors are saved, too: what the backward pass reads has to be what the forward pass read.
        pasts = [x for entry in plan.past_dicts for x in entry[layer][:2]]
        ctx.save_for_backward(q, k, v, out, lse, *pasts)
        ctx.tables, ctx.past = t, plan.past_tables[layer]
        ctx.num_pasts, ctx.scale = len(plan.past_dicts), args[6]
        return out

    @staticmethod
    @_layer.once("attend_train")
    def backward(ctx, grad):
        q, k, v, out, lse = ctx.saved_tensors[:5]
        _decode.check_capture(q.device.index, "attend_train")
        if torch._C._cuda_getDevice() != q.device.index:  # (the engine's thread is on the gradient's device)
            with torch.cuda.device(q.device):
                return *_backward(ctx, q, k, v, out, lse, grad), None, None, None
        return *_backward(ctx, q, k, v, out, lse, grad), None, None, None


def _backward(ctx, q, k, v, out, lse, grad):
    from . import attention as A

    (h, n, d), hkv, t = q.shape, k.shape[0], ctx.tables
    new = torch.empty if t.covered else torch.zeros  # rows of no segment have no gradient
    dq, dk, dv = (new((n, x.shape[0], d), dtype=q.dtype, device=q.device).transpose(0, 1) for x in (q, k, v))
    if n:
        q, k, v, grad = (A._kernel_view(x) for x in (q, k, v, grad))
        nbytes = workspace_size(h, hkv, d, n, t.key_splits)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
        rows = [f for x in (q, k, v, out, grad) for f in (x.data_ptr(), x.stride(1), x.stride(0))]
        grads = [f for x in (dq, dk, dv) for f in (x.data_ptr(), x.stride(1), x.stride(0))]
        call_backward(_native.stream(q.device), GRAD_ABI_VERSION, A._DTYPES[q.dtype], h, hkv, d, n, _native.f32(ctx.scale), t.key_rows,
                      *rows, lse.data_ptr(), *grads, t.keys, t.num_keys, t.queries, t.num_queries, t.row_lo, t.row_end,
                      ctx.past[0].data_ptr(), ctx.num_pasts, ws.data_ptr(), nbytes, t.key_splits, 0)
    return tuple(x if need else None for x, need in zip((dq, dk, dv), ctx.needs_input_grad))
