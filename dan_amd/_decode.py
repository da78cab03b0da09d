"""ctypes binding of include/dan_paged.h and include/dan_readout.h: the argument
structures and entry points of a decode step's operators, in the library that
``_native`` loads."""
import ctypes
import functools
import importlib.machinery
import importlib.util
import os

from . import _native

_i32, _i64, _f32, _vp = ctypes.c_int32, ctypes.c_int64, ctypes.c_float, ctypes.c_void_p

PAGED_ABI_VERSION = 1
KEY_BLOCK = 16  # DAN_PAGED_KEY_BLOCK
READOUT_ABI_VERSION = 2
MAX_TOP, MAX_TOP_VOCAB = 32, 524288  # DAN_READOUT_MAX_TOP, DAN_READOUT_MAX_TOP_VOCAB


class DanPagedAppendArgs(ctypes.Structure):
    _fields_ = [("abi_version", _i32), ("dtype", _i32), ("cache_dtype", _i32), ("table_dtype", _i32), ("num_tokens", _i32),
                ("num_heads", _i32), ("num_kv_heads", _i32), ("head_dim", _i32), ("rotary_dim", _i32), ("norm", _i32),
                ("page_size", _i32), ("num_pages", _i32), ("table_width", _i32), ("num_seqs", _i32), ("num_rope_rows", _i32),
                ("eps", _f32),
                ("q", _vp), ("q_stride_tok", _i64), ("q_stride_head", _i64),
                ("k", _vp), ("k_stride_tok", _i64), ("k_stride_head", _i64),
                ("v", _vp), ("v_stride_tok", _i64), ("v_stride_head", _i64),
                ("cos", _vp), ("sin", _vp), ("cs_stride_tok", _i64),
                ("q_norm_weight", _vp), ("k_norm_weight", _vp),
                ("q_out", _vp), ("qo_stride_tok", _i64), ("qo_stride_head", _i64),
                ("k_cache", _vp), ("kc_stride_page", _i64), ("kc_stride_head", _i64), ("kc_stride_tok", _i64),
                ("v_cache", _vp), ("vc_stride_page", _i64), ("vc_stride_head", _i64), ("vc_stride_tok", _i64),
                ("k_scale", _vp), ("v_scale", _vp), ("table", _vp), ("table_stride", _i64),
                ("places", _vp), ("seqs", _vp), ("rope_rows", _vp)]


class DanPagedAttnArgs(ctypes.Structure):
    _fields_ = [("abi_version", _i32), ("dtype", _i32), ("cache_dtype", _i32), ("num_seqs", _i32),
                ("num_heads", _i32), ("num_kv_heads", _i32), ("head_dim", _i32),
                ("page_size", _i32), ("num_pages", _i32), ("table_width", _i32), ("max_len", _i32), ("scale", _f32),
                ("q", _vp), ("q_stride_seq", _i64), ("q_stride_head", _i64),
                ("out", _vp), ("o_stride_seq", _i64), ("o_stride_head", _i64), ("lse", _vp),
                ("k_cache", _vp), ("kc_stride_page", _i64), ("kc_stride_head", _i64), ("kc_stride_tok", _i64),
                ("v_cache", _vp), ("vc_stride_page", _i64), ("vc_stride_head", _i64), ("vc_stride_tok", _i64),
                ("k_scale", _vp), ("v_scale", _vp), ("table", _vp), ("table_stride", _i64), ("lens", _vp),
                ("workspace", _vp), ("workspace_bytes", _i64)]


class DanLogprobsArgs(ctypes.Structure):
    _fields_ = [("abi_version", _i32), ("dtype", _i32), ("rows", _i32), ("vocab", _i32), ("labels", _i32), ("top", _i32),
                ("logits", _vp), ("logits_stride", _i64), ("tokens", _vp), ("tokens_stride", _i64),
                ("logprobs", _vp), ("logsumexp", _vp), ("entropy", _vp), ("top_logprobs", _vp), ("top_ids", _vp),
                ("workspace", _vp), ("workspace_bytes", _i64), ("logsumexp_rest", _vp)]


class DanLogprobsGradArgs(ctypes.Structure):
    _fields_ = [("abi_version", _i32), ("dtype", _i32), ("rows", _i32), ("vocab", _i32), ("labels", _i32), ("top", _i32),
                ("logits", _vp), ("logits_stride", _i64), ("tokens", _vp), ("tokens_stride", _i64),
                ("logsumexp", _vp), ("entropy", _vp), ("top_ids", _vp),
                ("g_logprobs", _vp), ("g_logsumexp", _vp), ("g_entropy", _vp), ("g_top", _vp),
                ("grad", _vp), ("grad_stride", _i64), ("logsumexp_rest", _vp)]


EXPORTS = ("dan_paged_append", "dan_paged_attn", "dan_paged_attn_workspace_size", "dan_paged_abi_version",
           "dan_logprobs_fwd", "dan_logprobs_bwd", "dan_logprobs_workspace_size", "dan_readout_abi_version")

call_append = _native.Entry("dan_paged_append", DanPagedAppendArgs)
call_paged_attn = _native.Entry("dan_paged_attn", DanPagedAttnArgs)
call_logprobs = _native.Entry("dan_logprobs_fwd", DanLogprobsArgs)
call_logprobs_grad = _native.Entry("dan_logprobs_bwd", DanLogprobsGradArgs)


def _sized(name, *types):
    fn = _native.load()[name]
    fn.argtypes, fn.restype = list(types), _i64
    return fn


@functools.lru_cache(maxsize=1024)
def paged_attn_workspace_size(device_index, cache_dtype, num_seqs, num_heads, num_kv_heads, head_dim, max_len):
    """Bytes of workspace of one attention call on the (current) device (0: none; -1: invalid arguments)."""
    return _sized("dan_paged_attn_workspace_size", *[_i32] * 6)(cache_dtype, num_seqs, num_heads, num_kv_heads, head_dim, max_len)


@functools.lru_cache(maxsize=1024)
def logprobs_workspace_size(dtype, rows, vocab, top):
    """Bytes of workspace of one forward call (0: invalid arguments)."""
    return _sized("dan_logprobs_workspace_size", *[_i32] * 4)(dtype, rows, vocab, top)


@functools.lru_cache(maxsize=None)
def calls():
    """The host module of the plain calls (csrc/decode_calls.cpp), bound to the library. Like the
    library it has to be there: there is no fallback for a missing one."""
    return load_calls("_decode_calls", ("dan_paged_append", "dan_paged_attn", "dan_paged_attn_workspace_size", "dan_logprobs_fwd", "dan_logprobs_bwd",
                                        "dan_logprobs_workspace_size", "dan_tree_attn_last_error"))


def load_calls(name, entries):
    """The host module ``name``, bound to the library's ``entries``."""
    lib, path = _native.load(), os.path.join(_native.LIB_DIR, name + ".so")
    if not os.path.exists(path):
        raise RuntimeError(f"{path} is not built; run __graft_entry__.build()")
    loader = importlib.machinery.ExtensionFileLoader(name, path)
    module = importlib.util.module_from_spec(importlib.util.spec_from_loader(name, loader))
    loader.exec_module(module)
    module.bind(*(ctypes.cast(lib[entry], ctypes.c_void_p).value for entry in entries))
    return module


_host = calls


def check_capture(device_index, name="token_logprobs"):
    """Inside a backward of ``name``: refuses to run in a capture that torch's engine would make the stream of an eager graph wait for."""
    _host().check_capture(device_index, name)
