"""Log probabilities of given tokens on gfx950, with their distribution's
logsumexp, entropy and top tokens, and the gradient of the logits.

dan answers with the softmax over a read row's label logits (dan/readout.py:13-17,
dan/models/llama.py:163-165). ``token_logprobs`` takes the whole row: each
label's (or any given token's) log probability among the whole vocabulary, how
sure the row is, and what it would rather say. Training through the read path
(dan/tuning.py:82-133) needs its gradient.

There is no CPU path: CPU tensors raise (oracle/readout.py is the test oracle).
"""
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import _decode, _native
from .attention import _DTYPES, has_tangent


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor  # fp32, of the shape of ``tokens``
    logsumexp: torch.Tensor  # fp32 [N]
    entropy: Optional[torch.Tensor]  # fp32 [N], in nats
    top_logprobs: Optional[torch.Tensor]  # fp32 [N, top]
    top_ids: Optional[torch.Tensor]  # int64 [N, top]


def _forward(logits, tokens, top, entropy, rest=None):
    """The five outputs; what rounding took from logsumexp into ``rest`` (fp32 [N])."""
    n, vocab = logits.shape
    dev, dtype = logits.device, _DTYPES[logits.dtype]
    labels = tokens.shape[1] if tokens.dim() == 2 else 1
    logprobs, lse = torch.empty(tokens.shape, dtype=torch.float32, device=dev), torch.empty(n, dtype=torch.float32, device=dev)
    ent = top_lp = top_ids = None
    ent_p = lp_p = id_p = 0
    if entropy:
        ent = torch.empty(n, dtype=torch.float32, device=dev)
        ent_p = ent.data_ptr()
    if top:
        top_lp = torch.empty((n, top), dtype=torch.float32, device=dev)
        top_ids = torch.empty((n, top), dtype=torch.int64, device=dev)
        lp_p, id_p = top_lp.data_ptr(), top_ids.data_ptr()
    need = _decode.logprobs_workspace_size(dtype, n, vocab, top)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    _decode.call_logprobs(
        _native.stream(dev), _decode.READOUT_ABI_VERSION, dtype, n, vocab, labels, top, logits.data_ptr(), logits.stride(0),
        tokens.data_ptr(), tokens.stride(0), logprobs.data_ptr(), lse.data_ptr(), ent_p, lp_p, id_p, ws.data_ptr(), need,
        0 if rest is None else rest.data_ptr())
    return logprobs, lse, ent, top_lp, top_ids


class _Logprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top, entropy):
        rest = torch.empty(logits.shape[0], dtype=torch.float32, device=logits.device)
        logprobs, lse, ent, top_lp, top_ids = _forward(logits, tokens, top, entropy, rest)
        ctx.save_for_backward(logits, tokens, lse, rest, ent, top_ids)
        ctx.top = top
        ctx.set_materialize_grads(False)
        if top:
            ctx.mark_non_differentiable(top_ids)
        return logprobs, lse, ent, top_lp, top_ids

    @staticmethod
    @once_differentiable
    def backward(ctx, g_logprobs, g_lse, g_entropy, g_top, _g_ids):
        saved = ctx.saved_tensors
        logits = saved[0]
        _decode.check_capture(logits.device.index)
        if torch._C._cuda_getDevice() != logits.device.index:  # (the engine's thread is on the gradients' device)
            with torch.cuda.device(logits.device):
                return _backward(*saved, ctx.top, g_logprobs, g_lse, g_entropy, g_top), None, None, None
        return _backward(*saved, ctx.top, g_logprobs, g_lse, g_entropy, g_top), None, None, None


def _backward(logits, tokens, lse, rest, ent, top_ids, top, *grads):
    grads = [g if g is None or g.is_contiguous() else g.contiguous() for g in grads]
    n, vocab = logits.shape
    dtype = logits.dtype
    grad = torch.empty((n, vocab), dtype=dtype, device=logits.device)
    g_logp, g_lse, g_ent, g_top = (0 if g is None else g.data_ptr() for g in grads)
    _decode.call_logprobs_grad(
        _native.stream(logits.device), _decode.READOUT_ABI_VERSION, _DTYPES[dtype], n, vocab, tokens.shape[1] if tokens.dim() == 2 else 1, top,
        logits.data_ptr(), logits.stride(0), tokens.data_ptr(), tokens.stride(0), lse.data_ptr(), 0 if ent is None else ent.data_ptr(),
        0 if top_ids is None else top_ids.data_ptr(), g_logp, g_lse, g_ent, g_top, grad.data_ptr(), vocab, rest.data_ptr())
    return grad


def token_logprobs(logits, tokens, *, top=0, entropy=False):
    """logits: [N, V] (bf16, fp16 or fp32; any row stride, unit stride along a
    row); tokens: integers [N], or [N, L] (a row's labels). Returns
    ``TokenLogprobs``:

    - ``logprobs``: ``logits[n, t] - logsumexp[n]`` for each given token, fp32, of
      the shape of ``tokens``. A negative token is padding and gives 0 (and has no
      gradient); one past the vocabulary gives NaN.
    - ``logsumexp``: fp32 [N].
    - ``entropy`` (with ``entropy=True``): fp32 [N], in nats.
    - ``top_logprobs``, ``top_ids`` (with ``top`` > 0, at most 32 and V, for V up
      to 524288): the most probable tokens by falling logit, equal ones by
      rising id.

    Logits of -inf (masked tokens) have probability 0. A row whose every logit is
    -inf has logsumexp and log probabilities -inf, entropy 0 and no gradient; a row
    that holds NaN or +inf gives NaN throughout, its ``top_ids`` then being some
    ids of the row. Sums are fp32, in an order that the sizes alone fix.

    Where ``logits`` requires grad, every output but ``top_ids`` is
    differentiable (once): the gradient has the logits' dtype, computed in fp32
    and rounded once; a token given twice adds up. A backward that is captured into
    a HIP graph must have its forward in the same capture, and no earlier, eager
    result that holds the graph of the same leaves may be alive (torch's engine would join
    the two streams): where ``logits`` is such a leaf itself, that raises."""
    made = _decode.calls().logprobs(logits, tokens, top, entropy)
    if made is not None:  # a plain call
        return TokenLogprobs._make(made)
    dev = logits.device
    if not logits.is_cuda:
        raise RuntimeError(f"dan_amd.token_logprobs runs on a gfx950 GPU only; got tensors on {dev}")
    if dev.index != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            return token_logprobs(logits, tokens, top=top, entropy=entropy)
    if logits.dim() != 2 or logits.shape[1] == 0 or logits.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError(f"logits must be [N, V] in bf16, fp16 or fp32; got {tuple(logits.shape)} {logits.dtype}")
    n, vocab = logits.shape
    if tokens.dim() not in (1, 2) or tokens.shape[0] != n or tokens.dtype not in (torch.int64, torch.int32) or tokens.device != dev:
        raise ValueError(f"tokens must be int64 or int32 [{n}] or [{n}, L] on {dev}; got {tokens.dtype} {tuple(tokens.shape)} on {tokens.device}")
    if top != int(top):
        raise ValueError(f"top {top}: a whole number")
    if not 0 <= top <= min(vocab, _decode.MAX_TOP) or (top and vocab > _decode.MAX_TOP_VOCAB):
        raise ValueError(f"top {top}: at most {_decode.MAX_TOP} and the vocabulary's {vocab}, for at most {_decode.MAX_TOP_VOCAB} values")
    if has_tangent(logits):
        raise NotImplementedError("token_logprobs has no forward-mode derivative")
    spread = logits.stride(1) != 1 and vocab > 1
    if spread or tokens.dtype != torch.int64 or (tokens.dim() == 2 and tokens.stride(1) != 1 and tokens.shape[1] > 1):
        return token_logprobs(logits.contiguous() if spread else logits, tokens.long().contiguous(), top=top, entropy=entropy)
    call = _Logprobs.apply if logits.requires_grad and torch.is_grad_enabled() else _forward
    return TokenLogprobs(*call(logits, tokens, int(top), bool(entropy)))
