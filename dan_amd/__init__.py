"""dan_amd: gfx950 (MI355X) tree-masked prefill attention for dan-style packed reads.

``dan_amd.attention`` is the drop-in for dan/attention.py; its ``attend`` runs
one fused HIP kernel (dan_amd/csrc/tree_attn.hip) through the C ABI declared in
include/dan_tree_attn.h.

``dan_amd.paged`` and ``dan_amd.readout`` hold what a sequence needs that goes on
token by token behind its read: ``append_paged`` (norm, rotary and a paged
key-value cache), ``attend_paged`` (one new token over that cache) and
``token_logprobs`` (log probabilities of given tokens, with their gradient).
"""
from .attention import Batch, Segment, attend, branch_rows_mask, repeat_heads, segment, to_device, tree_mask
from .paged import append_paged, attend_paged
from .readout import TokenLogprobs, token_logprobs

__all__ = ["Batch", "Segment", "TokenLogprobs", "append_paged", "attend", "attend_paged", "branch_rows_mask", "repeat_heads", "segment",
           "to_device", "token_logprobs", "tree_mask"]
