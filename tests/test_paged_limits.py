"""Paged attention's limits without a GPU: fewer than 2^32 threads a launch, whose number goes by the waves of a work group, and the largest scale."""
import os

import pytest

from dan_amd import _build, _decode, _native
from test_decode_abi import ATTN


@pytest.mark.parametrize("change", [
    dict(num_seqs=1 << 22, num_heads=2, num_kv_heads=2, table_width=64, max_len=1024),    # 2^23 work groups of eight waves
    dict(num_seqs=1 << 23, num_heads=2, num_kv_heads=2, table_width=64, max_len=64),      # 2^24 of four
    dict(num_seqs=1 << 23, num_heads=2, num_kv_heads=1, table_width=64, max_len=64),      # 2^24 sequences x heads
], ids=["eight waves", "four waves", "heads"])
def test_more_threads_than_a_launch_has_are_refused(change):
    if not os.path.exists(_native.LIB_PATH):
        _build.build()
    fields = {**ATTN, **change}
    with pytest.raises(RuntimeError, match="one launch"):
        _decode.call_paged_attn(0, *(fields.get(n, 0) for n, _ in _decode.DanPagedAttnArgs._fields_))


def test_a_scale_that_overflows_with_log2_e_is_refused():
    if not os.path.exists(_native.LIB_PATH):
        _build.build()
    for scale, ok in ((2.0 ** 127, True), (2.5e38, False), (3.4e38, False)):
        fields = {**ATTN, "scale": scale, "num_seqs": 0}  # nothing to do where it is taken
        args = [fields.get(n, 0) for n, _ in _decode.DanPagedAttnArgs._fields_]
        if ok:
            _decode.call_paged_attn(0, *args)
        else:
            with pytest.raises(RuntimeError, match="scale"):
                _decode.call_paged_attn(0, *args)
