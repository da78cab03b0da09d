"""include/dan_readout.h without a GPU: calls of version 1, whose structures end before logsumexp_rest, are still taken."""
import ctypes
import os

import pytest

from dan_amd import _build, _decode, _native

ENTRIES = [("dan_logprobs_fwd", _decode.DanLogprobsArgs), ("dan_logprobs_bwd", _decode.DanLogprobsGradArgs)]


@pytest.mark.parametrize("name,args", ENTRIES, ids=[n for n, _ in ENTRIES])
def test_versions(name, args):
    """No rows, so nothing to do: versions 1 and 2 pass, all others are refused. A structure of version 1 ends in front of a guard."""
    if not os.path.exists(_native.LIB_PATH):
        _build.build()
    fn = _native.load()[name]
    fn.argtypes, fn.restype = [ctypes.c_void_p, ctypes.c_void_p], ctypes.c_int
    assert args._fields_[-1][0] == "logsumexp_rest" and args.logsumexp_rest.offset == ctypes.sizeof(args) - 8
    a = args(dtype=2, vocab=10, labels=1)
    a.logsumexp_rest = 0xDEAD
    for version, want in ((1, 0), (2, 0), (0, None), (3, None), (-1, None)):
        a.abi_version = version
        rc = fn(ctypes.addressof(a), None)
        assert (rc == 0) == (want == 0), version
        if want is None:
            assert "abi_version" in _native.last_error(_native.load())
