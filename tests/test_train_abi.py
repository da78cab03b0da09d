"""What adapters are trained and served with, without a GPU: the ctypes mirrors have the headers' layouts, argument
errors come back before any launch, and the backward pass's tables cover what each row sees."""
import ctypes
import os
import re
import subprocess

import numpy as np
import pytest
import torch

from dan_amd import _grad, _layer, _native, workloads
from dan_amd.adapters import adapt
from dan_amd.attention import Batch, attend_train, segment
from dan_amd.norm import add_norm
from test_abi import HEADER, lib  # noqa: F401  -- the library fixture

INCLUDE = os.path.dirname(HEADER)
HEADERS = {"dan_tree_grad.h": _grad.EXPORTS, "dan_norm.h": _layer.EXPORTS[:4], "dan_adapt.h": _layer.EXPORTS[4:]}
STRUCTS = {"DanTreeGradArgs": ("dan_tree_grad.h", _grad.DanTreeGradArgs), "DanNormArgs": ("dan_norm.h", _layer.DanNormArgs),
           "DanNormGradArgs": ("dan_norm.h", _layer.DanNormGradArgs), "DanAdaptArgs": ("dan_adapt.h", _layer.DanAdaptArgs),
           "DanAdaptGradArgs": ("dan_adapt.h", _layer.DanAdaptGradArgs)}


@pytest.mark.parametrize("header", HEADERS)
def test_exports_are_what_the_header_declares(lib, header):  # noqa: F811
    text = open(os.path.join(INCLUDE, header)).read()
    names = set(re.findall(r"^\s*(?:const\s+)?\w+\s*\*?\s*(dan_\w+)\s*\(", text, re.M))
    assert names == set(HEADERS[header])
    out = subprocess.run(["nm", "-D", "--defined-only", _native.LIB_PATH], capture_output=True, text=True, check=True).stdout
    assert names <= set(re.findall(r" T (dan_\w+)", out))


@pytest.mark.parametrize("name", STRUCTS)
def test_struct_layout(name, tmp_path):
    header, cls = STRUCTS[name]
    src, exe = tmp_path / "p.c", tmp_path / "p"
    src.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "{header}"\nint main(void) {{\nprintf("%zu\\n", sizeof({name}));\n'
                   + "".join(f'printf("%zu\\n", offsetof({name}, {f}));\n' for f, _ in cls._fields_) + "return 0; }\n")
    subprocess.run(["gcc", "-std=c99", "-I", INCLUDE, str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f, _ in cls._fields_]


def test_unit_and_limit_constants_follow_the_headers(tmp_path):
    src, exe = tmp_path / "p.c", tmp_path / "p"
    src.write_text('#include <stdio.h>\n#include "dan_tree_grad.h"\n#include "dan_norm.h"\n#include "dan_adapt.h"\nint main(void) {\n'
                   'printf("%zu %zu %d %d %d %d %d\\n", sizeof(DanGradKeyUnit), sizeof(DanGradQueryUnit), DAN_TREE_GRAD_ABI_VERSION, DAN_NORM_ABI_VERSION,'
                   ' DAN_ADAPT_ABI_VERSION, DAN_NORM_MAX_COLS, DAN_ADAPT_MAX_RANK);\nreturn 0; }\n')
    subprocess.run(["gcc", "-std=c99", "-I", INCLUDE, str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [32, 32, _grad.GRAD_ABI_VERSION, _layer.NORM_ABI_VERSION, _layer.ADAPT_ABI_VERSION, _layer.MAX_COLS, _layer.MAX_RANK]


BAD, UNSUPPORTED, VERSION, OK = _native.ERR_INVALID_ARGUMENT, _native.ERR_UNSUPPORTED, _native.ERR_VERSION, _native.OK
P = 4096  # an aligned address that no call reads
GRAD = dict(abi_version=1, dtype=_native.DTYPE_BF16, num_heads=4, num_kv_heads=2, head_dim=64, num_tokens=8, scale=0.125,
            **{f: P for f in ("q", "k", "v", "out", "grad", "lse", "dq", "dk", "dv", "key_units", "query_units", "row_lo", "row_end", "workspace")},
            **{f"{t}_stride_tok": 512 for t in ("q", "k", "v", "o", "g", "dq", "dk", "dv")},
            **{f"{t}_stride_head": 64 for t in ("q", "k", "v", "o", "g", "dq", "dk", "dv")},
            num_key_units=1, num_query_units=1, key_splits=1, workspace_bytes=1 << 20)
NORM = dict(abi_version=1, dtype=_native.DTYPE_BF16, rows=3, cols=64, norm=0, layout=0, eps=1e-6, x=P, x_stride=64, weight=P, out=P, out_stride=64)
NORM_GRAD = dict(abi_version=1, dtype=_native.DTYPE_BF16, rows=3, cols=64, norm=0, s=P, s_stride=64, weight=P, rstd=P, g=P, g_stride=64, ds=P, ds_stride=64)
ADAPT = dict(abi_version=1, dtype=_native.DTYPE_BF16, rows=3, n_in=64, n_out=32, rank=8, adapters=2, x=P, x_stride=64, y=P, y_stride=32, a=P, b=P,
             index=P, scale_value=1.0, out=P, out_stride=32, workspace=P, workspace_bytes=1 << 20)
ADAPT_GRAD = dict(abi_version=1, dtype=_native.DTYPE_BF16, rows=3, n_in=64, n_out=32, rank=8, adapters=2, x=P, x_stride=64, g=P, g_stride=32, a=P, b=P,
                  index=P, scale_value=1.0, down=P, dx=P, dx_stride=64, da=P, db=P, workspace=P, workspace_bytes=1 << 20)
ERRORS = [
    ("dan_tree_attn_bwd", kw, status, needle) for kw, status, needle in (
        (dict(abi_version=2), VERSION, "abi_version"), (dict(num_heads=3), BAD, "num_heads"), (dict(num_kv_heads=0), BAD, "num_heads"),
        (dict(head_dim=96), UNSUPPORTED, "head_dim"), (dict(dtype=_native.DTYPE_F32), UNSUPPORTED, "dtype"), (dict(num_tokens=-1), BAD, "negative"),
        (dict(scale=float("nan")), BAD, "scale"), (dict(scale=-0.1), BAD, "scale"), (dict(scale=0.0), BAD, "scale"), (dict(scale=2.0 ** 101), BAD, "scale"),
        (dict(key_rows=32), BAD, "key_rows"), (dict(key_splits=0), BAD, "key_splits"), (dict(key_splits=3), BAD, "key_splits"), (dict(lse=None), BAD, "NULL"), (dict(num_pasts=1), BAD, "NULL"), (dict(workspace_bytes=64), BAD, "workspace"),
        (dict(workspace=P + 16), BAD, "workspace"), (dict(q=P + 8), BAD, "aligned"), (dict(dk=P + 2), BAD, "aligned"), (dict(g_stride_tok=510), BAD, "strides"),
        (dict(k_stride_tok=1 << 25), UNSUPPORTED, "token stride"), (dict(v_stride_tok=-512), UNSUPPORTED, "token stride"), (dict(num_tokens=0, q=None), OK, ""))
] + [
    ("dan_add_norm", kw, status, needle) for kw, status, needle in (
        (dict(abi_version=2), VERSION, "abi_version"), (dict(dtype=_native.DTYPE_F32), UNSUPPORTED, "dtype"), (dict(rows=-1), BAD, "rows"),
        (dict(rows=1 << 24), BAD, "rows"), (dict(cols=60), UNSUPPORTED, "cols"), (dict(cols=0), UNSUPPORTED, "cols"), (dict(cols=16392), UNSUPPORTED, "cols"),
        (dict(norm=2), BAD, "norm"), (dict(layout=2), BAD, "layout"), (dict(eps=float("nan")), BAD, "eps"), (dict(eps=-1.0), BAD, "eps"),
        (dict(x=None), BAD, "NULL"), (dict(out=None), BAD, "NULL"), (dict(codes=P), BAD, "NULL"), (dict(codes=P, scale=P, cols=72), UNSUPPORTED, "16"),
        (dict(x=P + 2), BAD, "aligned"), (dict(x_stride=60), BAD, "aligned"), (dict(out_stride=56), BAD, "overlap"), (dict(rows=0, x=None), OK, ""))
] + [
    ("dan_add_norm_grad", kw, status, needle) for kw, status, needle in (
        (dict(abi_version=0), VERSION, "abi_version"), (dict(cols=12), UNSUPPORTED, "cols"), (dict(norm=-1), BAD, "norm"), (dict(rstd=None), BAD, "NULL"),
        (dict(g_stride=4), BAD, "aligned"), (dict(ds_stride=8), BAD, "overlap"), (dict(dw=P), BAD, "workspace"),
        (dict(dw=P, workspace=P, workspace_bytes=8), BAD, "workspace"), (dict(rows=0, s=None), OK, ""))
] + [
    (name, kw, status, needle) for name in ("dan_adapt", "dan_adapt_grad") for kw, status, needle in (
        (dict(abi_version=2), VERSION, "abi_version"), (dict(dtype=_native.DTYPE_E4M3), UNSUPPORTED, "dtype"), (dict(rows=-1), UNSUPPORTED, "rows"),
        (dict(rows=(1 << 20) + 1), UNSUPPORTED, "rows"), (dict(n_in=60), UNSUPPORTED, "n_in"), (dict(n_out=0), UNSUPPORTED, "n_out"),
        (dict(n_in=(1 << 20) + 8), UNSUPPORTED, "n_in"), (dict(rank=0), UNSUPPORTED, "rank"), (dict(rank=136), UNSUPPORTED, "rank"),
        (dict(adapters=0), UNSUPPORTED, "adapters"), (dict(adapters=65536), UNSUPPORTED, "adapters"), (dict(scale_value=float("inf")), BAD, "scale_value"),
        (dict(rows=1 << 20, n_in=1 << 20), UNSUPPORTED, "launch"), (dict(x=None), BAD, "NULL"), (dict(x=P + 8), BAD, "aligned"),
        (dict(workspace=None), BAD, "workspace"), (dict(workspace_bytes=8), BAD, "workspace"), (dict(rows=0, x=None), OK, ""))
] + [
    ("dan_adapt", dict(out_stride=24), BAD, "overlap"), ("dan_adapt", dict(down=P + 4), BAD, "aligned"),
    ("dan_adapt_grad", dict(dx_stride=8), BAD, "overlap"), ("dan_adapt_grad", dict(down=None), BAD, "NULL")]
BASES = {"dan_tree_attn_bwd": (GRAD, _grad.DanTreeGradArgs), "dan_add_norm": (NORM, _layer.DanNormArgs), "dan_add_norm_grad": (NORM_GRAD, _layer.DanNormGradArgs),
         "dan_adapt": (ADAPT, _layer.DanAdaptArgs), "dan_adapt_grad": (ADAPT_GRAD, _layer.DanAdaptGradArgs)}


@pytest.mark.parametrize("name,kw,status,needle", ERRORS)
def test_argument_errors_come_before_any_launch(lib, name, kw, status, needle):  # noqa: F811
    base, cls = BASES[name]
    if name == "dan_tree_attn_bwd":
        base = {"key_rows": lib.dan_tree_grad_key_rows(64, 0), **base}
    a = cls()
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    assert lib[name](ctypes.byref(a), None) == status
    assert needle in _native.last_error(lib)
    assert lib[name](None, None) == BAD


def test_sizes_of_what_the_entries_do_not_take_are_0(lib):  # noqa: F811
    assert lib.dan_tree_grad_key_rows(96, 0) == 0 and lib.dan_tree_grad_query_rows(3, 2, 64) == 0 and lib.dan_tree_grad_query_rows(4, 2, 96) == 0
    assert _grad.workspace_size(0, 2, 64, 5) == 0 and _grad.workspace_size(4, 2, 64, -1) == 0
    assert _grad.workspace_size(4, 2, 64, 5, 0) == 0 and _grad.workspace_size(4, 2, 64, 5, 3) == 0 and _grad.workspace_size(4, 2, 64, 5, 2) > _grad.workspace_size(4, 2, 64, 5)
    assert _layer.norm_grad_workspace_size(-1, 64) == 0 and _layer.norm_grad_workspace_size(4, 60) == 0
    assert _layer.adapt_workspace_size(0, 64, 16, 1) == 0 and _layer.adapt_workspace_size(4, 64, 129, 1) == 0
    assert _layer.adapt_grad_workspace_size(4, 60, 64, 16, 1) == 0 and _layer.adapt_grad_workspace_size(4, 64, 64, 16, 0) == 0


# ---------------------------------------------------------------- the backward pass's tables
def batch_of(structure, gap=0):
    segs, at = Batch(), gap
    for t, ls in structure:
        ids = workloads.branch_ids(t, ls)
        segs.append(segment(at, ids, None, 0, 0, "cpu"))
        at += len(ids) + gap
    return segs, at


@pytest.mark.parametrize("key_rows,query_rows", [(64, 32), (128, 64), (64, 128), (128, 128)])
@pytest.mark.parametrize("gap", [0, 3])
@pytest.mark.parametrize("structure", [[(1, [])], [(0, [3, 40, 2])], [(40, [5, 9, 1]), (7, [30]), (1, [3] * 6), (64, [])], [(257, [40, 3, 70])], [(128, [64, 64])]])
def test_units_cover_what_each_row_sees(structure, gap, key_rows, query_rows):
    segs, n = batch_of(structure, gap)
    rows = [(s.start, s.end - s.start, s.trunk, 10 * i, i) for i, s in enumerate(segs)]
    keys, queries, row_lo, row_end, covered = _grad.build_units(np.array(rows), [s.branches for s in segs], n, key_rows, query_rows)
    assert covered == (gap == 0)
    sees = np.zeros((n, n), bool)  # [row, key]
    for s in segs:
        for j, (a, b) in enumerate([(s.start, s.start + s.trunk)] + list(s.branches)):
            for i in range(a, b):
                sees[i, s.start:(i + 1 if j == 0 else s.start + s.trunk)] = True
                if j:
                    sees[i, a:i + 1] = True
    own = sum(s.end - s.start for s in segs)
    seen = np.zeros(n, int)
    for start, m, trunk, k0, count, q_end, *_ in keys:  # every key in one unit, whose rows hold all that see it
        assert 0 < count <= key_rows and k0 + count <= m and k0 < q_end <= m
        seen[start + k0:start + k0 + count] += 1
        who = np.flatnonzero(sees[:, start + k0:start + k0 + count].any(1))
        assert who.min() >= start + k0 and who.max() < start + q_end
        for k in range(start + k0, start + k0 + count):  # a key's rows: those of [key, row_end)
            assert np.array_equal(np.flatnonzero(sees[:, k]), np.arange(k, start + row_end[k]))
    assert seen.sum() == own and seen.max() == 1
    seen[:] = 0
    for start, m, trunk, t0, count, past, idx, b0 in queries:
        assert 0 < count <= query_rows and t0 + count <= m and past == 10 * idx
        seen[start + t0:start + t0 + count] += 1
        for r in range(t0, t0 + count):  # a row's keys: the trunk up to it, and from b0 on those of [row_lo, r]
            want = set(np.flatnonzero(sees[start + r]) - start)
            got = set(range(0, min(r + 1, trunk)))
            if r >= trunk:
                assert b0 <= row_lo[start + r]
                got |= set(range(row_lo[start + r], r + 1))
            assert got == want
    assert seen.sum() == own and seen.max() == 1


def test_longest_units_come_first():
    segs, n = batch_of([(40, [5, 9]), (513, [70, 64])])
    rows = np.array([(s.start, s.end - s.start, s.trunk, 0, -1) for s in segs])
    keys, queries, *_ = _grad.build_units(rows, [s.branches for s in segs], n, 64, 64)
    steps = -(-(keys[:, 5] - keys[:, 3]) // 32)
    assert (np.diff(steps) <= 0).all()


def test_segments_that_share_rows_are_refused():
    rows = np.array([(0, 10, 10, 0, -1), (9, 5, 5, 0, -1)])
    with pytest.raises(ValueError, match="another segment"):
        _grad.build_units(rows, [[], []], 14, 64, 64)


# ---------------------------------------------------------------- refusals on the CPU
def test_there_is_no_cpu_path():
    x, w = torch.zeros(2, 64, dtype=torch.bfloat16), torch.ones(64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU only"):
        add_norm(x, None, w)
    with pytest.raises(RuntimeError, match="GPU only"):
        adapt(x, x, torch.zeros(1, 8, 64, dtype=torch.bfloat16), torch.zeros(1, 64, 8, dtype=torch.bfloat16))


@pytest.mark.parametrize("scale", [0.0, -0.125, float("nan"), float("inf"), 2.0 ** 101])
def test_attend_train_refuses_a_scale_out_of_range(scale):
    segs, n = batch_of([(4, [2])])
    q, k = torch.zeros(2, n, 64, dtype=torch.bfloat16), torch.zeros(1, n, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="scale"):
        attend_train(q, k, k, segs, 0, scale)


def test_attend_train_refuses_other_types_and_prefixes_that_want_a_gradient():
    segs, n = batch_of([(4, [2])])
    q = torch.zeros(1, n, 64)
    with pytest.raises(ValueError, match="bf16 or fp16"):
        attend_train(q, q, q, segs, 0)
    entry = torch.zeros(1, 3, 64, dtype=torch.bfloat16, requires_grad=True)
    segs = Batch([segment(0, workloads.branch_ids(4, [2]), {0: (entry, entry.detach())}, 0, 3, "cpu")])
    q = torch.zeros(1, n, 64, dtype=torch.bfloat16)
    with pytest.raises(NotImplementedError, match="constants"):
        attend_train(q, q, q, segs, 0)
