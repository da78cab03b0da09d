"""include/dan_paged.h and dan_readout.h without a GPU: exports, struct layouts and
packed buffers, refusals before any launch, the index arithmetic of the paged
cache (csrc/paged_index.h, compiled for the host) against wrong places and
pages, and the CPU oracles against torch's own."""
import ctypes
import math
import os
import random
import re
import subprocess

import pytest
import torch

from dan_amd import _build, _decode, _native
from oracle import paged as OP
from oracle import readout as OR

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADERS = [os.path.join(ROOT, "include", f) for f in ("dan_paged.h", "dan_readout.h")]
STRUCTS = {n: c for n, c in vars(_decode).items() if isinstance(c, type) and issubclass(c, ctypes.Structure)}
ENTRIES = [(_decode.call_append, _decode.DanPagedAppendArgs), (_decode.call_paged_attn, _decode.DanPagedAttnArgs),
           (_decode.call_logprobs, _decode.DanLogprobsArgs), (_decode.call_logprobs_grad, _decode.DanLogprobsGradArgs)]


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_native.LIB_PATH):
        _build.build()
    return _native.load()


def test_exports_every_declared_function(lib):
    text = "".join(open(h).read() for h in HEADERS)
    names = set(re.findall(r"^\s*(?:const\s+)?\w+\s*\*?\s*(dan_\w+)\s*\(", text, re.M))
    assert names == set(_decode.EXPORTS)
    out = subprocess.run(["nm", "-D", "--defined-only", _native.LIB_PATH], capture_output=True, text=True).stdout
    assert names <= set(re.findall(r" T (dan_\w+)", out))
    assert lib["dan_paged_abi_version"]() == _decode.PAGED_ABI_VERSION
    assert lib["dan_readout_abi_version"]() == _decode.READOUT_ABI_VERSION


def test_ctypes_layout_matches_headers(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "dan_paged.h"', '#include "dan_readout.h"', "int main(void) {"]
    for name, cls in STRUCTS.items():
        lines += [f'printf("{name} %zu\\n", sizeof({name}));'] + [f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    lines.append('printf("CONST %d,%d,%d,%d,%d\\n", DAN_PAGED_ABI_VERSION, DAN_PAGED_KEY_BLOCK, DAN_READOUT_ABI_VERSION, '
                 'DAN_READOUT_MAX_TOP, DAN_READOUT_MAX_TOP_VOCAB); return 0; }')
    (tmp_path / "probe.c").write_text("\n".join(lines))
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(tmp_path / "probe.c"), "-o",
                    str(tmp_path / "probe")], check=True)
    out = subprocess.run([str(tmp_path / "probe")], capture_output=True, text=True, check=True).stdout
    got = dict(line.rsplit(" ", 1) for line in out.splitlines())
    for name, cls in STRUCTS.items():
        assert int(got[name]) == ctypes.sizeof(cls), name
        for f, _ in cls._fields_:
            assert int(got[f"{name}.{f}"]) == getattr(cls, f).offset, f"{name}.{f}"
    assert got["CONST"] == (f"{_decode.PAGED_ABI_VERSION},{_decode.KEY_BLOCK},{_decode.READOUT_ABI_VERSION},{_decode.MAX_TOP},"
                            f"{_decode.MAX_TOP_VOCAB}")


@pytest.mark.parametrize("entry,args", ENTRIES, ids=[e.name for e, _ in ENTRIES])
def test_packed_fields_lie_where_the_structure_has_them(entry, args):
    values = [{ctypes.c_int32: -7 - i, ctypes.c_int64: -(1 << 40) - i, ctypes.c_float: 0.5 + i,
               ctypes.c_void_p: (1 << 46) + 16 * i}[t] for i, (_, t) in enumerate(args._fields_)]
    packed = args.from_buffer_copy(entry.pack(*values))
    assert [getattr(packed, n) for n, _ in args._fields_] == values


BUF = 1 << 20  # an address that is aligned, and never read: every call below is refused, or has nothing to do

APPEND = dict(abi_version=1, dtype=0, cache_dtype=0, table_dtype=0, num_tokens=4, num_heads=8, num_kv_heads=2, head_dim=128, rotary_dim=64,
              norm=1, page_size=16, num_pages=8, table_width=4, num_seqs=4, num_rope_rows=4, eps=1e-6, q=BUF, q_stride_tok=1024,
              q_stride_head=128, k=BUF, k_stride_tok=256, k_stride_head=128, v=BUF, v_stride_tok=256, v_stride_head=128, cos=BUF,
              sin=BUF, cs_stride_tok=64, q_norm_weight=BUF, k_norm_weight=BUF, q_out=BUF, qo_stride_tok=1024, qo_stride_head=128,
              k_cache=BUF, kc_stride_page=4096, kc_stride_head=2048, kc_stride_tok=128, v_cache=BUF, vc_stride_page=4096,
              vc_stride_head=2048, vc_stride_tok=128, table=BUF, table_stride=4, places=BUF)
ATTN = dict(abi_version=1, dtype=0, cache_dtype=0, num_seqs=4, num_heads=8, num_kv_heads=2, head_dim=128, page_size=16, num_pages=8,
            table_width=4, max_len=64, scale=0.1, q=BUF, q_stride_seq=1024, q_stride_head=128, out=BUF, o_stride_seq=1024,
            o_stride_head=128, k_cache=BUF, kc_stride_page=4096, kc_stride_head=2048, kc_stride_tok=128, v_cache=BUF,
            vc_stride_page=4096, vc_stride_head=2048, vc_stride_tok=128, table=BUF, table_stride=4, lens=BUF)
LOGP = dict(abi_version=1, dtype=0, rows=4, vocab=100, labels=1, top=5, logits=BUF, logits_stride=100, tokens=BUF, tokens_stride=1,
            logprobs=BUF, logsumexp=BUF, top_logprobs=BUF, top_ids=BUF, workspace=BUF, workspace_bytes=1 << 20)
GRAD = dict(abi_version=1, dtype=0, rows=4, vocab=100, labels=1, top=0, logits=BUF, logits_stride=100, tokens=BUF, tokens_stride=1,
            logsumexp=BUF, g_logprobs=BUF, grad=BUF, grad_stride=100)
REFUSED = [
    (0, APPEND, dict(abi_version=2), "abi_version"), (0, APPEND, dict(head_dim=96), "head_dim"), (0, APPEND, dict(dtype=2), "dtype"),
    (0, APPEND, dict(cache_dtype=1), "cache_dtype"), (0, APPEND, dict(table_dtype=1), "table_dtype"), (0, APPEND, dict(rotary_dim=24), "rotary_dim"),
    (0, APPEND, dict(rotary_dim=144), "rotary_dim"), (0, APPEND, dict(norm=3), "norm"), (0, APPEND, dict(k_norm_weight=0), "norm"),
    (0, APPEND, dict(eps=-1.0), "eps"), (0, APPEND, dict(eps=math.nan), "eps"), (0, APPEND, dict(page_size=8), "page_size"),
    (0, APPEND, dict(page_size=0), "page_size"), (0, APPEND, dict(num_rope_rows=3), "rows of cos"), (0, APPEND, dict(k=0), "NULL"),
    (0, APPEND, dict(places=0), "NULL"), (0, APPEND, dict(cache_dtype=3), "k_scale"), (0, APPEND, dict(k_stride_tok=132), "multiples of 8"),
    (0, APPEND, dict(kc_stride_tok=132), "16 bytes"), (0, APPEND, dict(v_cache=BUF + 8), "aligned"), (0, APPEND, dict(cs_stride_tok=32), "cs_stride"),
    (0, APPEND, dict(num_tokens=-1), "num_tokens"), (0, APPEND, dict(num_heads=1 << 30), "too many"),
    (1, ATTN, dict(abi_version=0), "abi_version"), (1, ATTN, dict(num_heads=9), "multiple"), (1, ATTN, dict(head_dim=80), "head_dim"),
    (1, ATTN, dict(dtype=3), "dtype"), (1, ATTN, dict(cache_dtype=2), "cache_dtype"), (1, ATTN, dict(page_size=24), "page_size"),
    (1, ATTN, dict(max_len=65), "max_len"), (1, ATTN, dict(max_len=-1), "max_len"), (1, ATTN, dict(scale=0.0), "scale"),
    (1, ATTN, dict(scale=math.inf), "scale"), (1, ATTN, dict(scale=math.nan), "scale"), (1, ATTN, dict(lens=0), "NULL"),
    (1, ATTN, dict(num_pages=0), "pages"), (1, ATTN, dict(cache_dtype=3), "k_scale"), (1, ATTN, dict(kc_stride_tok=64), "token strides"),
    (1, ATTN, dict(q_stride_head=4), "multiples of 8"), (1, ATTN, dict(q=BUF + 2), "aligned"),
    (1, ATTN, dict(num_seqs=1, table_width=1 << 20, max_len=1 << 24), "workspace"),
    (2, LOGP, dict(abi_version=7), "abi_version"), (2, LOGP, dict(dtype=3), "dtype"), (2, LOGP, dict(vocab=0), "vocab"),
    (2, LOGP, dict(top=33), "top"), (2, LOGP, dict(vocab=4), "top"), (2, LOGP, dict(vocab=524289), "top tokens"), (2, LOGP, dict(rows=-1), "rows"),
    (2, LOGP, dict(logits=0), "NULL"), (2, LOGP, dict(top_ids=0), "NULL"), (2, LOGP, dict(logits=BUF + 1), "aligned"),
    (2, LOGP, dict(workspace_bytes=16), "workspace"), (2, LOGP, dict(workspace=BUF + 4), "workspace"), (2, LOGP, dict(rows=1 << 30, vocab=1 << 20, top=0), "too many"),
    (3, GRAD, dict(abi_version=7), "abi_version"), (3, GRAD, dict(grad=0), "NULL"), (3, GRAD, dict(g_entropy=BUF), "NULL"),
    (3, GRAD, dict(top=3, g_top=BUF), "NULL"), (3, GRAD, dict(tokens=0), "NULL"), (3, GRAD, dict(grad_stride=99), "grad_stride"),
    (3, GRAD, dict(dtype=2, grad=BUF + 2), "aligned"),
    # more threads than a launch has
    (0, APPEND, dict(num_tokens=1 << 25, num_rope_rows=1 << 25), "one launch"), (1, ATTN, dict(num_seqs=1 << 24, num_heads=2), "one launch"),
    (1, ATTN, dict(num_seqs=1 << 21, num_heads=16, num_kv_heads=1), "one launch"), (2, LOGP, dict(rows=1 << 24), "one launch"),
    (2, LOGP, dict(rows=1 << 26, top=0), "one launch"), (3, GRAD, dict(rows=1 << 26), "one launch"),
]


@pytest.mark.parametrize("which,base,change,message", REFUSED, ids=[f"{w}-{'-'.join(map(str, c))}-{i}" for i, (w, _, c, _) in enumerate(REFUSED)])
def test_refusals(lib, which, base, change, message):
    entry, args = ENTRIES[which]
    fields = {**base, **change}
    with pytest.raises(RuntimeError, match=message):
        entry(0, *(fields.get(n, 0) for n, _ in args._fields_))


def test_nothing_to_do_is_no_error(lib):
    for which, base, change in ((0, APPEND, dict(num_tokens=0)), (1, ATTN, dict(num_seqs=0)), (2, LOGP, dict(rows=0)), (3, GRAD, dict(rows=0))):
        entry, args = ENTRIES[which]
        entry(0, *({**base, **change}.get(n, 0) for n, _ in args._fields_))


def test_workspace_sizes(lib):
    """None for no sequences or keys; -1 (0 for the readout) for what the calls refuse."""
    size = _decode.paged_attn_workspace_size
    assert size(-1, 0, 0, 8, 2, 128, 4096) == 0
    assert size(-1, 0, 3, 8, 2, 128, 0) == 0 and size(-1, 0, 1, 8, 2, 128, 1 << 20) > 0 and size(-1, 3, 1, 8, 2, 128, 1 << 20) > 0
    assert all(size(-1, *a) == -1 for a in ((0, 1, 9, 2, 128, 16), (0, 1, 8, 0, 128, 16), (1, 1, 8, 2, 96, 16), (0, 1, 8, 2, 128, -1),
                                            (0, -1, 8, 2, 128, 1), (0, 1, 8, 2, 128, (1 << 30) + 1), (2, 1, 8, 2, 128, 1)))
    assert _decode.logprobs_workspace_size(0, 0, 100, 0) == 16 and _decode.logprobs_workspace_size(3, 1, 100, 0) == 0


def test_cpu_tensors_are_refused():
    from dan_amd.paged import append_paged, attend_paged
    from dan_amd.readout import token_logprobs

    x = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    cache, table, one = torch.zeros(1, 2, 16, 64, dtype=torch.bfloat16), torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="gfx950"):
        append_paged(x, x, x, None, None, cache, cache, table, one, norm=None)
    with pytest.raises(RuntimeError, match="gfx950"):
        attend_paged(x.transpose(0, 1), cache, cache, table, one)
    with pytest.raises(RuntimeError, match="gfx950"):
        token_logprobs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.long))


def test_host_module(lib):
    calls = _decode.calls()
    assert _decode.calls() is calls
    for addresses in ((), (1,) * 6, (0,) * 7):
        with pytest.raises((TypeError, ValueError)):
            calls.bind(*addresses)


def test_wrong_places_and_pages_find_no_row(tmp_path):
    """find_row: every value that a table, a place or a sequence may hold, against the oracle; the table lies
    between guard values that would be valid pages."""
    rng = random.Random(5)
    big = [-(1 << 31), -17, -1, 0, 1, 15, 16, 17, 47, 48, (1 << 31) - 1]
    cases = []
    for page, width, seqs, pages in ((16, 3, 2, 5), (48, 1, 4, 1), (64, 2, 1, 3), (16, 0, 1, 4), (16, 2, 0, 4)):
        table = [rng.choice([-1, 0, pages - 1, pages, 1 << 30, -(1 << 31)]) for _ in range(seqs * width)]
        cases += [(page, width, seqs, pages, table, s, t) for s in (-1, 0, 1, seqs - 1, seqs, 1 << 30, -(1 << 31)) for t in big + [page * width - 1, page * width]]
    body = []
    for i, (page, width, seqs, pages, table, s, t) in enumerate(cases):
        values = ",".join(f"(int32_t){x}LL" for x in [0] * 4 + table + [0] * 4)
        body.append(f"{{ static const int32_t m[] = {{{values}}}; dan::PageTable p = {{m + 4, {width}, {seqs}, {width}, {page}, {pages}}}; "
                    f'dan::PageRow r = dan::find_row(p, (int32_t){s}LL, (int32_t){t}LL); printf("%d %d\\n", r.page, r.row); }}')
    (tmp_path / "rows.cpp").write_text('#include <stdio.h>\n#include "paged_index.h"\nint main() {\n' + "\n".join(body) + "\n}\n")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-fsanitize=address,undefined", "-fno-sanitize-recover", "-I",
                    os.path.join(_build.HERE, "csrc"), str(tmp_path / "rows.cpp"), "-o", str(tmp_path / "rows")], check=True)
    env = {k: v for k, v in os.environ.items() if k != "LD_PRELOAD"}
    got = subprocess.run([str(tmp_path / "rows")], capture_output=True, text=True, check=True, env=env).stdout.splitlines()
    for line, (page, width, seqs, pages, table, s, t) in zip(got, cases, strict=True):
        want = OP.place_of(torch.tensor(table, dtype=torch.int64).view(seqs, width), s, t, page, pages)
        assert line == ("-1 0" if want is None else f"{want[0]} {want[1]}"), (page, width, seqs, pages, table, s, t)
    kernels = [open(os.path.join(_build.HERE, "csrc", f)).read() for f in ("paged_append.hip", "paged_attn.hip")]
    assert all("dan::find_row(" in k for k in kernels)


def test_oracle_attention_and_readout_against_torch():
    g = torch.Generator().manual_seed(0)
    kc, vc = (torch.randn(6, 2, 16, 64, generator=g, dtype=torch.float64) for _ in range(2))
    table = torch.tensor([[4, 1, 0], [2, 5, 3]])
    q = torch.randn(4, 2, 64, generator=g, dtype=torch.float64)
    out, lse, _, _ = OP.attend(q, kc, vc, table, torch.tensor([37, 48]))
    for b, n in enumerate((37, 48)):
        k, v = (c[table[b]].transpose(0, 1).reshape(2, 48, 64)[:, :n].repeat_interleave(2, 0) for c in (kc, vc))
        want = torch.nn.functional.scaled_dot_product_attention(q[:, b:b + 1], k, v)[:, 0]
        assert torch.allclose(out[:, b], want, atol=1e-12)
    x = torch.randn(3, 11, generator=g, dtype=torch.float64, requires_grad=True)
    t = torch.tensor([[0, 3, 3], [10, -1, 2], [5, 5, 5]])
    logp = torch.log_softmax(x, 1)
    lp, lse, ent, top, ids = OR.token_logprobs(x.detach(), t, 4)
    assert torch.allclose(lp, torch.where(t < 0, 0.0, logp.detach().gather(1, t.clamp(min=0))))
    assert torch.allclose(ent, -(logp.exp() * logp).sum(1).detach()) and torch.equal(ids, torch.topk(x, 4).indices)
    ws = [torch.randn(s, generator=g, dtype=torch.float64) for s in ((3, 3), (3,), (3,), (3, 4))]
    loss = (torch.where(t < 0, 0.0, logp.gather(1, t.clamp(min=0))) * ws[0]).sum() + (torch.logsumexp(x, 1) * ws[1]).sum() \
        - ((logp.exp() * logp).sum(1) * ws[2]).sum() + (logp.gather(1, ids) * ws[3]).sum()
    want = torch.autograd.grad(loss, x)[0]
    assert torch.allclose(OR.gradient(x.detach(), t, ids, *ws), want, atol=1e-12)
