"""Prompts on their way into the paged cache beside the reads' own path: qkv_front and attend over packed prompts, their keys appended as they
are, then the next token of each through append_paged and attend_paged."""
import math

import pytest
import torch

from dan_amd import append_paged, attend, attend_paged
from dan_amd.attention import Batch, segment
from dan_amd.front import qkv_front
from oracle import paged as OP

pytestmark = pytest.mark.gpu
H, HKV, D, PAGE = 8, 2, 128, 16
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prompts_go_on_token_by_token(gpu, dtype):
    """The cache's rows are the prefill's keys and values bit for bit. The next token's attention over them is within attend_paged's bound of the 64-bit
    one (one rounding of the output, 2^-14 of sum p |v| for fp32 work at these scores), and within that and attend's 2e-2 of the
    prefill's own answer for the same token."""
    print(f"[gpu-case] prompts through the front end, then the cache, {dtype}", flush=True)
    lens = [33, 1, 70]
    g = torch.Generator().manual_seed(2)
    whole = [n + 1 for n in lens]  # the prompt and the token that follows it
    rows = sum(whole)
    x = torch.randn(rows, (H + 2 * HKV) * D, generator=g).to(dtype).to(gpu)
    starts = [sum(whole[:i]) for i in range(3)]
    at = torch.cat([torch.arange(n) for n in whole])
    inv = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    angle = torch.cat((at[:, None] * inv,) * 2, 1)
    cos, sin = angle.cos().to(dtype).to(gpu), angle.sin().to(dtype).to(gpu)
    wq, wk = ((torch.randn(D, generator=g) * 0.2 + 1).to(dtype).to(gpu) for _ in range(2))
    q, k, v = x.view(rows, H + 2 * HKV, D).split([H, HKV, HKV], 1)
    qh, kh, vh = qkv_front(q, k, v, cos, sin, q_norm_weight=wq, k_norm_weight=wk)
    whole_read = attend(qh, kh, vh, Batch([segment(s, [0] * n, device=gpu) for s, n in zip(starts, whole)]), 0)

    width = 6
    table = torch.randperm(3 * width, generator=g).int().view(3, width).to(gpu)
    kc, vc = (torch.full((3 * width, HKV, PAGE, D), math.nan, dtype=dtype, device=gpu) for _ in range(2))
    prompt = torch.cat([torch.arange(s, s + n) for s, n in zip(starts, lens)]).to(gpu)
    ints = lambda y: torch.tensor(y, dtype=torch.int32, device=gpu)
    append_paged(None, kh.transpose(0, 1)[prompt], vh.transpose(0, 1)[prompt], None, None, kc, vc, table, ints([t for n in lens for t in range(n)]),
                 seqs=ints([i for i, n in enumerate(lens) for _ in range(n)]), norm=None)
    for i, (s, n) in enumerate(zip(starts, lens)):
        for cache, rows_ in ((kc, kh), (vc, vh)):
            assert torch.equal(cache[table[i].long()].transpose(0, 1).reshape(HKV, width * PAGE, D)[:, :n], rows_[:, s:s + n])

    last = torch.tensor([s + n for s, n in zip(starts, lens)], device=gpu)
    qn = append_paged(q[last], k[last], v[last], cos[last], sin[last], kc, vc, table, ints(lens), q_norm_weight=wq, k_norm_weight=wk)
    out = attend_paged(qn, kc, vc, table, ints(whole)).cpu().double()
    ref, _, mag, _ = OP.attend(qn.cpu(), kc.cpu().double().nan_to_num(), vc.cpu().double().nan_to_num(), table.cpu(), whole)
    assert ((out - ref).abs() <= HALF[dtype] * ref.abs() + 2.0 ** -14 * mag).all()
    assert (out - whole_read[:, last].cpu().double()).abs().max() <= 2e-2 + 2.0 ** -7


@pytest.mark.parametrize("pages,seqs_of_table,width", [(0, 3, 2), (4, 3, 0), (0, 0, 0), (4, 0, 2)])
def test_a_cache_or_table_without_pages_stores_nothing(gpu, pages, seqs_of_table, width, monkeypatch):
    """No token has a page then: q comes back, nothing is written, through the host module and through Python."""
    print(f"[gpu-case] append: {pages} pages, a table of {seqs_of_table} x {width}", flush=True)
    from dan_amd import _decode

    x = torch.randn(3, 2, 64, generator=torch.Generator().manual_seed(0)).bfloat16().to(gpu)
    guard = torch.zeros(pages + 2, 2, PAGE, 64, dtype=torch.bfloat16, device=gpu)
    cache = guard[1:pages + 1] if pages else torch.empty(0, 2, PAGE, 64, dtype=torch.bfloat16, device=gpu)
    table = torch.zeros(seqs_of_table, width, dtype=torch.int32, device=gpu)
    places, seqs = (torch.tensor(t, dtype=torch.int32, device=gpu) for t in ([0, 17, -1], [0, 1, 2]))
    rest = type("Rest", (), dict(append=staticmethod(lambda *a: None)))
    for real in (True, False):
        if not real:
            monkeypatch.setattr(_decode, "calls", lambda: rest)
        q = append_paged(x, x, x, None, None, cache, cache.clone(), table, places, seqs=seqs, norm=None)
        torch.cuda.synchronize()
        assert torch.equal(q, x.transpose(0, 1)) and not guard.any()
