"""append_paged and attend_paged on the GPU against the CPU oracle in float64
(oracle/paged.py).

Tolerances. u = finfo(dtype).eps / 2 is the rounding of a stored value (bf16
2^-8, fp16 2^-11; fp16 values below 2^-14 are off by at most 2^-25; e4m3 codes by 2^-4 of
their value or 2^-10, once scaled). fp32 work in front of it:
- append: two products and a sum on top of a norm factor whose sum of squares has at most 2 + log2(D)
  + D / 8 roundings in a row, so at most 64 units of 2^-24 of the terms' magnitudes: 2^-18.
- attend: a score is a sum of D exact products, off by at most (D + 8) 2^-24 of sum |q_d k_jd| scale = E,
  with 4 more units for exp's argument; weights are split into two roundings, 2 u^2 together
  (fp16: or 2^-25 each, at most n 2^-25 together, as the largest weight is 1), and summed with at most n + 64 roundings.
  So each output is off by u |o| + (2 u^2 + 2 E + |s| 2^-22 + (n + 64) 2^-23) sum p |v|, with |s| <= the largest
  sum |q_d k_jd| scale."""
import math

import pytest
import torch

from dan_amd.paged import append_paged, attend_paged
from oracle import paged as OP

pytestmark = pytest.mark.gpu
BF16, F16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
HALF = {BF16: 2.0 ** -8, F16: 2.0 ** -11}


def say(msg):
    print(f"[gpu-case] {msg}", flush=True)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def paged_table(g, lens, page, width, pages):
    """Pages in random order; entries behind a sequence's last page name none."""
    order = torch.randperm(pages, generator=g)
    table, at = torch.full((len(lens), width), -7, dtype=torch.int32), 0
    for i, n in enumerate(lens):
        need = -(-n // page)
        table[i, :need] = order[at:at + need].int()
        at += need
    assert at <= pages
    return table


def make_cache(g, pages, hkv, page, d, dtype, std=1.0):
    x = torch.randn(2, pages, hkv, page, d, generator=g) * std
    if dtype == E4M3:
        return [(x[i] / (0.02 * std)).clamp(-448, 448).to(E4M3) for i in range(2)], [torch.tensor([0.02 * std]), torch.tensor([0.02 * std])]
    return [x[i].to(dtype) for i in range(2)], [None, None]


def values(cache, scale):
    return cache.double() * (1.0 if scale is None else scale.double())


# ------------------------------------------------------------------ append


def stored_error(got, ref, mag, dtype, scale=None):
    """The largest error in units of its tolerance."""
    got, ref = got.double(), ref.double()
    if dtype == E4M3:
        s = scale.double()
        ref = (ref / s).clamp(-448, 448)
        tol = torch.maximum(ref.abs() * 2.0 ** -4, torch.tensor(2.0 ** -10, dtype=torch.float64)) + 2.0 ** -17 * mag / s
    else:
        tol = ref.abs() * HALF[dtype] + 2.0 ** -18 * mag + (2.0 ** -25 if dtype == F16 else 1e-37)
    return ((got - ref).abs() / tol).max().item() if got.numel() else 0.0


def magnitude(x, w, norm, cos, sin):
    """|terms| of the rotation of the normalized row."""
    n = OP.rotate_norm(x, w, norm, None, None).abs()
    if cos is None:
        return n
    r = cos.shape[-1]
    a, b = n[..., :r // 2], n[..., r // 2:r]
    c, s = cos.double().abs()[:, None], sin.double().abs()[:, None]
    return torch.cat((torch.cat((a, b), -1) * c + torch.cat((b, a), -1) * s, n[..., r:]), -1)


def run_append(gpu, n, h, hkv, d, r, norm, dtype=BF16, cache=None, page=16, decode=True, table32=False, rows=False, seed=0, token_major=False):
    g = gen(seed)
    cache = cache or dtype
    qkv = torch.randn(n, h * d + 2 * hkv * d, generator=g).to(dtype)
    split = lambda t: (t[:, :h * d].reshape(n, h, d) if h else None, t[:, h * d:(h + hkv) * d].unflatten(1, (hkv, d)), t[:, (h + hkv) * d:].unflatten(1, (hkv, d)))
    q, k, v = split(qkv)
    if decode:
        seqs, places = None, torch.randint(0, 5 * page, (n,), generator=g)
        lens = (places + 1).tolist()
    else:
        each = -(-n // 3)
        seqs, places = torch.arange(n) // each, torch.arange(n) % each
        lens = torch.bincount(seqs, minlength=3).tolist()
    width = max(-(-x // page) for x in lens) + 1
    pages = sum(-(-x // page) for x in lens) + 2
    table = paged_table(g, lens, page, width, pages)
    if n > 4:
        places[2] = -1  # a padded row
    (kc, vc), (ks, vs) = make_cache(g, pages, hkv, page, d, cache)
    wq, wk = (torch.randn(d, generator=g).mul(0.3).add(1.0 if norm == "rms" else 0.0).to(dtype) for _ in range(2))
    cos = sin = rope = None
    if r:
        positions = torch.randint(0, 5000, (n,), generator=g)
        count = 5000 if rows else n
        at = torch.arange(5000) if rows else positions
        inv = 10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)
        angle = torch.cat((at[:, None].double() * inv,) * 2, 1)
        cos, sin = (t.to(torch.float32 if table32 else dtype) for t in (angle.cos(), angle.sin()))
        assert cos.shape == (count, r)
        rope = positions.int() if rows else None
    dev = lambda t: None if t is None else t.to(gpu)
    kd, vd = kc.to(gpu), vc.to(gpu)
    if token_major:  # [pages, page, Hkv, D] storage
        kd, vd = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (kd, vd))
    qd, kx, vx = split(qkv.to(gpu))
    out = append_paged(qd, kx, vx, dev(cos), dev(sin), kd, vd, dev(table), dev(places.int()), seqs=None if seqs is None else seqs.int().to(gpu),
                       rope_rows=dev(rope), q_norm_weight=dev(wq), k_norm_weight=dev(wk), norm=norm, k_scale=dev(ks), v_scale=dev(vs))
    torch.cuda.synchronize()
    c, s = (cos[positions], sin[positions]) if rows else (cos, sin)
    worst = 0.0
    if h:
        assert out.shape == (h, n, d) and out.transpose(0, 1).is_contiguous()
        worst = stored_error(out.transpose(0, 1).cpu(), OP.rotate_norm(q, wq, norm, c, s), magnitude(q, wq, norm, c, s), dtype)
    else:
        assert out is None
    rk, rv = kc.double(), vc.double()
    where = OP.append(OP.rotate_norm(k, wk, norm, c, s), v.double(), rk, rv, table, places.tolist(), None if seqs is None else seqs.tolist())
    kept = [i for i, w in enumerate(where) if w is not None]
    assert len(kept) == n - (1 if n > 4 else 0)
    touched = torch.zeros(pages, page, dtype=torch.bool)
    for got, old, ref, mag, scale in ((kd, kc, rk, magnitude(k, wk, norm, c, s), ks), (vd, vc, rv, v.double().abs(), vs)):
        got = got.cpu()
        for i in kept:
            touched[where[i]] = True
        if kept:
            pg, row = torch.tensor([where[i][0] for i in kept]), torch.tensor([where[i][1] for i in kept])
            worst = max(worst, stored_error(got.float()[pg, :, row], ref[pg, :, row], mag[kept], cache, scale))
        same = got.view(torch.uint8).view(pages, hkv, page, -1) == old.view(torch.uint8).view(pages, hkv, page, -1)
        assert same.all(-1).all(1)[~touched].all(), "a row that no token has was written"
    say(f"append n={n} {h}/{hkv}x{d} r={r} {norm} {dtype} cache={cache}: {worst:.3f} of the tolerance")
    assert worst <= 1.0


@pytest.mark.parametrize("norm", [None, "rms", "zero_centered"])
@pytest.mark.parametrize("h,hkv,d,r", [(32, 8, 128, 128), (16, 2, 256, 64), (8, 2, 64, 64), (3, 1, 128, 48), (5, 5, 64, 0)])
def test_append_shapes(gpu, h, hkv, d, r, norm):
    for n in (1, 2, 37):
        run_append(gpu, n, h, hkv, d, r, norm, seed=n + d)


@pytest.mark.parametrize("dtype,cache", [(BF16, E4M3), (F16, F16), (F16, E4M3)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_append_types(gpu, dtype, cache, d):
    run_append(gpu, 45, 4, 2, d, d, "rms", dtype, cache, page=48, seed=d)
    run_append(gpu, 301, 4, 2, d, d // 2, None, dtype, cache, decode=False, seed=d + 1)


def test_append_prompts_tables_and_layouts(gpu):
    run_append(gpu, 1021, 32, 8, 128, 128, "rms", decode=False, page=64)
    run_append(gpu, 77, 8, 2, 128, 128, "rms", decode=False, table32=True)
    run_append(gpu, 77, 8, 2, 128, 96, None, rows=True)
    run_append(gpu, 77, 8, 2, 128, 96, None, rows=True, table32=True, dtype=F16)
    run_append(gpu, 33, 8, 2, 64, 64, "rms", token_major=True)
    run_append(gpu, 33, 0, 2, 128, 0, None, decode=False)  # a prefix moved in, without q


def test_append_takes_whole_prefix_entries_and_misaligned_views(gpu):
    """k, v as a prefix-cache entry has them ([Hkv, P, D]), and views whose rows start off 16 bytes."""
    say("append: prefix entry, misaligned views")
    g = gen(3)
    entry = torch.randn(2, 2, 50, 128, generator=g).to(BF16).to(gpu)
    kc, vc = (torch.zeros(5, 2, 16, 128, dtype=BF16, device=gpu) for _ in range(2))
    table = torch.tensor([[3, 0, 4, 1]], dtype=torch.int32, device=gpu)
    places, seqs = torch.arange(50, dtype=torch.int32, device=gpu), torch.zeros(50, dtype=torch.int32, device=gpu)
    assert append_paged(None, entry[0].transpose(0, 1), entry[1].transpose(0, 1), None, None, kc, vc, table, places, seqs=seqs, norm=None) is None
    for c, x in ((kc, entry[0]), (vc, entry[1])):
        assert torch.equal(c[table[0].long()].transpose(0, 1).reshape(2, 64, 128)[:, :50], x)
    off = torch.randn(50 * 256 + 3, generator=g).to(BF16).to(gpu)[3:].view(50, 2, 128)
    q = append_paged(off, off, off, None, None, kc, vc, table, places, seqs=seqs, norm=None)
    assert torch.equal(q, off.transpose(0, 1))
    assert torch.equal(kc[table[0].long()].transpose(0, 1).reshape(2, 64, 128)[:, :50], off.transpose(0, 1))


def test_append_leaves_out_what_has_no_place(gpu):
    """Places past the table, sequences and pages that do not exist, rotary rows that do not."""
    say("append: wrong places, sequences, pages and rotary rows")
    g = gen(4)
    n = 8
    x = torch.randn(n, 2, 128, generator=g).to(BF16).to(gpu)
    guard = [torch.zeros(6, 2, 16, 128, dtype=BF16, device=gpu) for _ in range(2)]
    kc, vc = (t[1:5] for t in guard)  # pages in front of and behind the cache must stay as they are
    table = torch.tensor([[0, -1], [4, 1], [1 << 30, 2], [3, 3]], dtype=torch.int32, device=gpu)
    seqs = torch.tensor([0, 0, 1, 2, -1, 4, 1 << 30, 3], dtype=torch.int32, device=gpu)
    places = torch.tensor([3, 16, 2, 0, 0, 0, 1, 32], dtype=torch.int32, device=gpu)
    cos = torch.ones(4, 128, dtype=BF16, device=gpu)
    rope = torch.tensor([0, 3, 4, -1, 1 << 30, -(1 << 31), 1, 2], dtype=torch.int32, device=gpu)
    q = append_paged(x, x, x, cos, torch.zeros_like(cos), kc, vc, table, places, seqs=seqs, rope_rows=rope, norm=None)
    torch.cuda.synchronize()
    bad = torch.tensor([False, False, True, True, True, True, False, False], device=gpu)
    assert torch.isnan(q[:, bad]).all() and torch.equal(q[:, ~bad], x.transpose(0, 1)[:, ~bad])
    for t in guard:
        want = torch.zeros_like(t)
        want[1, :, 3] = x[0]
        assert torch.equal(t, want)


def test_append_e4m3_keeps_infinities_in_range_and_nan(gpu):
    say("append: e4m3 range")
    x = torch.tensor([1e4, -1e4, math.inf, -math.inf, math.nan, 447.0, 0.0, -0.0]).repeat(8)[None, None].to(BF16).to(gpu)
    kc, vc = (torch.zeros(1, 1, 16, 64, device=gpu).to(E4M3) for _ in range(2))
    one = torch.ones(1, device=gpu)
    append_paged(None, x, x, None, None, kc, vc, torch.zeros(1, 1, dtype=torch.int32, device=gpu), torch.zeros(1, dtype=torch.int32, device=gpu),
                 norm=None, k_scale=one, v_scale=one)
    got = kc[0, 0, 0, :8].float().cpu()
    assert got[:4].tolist() == [448, -448, 448, -448] and math.isnan(got[4]) and got[5:].tolist() == [448, 0, 0]


def test_append_refusals(gpu):
    say("append: refusals")
    x = torch.zeros(2, 4, 64, dtype=BF16, device=gpu)
    kv = torch.zeros(2, 2, 64, dtype=BF16, device=gpu)
    kc, vc = (torch.zeros(3, 2, 16, 64, dtype=BF16, device=gpu) for _ in range(2))
    table, places = torch.zeros(2, 1, dtype=torch.int32, device=gpu), torch.zeros(2, dtype=torch.int32, device=gpu)
    cs = torch.zeros(2, 64, dtype=BF16, device=gpu)

    def call(q=x, k=kv, v=kv, cos=cs, sin=cs, kcache=kc, vcache=vc, table=table, places=places, norm=None, **kw):
        return append_paged(q, k, v, cos, sin, kcache, vcache, table, places, norm=norm, **kw)

    call()
    for bad in (dict(q=x.half()), dict(v=kv[:1]), dict(k=kv.float(), v=kv.float(), q=x.float()), dict(cos=cs[:1], sin=cs[:1]), dict(sin=None),
                dict(cos=cs.half()), dict(kcache=kc[..., :32]), dict(kcache=kc.half()), dict(kcache=kc[:, :1], vcache=vc[:, :1]),
                dict(table=table.long()), dict(table=table[:1]), dict(places=places.long()), dict(places=places[:1]), dict(seqs=places[:1]),
                dict(norm="rms"), dict(norm="layer"), dict(k_scale=torch.ones(1, device=gpu)), dict(places=places.cpu()),
                dict(kcache=kc[:1].expand(3, -1, -1, -1), vcache=vc), dict(kcache=kc.to(E4M3), vcache=vc.to(E4M3)),
                dict(rope_rows=places.long())):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(RuntimeError, match="page_size"):
        call(kcache=kc[:, :, :8], vcache=vc[:, :, :8])
    with pytest.raises(NotImplementedError):
        call(k=kv.clone().requires_grad_())
    assert call(q=x[:0], k=kv[:0], v=kv[:0], cos=cs[:0], sin=cs[:0], places=places[:0]).shape == (4, 0, 64)


# ------------------------------------------------------------------ attend


def run_attend(gpu, lens, h, hkv, d, dtype=BF16, cache=None, page=16, seed=0, std=1.0, scale=None, max_len=None, token_major=False, extra=1):
    g = gen(seed)
    cache = cache or dtype
    width = max(max(-(-n // page) for n in lens), 1) + extra
    pages = max(1, sum(-(-n // page) for n in lens)) + 2
    table = paged_table(g, lens, page, width, pages)
    (kc, vc), (ks, vs) = make_cache(g, pages, hkv, page, d, cache, std)
    # what lies behind each sequence's end, and in pages that none has, holds anything
    used = torch.zeros(pages, page, dtype=torch.bool)
    for i, n in enumerate(lens):
        for t in range(n):
            used[int(table[i, t // page]), t % page] = True
    kd, vd = kc.to(gpu), vc.to(gpu)
    hole = (~used)[:, None, :, None].to(gpu)
    kd, vd = (torch.where(hole, torch.tensor(math.nan, device=gpu), t.float()).to(cache) for t in (kd, vd))
    if token_major:
        kd, vd = (t.view(torch.uint8).view(pages, hkv, page, -1).transpose(1, 2).contiguous().transpose(1, 2).view(cache) for t in (kd, vd))
    q = (torch.randn(len(lens), h, d, generator=g) * 1.5).to(dtype)
    dl = torch.tensor(lens, dtype=torch.int32)
    dev = lambda t: None if t is None else t.to(gpu)
    out, lse = attend_paged(q.to(gpu).transpose(0, 1), kd, vd, table.to(gpu), dl.to(gpu), scale, k_scale=dev(ks), v_scale=dev(vs),
                            max_len=max_len, return_lse=True)
    torch.cuda.synchronize()
    assert out.shape == (h, len(lens), d) and out.dtype == dtype and out.transpose(0, 1).is_contiguous() and lse.shape == (h, len(lens))
    ref, rl, mag, big = OP.attend(q.transpose(0, 1), values(kc, ks), values(vc, vs), table, lens, scale)
    big = big * (1 / math.sqrt(d) if scale is None else scale)
    n = torch.tensor(lens, dtype=torch.float64)[None, :]
    u = HALF[dtype]
    rel = 2 * u * u + 2 * (d + 12) * 2.0 ** -24 * big + big * 2.0 ** -22 + (n + 64) * 2.0 ** -23
    tol = u * ref.abs() + rel[..., None] * mag + 1e-30
    if dtype == F16:
        tol = tol + 2.0 ** -25 + (n * 2.0 ** -25)[..., None] * float(values(vc, vs).abs().max())
    worst = ((out.cpu().double() - ref).abs() / tol).max().item()
    full = torch.tensor([x > 0 for x in lens])
    lerr = ((lse.cpu().double() - rl).abs() / (rel + rl.abs() * 2.0 ** -22 + 2.0 ** -21))[:, full]
    lerr = lerr.max().item() if full.any() else 0.0
    say(f"attend {len(lens)} sequences to {max(lens)}, {h}/{hkv}x{d} {dtype} cache={cache} page={page}: {worst:.3f}, lse {lerr:.3f} of the tolerance")
    assert worst <= 1.0 and lerr <= 1.0
    assert (lse.cpu()[:, ~full] == -math.inf).all() and (out.cpu()[:, ~full] == 0).all()


LENGTHS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 47, 64, 65, 127, 128, 129, 300]


@pytest.mark.parametrize("page", [16, 48, 64])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attend_lengths(gpu, d, page):
    run_attend(gpu, LENGTHS, 8, 2, d, page=page, seed=d + page)


@pytest.mark.parametrize("h,hkv", [(1, 1), (2, 2), (6, 2), (14, 2), (32, 8), (16, 1), (17, 1), (40, 1), (64, 2)])
def test_attend_heads(gpu, h, hkv):
    run_attend(gpu, [5, 130, 0, 777], h, hkv, 128, seed=h)
    run_attend(gpu, [97], h, hkv, 64, dtype=F16, seed=h)


@pytest.mark.parametrize("dtype,cache", [(BF16, E4M3), (F16, F16), (F16, E4M3)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attend_types(gpu, dtype, cache, d):
    run_attend(gpu, [1, 40, 333, 0, 1500], 8, 2, d, dtype, cache, page=32, seed=d)


def test_attend_long_and_many(gpu):
    run_attend(gpu, [20001], 8, 2, 128, page=64)
    run_attend(gpu, [9000, 4097], 16, 2, 256, page=16, cache=E4M3)
    g = gen(1)
    run_attend(gpu, torch.randint(0, 600, (150,), generator=g).tolist(), 8, 8, 64)
    run_attend(gpu, [100] * 70, 32, 8, 128, page=128)
    run_attend(gpu, [1] * 300, 8, 2, 64)


@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attend_many_heads_of_one_group(gpu, d, cache):
    """16 and more q heads of a kv head (the largest work group memory), in ranges of four and of eight waves."""
    run_attend(gpu, [60, 3001, 0, 1], 16, 1, d, cache=cache)
    run_attend(gpu, [1 + 17 * (i % 60) for i in range(300)], 18, 1, d, cache=cache, seed=1)
    run_attend(gpu, [2500] * 20 + [900, 2499, 0], 32, 16, d, cache=cache, seed=2)


@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attend_a_launch_sized_past_the_caches(gpu, d, cache):
    """A table that could hold more than 256 MB of keys and values: their loads pass the caches by."""
    run_attend(gpu, [60, 3001, 0, 1], 16, 1, d, cache=cache, extra=(1 << 28) // (4 * 16 * 2 * d * (2 if cache == BF16 else 1)) + 1)


def test_attend_short_ranges_past_the_caches(gpu):
    run_attend(gpu, [2100] + [3 * i for i in range(31)], 32, 8, 128)


def test_attend_captured_with_the_largest_work_groups(gpu):
    """16 heads of one kv head in ranges of eight waves take more LDS than a launch has unasked: asked for inside the capture too."""
    say("attend: captured, 16/1 x 128, 256 sequences of up to 1024 keys")
    g = gen(9)
    kc, vc = (torch.randn(64, 1, 16, 128, generator=g).to(BF16).to(gpu) for _ in range(2))
    table = torch.randperm(64, generator=g).int().to(gpu).expand(256, 64)  # all sequences share their pages
    q, lens = torch.zeros(16, 256, 128, dtype=BF16, device=gpu), torch.zeros(256, dtype=torch.int32, device=gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = attend_paged(q, kc, vc, table, lens, return_lse=True)
    for _ in range(3):
        q.copy_(torch.randn(16, 256, 128, generator=g))
        lens.copy_(torch.randint(0, 1025, (256,), generator=g))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone(), lse.clone()
        want = attend_paged(q, kc, vc, table, lens, return_lse=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and (got[1] > 0).sum() > 3000


def test_attend_scales_layouts_and_capacity(gpu):
    run_attend(gpu, [33, 500], 8, 2, 128, std=20.0)  # peaked weights
    run_attend(gpu, [33, 500], 8, 2, 128, scale=0.013)
    run_attend(gpu, [33, 500], 8, 2, 128, max_len=500)
    run_attend(gpu, [33, 500], 8, 2, 128, extra=3000)  # a table made for far more
    run_attend(gpu, [33, 500], 8, 2, 128, token_major=True)
    run_attend(gpu, [33, 500], 8, 2, 256, cache=E4M3, token_major=True)
    run_attend(gpu, [0, 0], 8, 2, 128)
    run_attend(gpu, [0], 8, 2, 128, max_len=0)


def simple(gpu, lens, h=8, hkv=2, d=128, page=16, seed=0, dtype=BF16):
    g = gen(seed)
    width = max(-(-n // page) for n in lens) + 1
    pages = sum(-(-n // page) for n in lens) + 1
    (kc, vc), _ = make_cache(g, pages, hkv, page, d, dtype)
    q = torch.randn(len(lens), h, d, generator=g).to(dtype).transpose(0, 1)
    return [t.to(gpu) for t in (q, kc, vc, paged_table(g, lens, page, width, pages), torch.tensor(lens, dtype=torch.int32))]


@pytest.mark.parametrize("b", [4, 300])
def test_attend_wrong_lengths_and_pages(gpu, b):
    """They make their own sequence NaN and no other differs by a bit (one launch, and one with a join)."""
    say(f"attend: wrong lengths and pages among {b}")
    q, kc, vc, table, lens = simple(gpu, [200, 33, 1, 150] * (b // 4))
    good, glse = attend_paged(q, kc, vc, table, lens, return_lse=True)
    for where, value in (((0, 3), -1), ((0, 12), kc.shape[0]), ((0, 0), 1 << 30), ((3, 9), -(1 << 31))):
        t = table.clone()
        t[where] = value
        out, lse = attend_paged(q, kc, vc, t, lens, return_lse=True)
        other = torch.arange(b, device=gpu) != where[0]
        assert torch.isnan(out[:, where[0]]).all() and torch.isnan(lse[:, where[0]]).all()
        assert torch.equal(out[:, other], good[:, other]) and torch.equal(lse[:, other], glse[:, other])
    for value in (-1, -(1 << 31), table.shape[1] * 16 + 1, (1 << 31) - 1):
        n = lens.clone()
        n[1] = value
        out = attend_paged(q, kc, vc, table, n)
        other = torch.arange(b, device=gpu) != 1
        assert torch.isnan(out[:, 1]).all() and torch.equal(out[:, other], good[:, other])
    n = lens.clone()
    n[0] = 201  # past max_len, though the table could hold it
    out = attend_paged(q, kc, vc, table, n, max_len=200)
    assert torch.isnan(out[:, 0]).all() and not torch.isnan(out[:, 1:]).any()


def test_attend_infinite_and_nan_scores(gpu):
    say("attend: NaN and infinities among the keys")
    q, kc, vc, table, lens = simple(gpu, [70, 70, 70], h=2, hkv=1, page=16)
    row = lambda b, t: (int(table[b, t // 16]), 0, t % 16)
    kc[row(0, 69)][3] = math.nan
    vc[row(1, 5)][7] = math.inf
    kc[row(2, 64)][:] = torch.finfo(BF16).min * torch.sign(q[0, 2].float()).to(BF16)  # head 0: the score overflows to -inf
    out = attend_paged(q, kc, vc, table, lens)
    assert torch.isnan(out[:, 0]).all()
    assert (out[:, 1, 7] == math.inf).all() and torch.isfinite(out[:, 1, :7]).all()
    assert torch.isfinite(out[0, 2]).all()
    # where every score is -inf there is no distribution
    q, kc, vc, table, lens = simple(gpu, [40], h=1, hkv=1)
    kc[:] = -torch.finfo(BF16).max * torch.sign(q[0, 0].float()).to(BF16)
    assert torch.isnan(attend_paged(q, kc, vc, table, lens)).all()


def test_attend_is_the_same_every_time_and_beside_any_neighbour(gpu):
    say("attend: repeatable, independent of the batch's other lengths")
    q, kc, vc, table, lens = simple(gpu, [700, 33, 411, 1])
    a = attend_paged(q, kc, vc, table, lens)
    for _ in range(3):
        assert torch.equal(a, attend_paged(q, kc, vc, table, lens))
    n = lens.clone()
    n[1:] = torch.tensor([0, 5, 1], device=gpu)
    assert torch.equal(a[:, 0], attend_paged(q, kc, vc, table, n)[:, 0])


def test_offsets_past_32_bits(gpu):
    """A cache of more than 4 GiB: append to its far pages and attend over them."""
    say("paged: a 5 GB cache")
    pages, hkv, page, d = 150000, 8, 16, 128
    kc = torch.empty(pages, hkv, page, d, dtype=BF16, device=gpu)
    vc = torch.empty(pages, hkv, page, d, dtype=BF16, device=gpu)
    g = gen(8)
    n = 40
    k, v = (torch.randn(n, hkv, d, generator=g).to(BF16).to(gpu) for _ in range(2))
    table = torch.tensor([[149999, 2, 140001]], dtype=torch.int32, device=gpu)
    seqs, places = torch.zeros(n, dtype=torch.int32, device=gpu), torch.arange(n, dtype=torch.int32, device=gpu)
    append_paged(None, k, v, None, None, kc, vc, table, places, seqs=seqs, norm=None)
    q = torch.randn(1, 32, d, generator=g).to(BF16).to(gpu)
    out = attend_paged(q.transpose(0, 1), kc, vc, table, torch.tensor([n], dtype=torch.int32, device=gpu))
    small = [torch.zeros(3, hkv, page, d, dtype=BF16, device=gpu) for _ in range(2)]
    near = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=gpu)
    append_paged(None, k, v, None, None, *small, near, places, seqs=seqs, norm=None)
    for big, little in zip((kc, vc), small):
        assert torch.equal(big[table[0].long()][:2], little[near[0].long()][:2])
    assert torch.equal(out, attend_paged(q.transpose(0, 1), *small, near, torch.tensor([n], dtype=torch.int32, device=gpu)))


def test_attend_refusals(gpu):
    say("attend: refusals")
    q, kc, vc, table, lens = simple(gpu, [20, 30])
    for bad in (dict(q=q.float()), dict(q=q[:7]), dict(q=q[..., :64]), dict(kc=kc.half()), dict(kc=kc[:2]), dict(table=table[:1]), dict(lens=lens.long()),
                dict(lens=lens[:1]), dict(scale=0.0), dict(scale=math.nan), dict(max_len=table.shape[1] * 16 + 1), dict(max_len=-1),
                dict(kc=kc.to(E4M3), vc=vc.to(E4M3)), dict(k_scale=torch.ones(1, device=gpu)), dict(kc=kc.transpose(2, 3), vc=vc.transpose(2, 3)),
                dict(table=table.cpu())):
        a = {**dict(q=q, kc=kc, vc=vc, table=table, lens=lens, scale=None), **bad}
        with pytest.raises(ValueError):
            attend_paged(a.pop("q"), a.pop("kc"), a.pop("vc"), a.pop("table"), a.pop("lens"), a.pop("scale"), **a)
    with pytest.raises(NotImplementedError):
        attend_paged(q.clone().requires_grad_(), kc, vc, table, lens)
    assert attend_paged(q[:, :0], kc, vc, table[:0], lens[:0]).shape == (8, 0, 128)
