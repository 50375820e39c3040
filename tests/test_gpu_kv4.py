"""The cache in 4 bits (paged.Cache4): codes and values against a restatement in 64 bits, bit by bit, and attention over it against
its definition over the values that the codes stand for, to the bound of test_gpu_paged.py (codes become those values exactly)."""
import math

import pytest
import torch

from dsv41_flash_offload_b200 import Dsv41Error, paged
import test_gpu_paged as base
import test_gpu_window as win
from test_gpu_paged import DEV, build

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def quantize(x):
    """x [..., dim] -> (codes, s, lo, values) by group of 32, decisions in 64 bits."""
    g = x.cpu().unflatten(-1, (-1, 32)).double()
    lo, hi = g.amin(-1), g.amax(-1)
    s = ((hi - lo).float() / 15.0).to(x.dtype)
    over = (lo + 15 * s.double()).to(x.dtype).isinf()
    s = torch.where(over, (s.view(torch.int16) - 1).view(x.dtype), s)
    step = s.double()[..., None]
    code = torch.where(step > 0, torch.round((g - lo[..., None]) / torch.where(step > 0, step, torch.ones_like(step))), torch.zeros_like(g)).clamp(0, 15)
    value = (lo[..., None] + step * code).to(x.dtype)
    bad = ~torch.isfinite(g).all(-1) | ~torch.isfinite(s)
    value[bad], code[bad] = math.nan, 0
    return code.to(torch.uint8), s, lo.to(x.dtype), value.flatten(-2)


def places(chunks):
    """Where token t of chunk c has its codes within the chunk's 8 places: [chunks, 8]."""
    return torch.arange(8) ^ torch.tensor([0, 5, 2, 7]).repeat(2)[:chunks, None]


def codes_of(cache, slots):
    """(codes [N, heads, 2, chunks, 32], scales [N, heads, 2, chunks, 2]) as they lie in the cache."""
    d, page = cache.data.cpu(), cache.page_size
    chunks = cache.head_dim // 32
    rec = d.view(cache.num_pages, cache.kv_heads, 2, page // 8, chunks * 160)
    words = rec[..., :chunks * 128].reshape(*rec.shape[:4], chunks, 8, 4, 4).to(torch.int64)      # [.., token, word, byte]
    word = (words << torch.tensor([0, 8, 16, 24])).sum(-1)                                         # [page, h, kv, group, chunk, place, word]
    word = word.gather(5, places(chunks)[..., None].expand(*word.shape))
    column = torch.arange(8)
    shift = 4 * (column // 2) + 16 * (column % 2)
    code = ((word[..., None] >> shift) & 15).flatten(-2)                                           # [page, h, kv, group, chunk, token, 32]
    scales = rec[..., chunks * 128:].reshape(*rec.shape[:4], chunks, 8, 4).contiguous().view(cache.dtype)
    pg, at = slots // page, slots % page
    pick = lambda t: t[pg, :, :, at // 8, :, at % 8]
    return pick(code.to(torch.uint8)), pick(scales)


def stored(k, v, page, dtype, seed=0, extra=2):
    n, heads, dim = k.shape
    cache = paged.Cache4(-(-n // page) + extra, page, heads, dim, dtype=dtype, device=DEV)
    g = torch.Generator().manual_seed(seed)
    slots = torch.randperm(cache.num_pages * page, generator=g)[:n]
    paged.store_kv4(k.to(DEV), v.to(DEV), slots.to(DEV), cache)
    return cache, slots


def check_store(k, v, page, dtype):
    cache, slots = stored(k, v, page, dtype)
    code, scales = codes_of(cache, slots)
    back = paged.load_kv4(slots.to(DEV), cache)
    for i, x in enumerate((k, v)):
        c, s, lo, value = quantize(x)
        nan = torch.isnan(value.unflatten(-1, (-1, 32))).any(-1)
        assert torch.equal(code[:, :, i], c)
        assert torch.equal(scales[:, :, i, :, 0][~nan], s[~nan]) and torch.equal(scales[:, :, i, :, 1][~nan], lo[~nan])
        got = back[i].cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(value)) and torch.equal(got.nan_to_num(7.0), value.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n,heads,dim,page", [(1, 1, 32, 8), (5, 3, 64, 16), (33, 2, 96, 24), (100, 8, 128, 16), (70, 1, 256, 64), (41, 4, 160, 8),
                                              (2000, 8, 128, 128)])
def test_store_and_load(n, heads, dim, page, dtype):
    g = torch.Generator().manual_seed(n)
    check_store(torch.randn(n, heads, dim, generator=g).to(dtype), (3 * torch.randn(n, heads, dim, generator=g)).to(dtype), page, dtype)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_store_edges(dtype):
    """Constant groups, halves between codes, the ends of the type, its smallest numbers, infinities and NaN."""
    top, tiny = torch.finfo(dtype).max, torch.finfo(dtype).tiny
    g = torch.Generator().manual_seed(1)
    rows = [torch.zeros(32), torch.full((32,), -0.0), torch.full((32,), 1.5), torch.arange(32) * 0.5, -torch.arange(32) * 0.5,
            torch.arange(32) / 31 * 15, torch.where(torch.arange(32) % 2 == 0, 0.0, 15.0) * torch.rand(32, generator=g).round(),
            torch.linspace(0, top, 32), torch.linspace(-top / 2, top / 2, 32), torch.linspace(-top, 0, 32),
            torch.linspace(0, 40 * tiny, 32), torch.arange(32) * tiny * torch.finfo(dtype).eps, torch.linspace(-tiny, tiny, 32),
            torch.cat((torch.tensor([-2.5, 12.5]), torch.zeros(30))),                         # a half: 2.5 steps above lo
            torch.cat((torch.tensor([-2.5, 12.5]), torch.full((15,), 2.0 ** -24), torch.full((15,), -2.0 ** -24))),   # beside it, past fp32
            torch.cat((torch.tensor([1000.0, 1000.5]), torch.full((30,), 1000.25)))]
    for bad in (math.nan, math.inf, -math.inf):
        r = torch.randn(32, generator=g)
        r[7 + len(rows) % 5] = bad
        rows.append(r)
    x = torch.stack(rows)
    if dtype is F16:      # (in bf16 the range of both ends passes fp32: checked below)
        x = torch.cat((x, torch.linspace(-top, top, 32)[None]))
    x = x.to(dtype)
    x = torch.cat((x, x.flip(0)), 1)[:, None].contiguous()
    check_store(x, x.flip(0).contiguous(), 8, dtype)
    if dtype is BF16:
        ends = torch.linspace(-1, 1, 32).double().mul(top).to(dtype)[None, None].contiguous()
        cache, slots = stored(ends, ends, 8, dtype)
        assert bool(torch.isnan(paged.load_kv4(slots.to(DEV), cache)[0]).all())


def test_store_slots_and_strides():
    """Slices of a fused projection; tokens without a slot store nothing and read as zeros; nothing else changes."""
    g = torch.Generator().manual_seed(2)
    fused = torch.randn(30, 8, 64, generator=g).half().to(DEV)
    k, v = fused[:, 2:4], fused[:, 5:7]
    cache = paged.Cache4(5, 16, 2, 64, dtype=F16, device=DEV)
    cache.data.fill_(0x5A)
    before = cache.data.clone()
    slots = torch.arange(30, device=DEV) * 2 + 1
    slots[4], slots[9], slots[11] = -1, 5 * 16, 2 ** 40
    paged.store_kv4(k, v, slots, cache)
    kk, vv = paged.load_kv4(slots, cache)
    live = [i for i in range(30) if i not in (4, 9, 11)]
    assert torch.equal(kk[live].cpu(), quantize(k[live])[3]) and torch.equal(vv[live].cpu(), quantize(v[live])[3])
    assert not bool(kk[[4, 9, 11]].any()) and not bool(vv[[4, 9, 11]].any())
    other = torch.tensor([s for s in range(80) if s not in set(slots.tolist())])
    for a, b in zip(codes_of(cache, other), codes_of(paged.Cache4(5, 16, 2, 64, dtype=F16, data=before.flatten()), other)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    paged.store_kv4(k[:0], v[:0], slots[:0], cache)
    assert paged.load_kv4(slots[:0], cache)[0].shape == (0, 2, 64)


def test_move():
    """Overlapping moves read everything first; bits are kept."""
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(64, 3, 96, generator=g).to(BF16) for _ in range(2))
    cache = paged.Cache4(8, 8, 3, 96, dtype=BF16, device=DEV)
    slots = torch.arange(64, device=DEV)
    paged.store_kv4(k.to(DEV), v.to(DEV), slots, cache)
    was = codes_of(cache, slots.cpu())
    src = torch.tensor([5, 6, 7, 10, 63, 0, -1, 20], device=DEV)
    dst = torch.tensor([4, 5, 6, 7, 0, 63, 30, -1], device=DEV)
    paged.move_kv4(src, dst, cache)
    want = list(range(64))
    for a, b in zip(src.tolist()[:6], dst.tolist()[:6]):
        want[b] = a
    now = codes_of(cache, slots.cpu())
    assert torch.equal(now[0], was[0][want]) and torch.equal(now[1], was[1][want])
    paged.move_kv4(src[:0], dst[:0], cache)


# ------------------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------------------
def in4(s):
    """The same step over a cache in 4 bits; kc and vc become what it stands for."""
    pages, page, heads, dim = s["kc"].shape
    cache = paged.Cache4(pages, page, heads, dim, dtype=s["q"].dtype, device=DEV)
    slots = torch.arange(pages * page, device=DEV)
    paged.store_kv4(s["kc"].reshape(-1, heads, dim), s["vc"].reshape(-1, heads, dim), slots, cache)
    k, v = (x.view(pages, page, heads, dim) for x in paged.load_kv4(slots, cache))
    return dict(s, cache=cache, kc=k, vc=v)


def attend4(s, **kw):
    return paged.tree_attention4(s["q"], s["cache"], s["table"], s["seq"], s["cu"], max(s["new"] + [0]), tree_mask=s["mask"], **kw)


def check4(s, monkeypatch, window=None, sinks=0, scale=None):
    if window is None:
        monkeypatch.setattr(base, "attend", attend4)
        return base.check(s, scale=scale)
    monkeypatch.setattr(win, "attend", attend4)
    return win.check(s, window, sinks)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,kv,dim", [(1, 1, 32), (8, 8, 64), (8, 2, 128), (12, 4, 96), (5, 1, 64), (16, 1, 128), (40, 8, 128), (4, 2, 256),
                                          (6, 3, 192), (8, 1, 256), (2, 2, 160), (3, 1, 224), (64, 2, 128)])
def test_attention_heads(heads, kv, dim, dtype, monkeypatch):
    check4(in4(build([70, 3, 0, 129], [5, 1, 4, 9], heads, kv, dim, 16, dtype, seed=heads + dim)), monkeypatch)


@pytest.mark.parametrize("heads,kv,dim", [(4, 4, 32), (4, 1, 64), (8, 1, 96), (8, 1, 128), (4, 1, 160), (4, 1, 192), (4, 1, 224), (4, 1, 256)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_single_tokens(heads, kv, dim, dtype, monkeypatch):
    check4(in4(build([0, 1, 7, 8, 15, 63, 64, 300, 2000], [1] * 9, heads, kv, dim, 24, dtype, seed=dim, tree=False)), monkeypatch)


@pytest.mark.parametrize("page", [8, 24, 64, 128, 256])
@pytest.mark.parametrize("tree", [False, True])
def test_pages_and_lengths(page, tree, monkeypatch):
    check4(in4(build([0, 1, 63, 64, 127, 128, 129, 500], [1, 3, 1, 4, 2, 2, 60, 7], 4, 2, 64, page, BF16, seed=page, tree=tree)), monkeypatch)


@pytest.mark.parametrize("heads,kv,dim,new", [(4, 2, 128, [3, 1, 2]), (8, 1, 128, [1, 2, 1]), (16, 2, 64, [9, 2, 4]), (32, 2, 128, [9, 30, 4]),
                                              (4, 1, 256, [2, 1, 2])])
def test_long_and_split(heads, kv, dim, new, monkeypatch):
    check4(in4(build([9000, 123, 4567], new, heads, kv, dim, 16, F16, seed=dim)), monkeypatch)


@pytest.mark.parametrize("new,words", [([70, 3], 2), ([200, 130], 4), ([256, 1], 4)])
def test_trees_past_one_word(new, words, monkeypatch):
    check4(in4(build([33, 0], new, 4, 2, 64, 16, BF16, words=words)), monkeypatch)


def test_causal_chunks(monkeypatch):
    check4(in4(build([0, 100], [500, 333], 4, 1, 64, 16, F16, tree=False)), monkeypatch)


@pytest.mark.parametrize("window,sinks", [(1, 0), (3, 4), (64, 130), (200, 1), (1000, 4)])
@pytest.mark.parametrize("heads,kv,dim,new", [(4, 2, 64, [3, 1, 2]), (16, 2, 128, [9, 1, 12]), (32, 1, 128, [20, 40, 9]), (8, 1, 256, [4, 30, 2])])
@pytest.mark.parametrize("tree", [False, True])
def test_windows(window, sinks, heads, kv, dim, new, tree, monkeypatch):
    check4(in4(build([700, 3, 129], new, heads, kv, dim, 24, BF16, seed=window, tree=tree)), monkeypatch, window, sinks)


def test_prompt_chunks_through_a_window(monkeypatch):
    check4(in4(build([0, 350], [400, 90], 8, 2, 64, 16, F16, tree=False)), monkeypatch, 100, 3)


def test_large_scores_and_scales(monkeypatch):
    s = in4(build([300, 40], [4, 2], 8, 2, 128, 16, F16, q_scale=30.0))
    check4(s, monkeypatch)
    check4(s, monkeypatch, scale=-0.05)
    check4(s, monkeypatch, scale=0.0)


def test_rows_that_see_nothing():
    s = in4(build([0, 20, 0], [3, 2, 1], 4, 2, 64, 16, F16))
    s["mask"][0] = 0
    s["mask"][5] = 0
    out, lse = attend4(s, return_lse=True)
    for row in (0, 5):
        assert bool((out[row] == 0).all()) and bool((lse[row] == -math.inf).all())
    assert bool(out[1].any()) and paged.read_status() == 0
    s["seq"][1] = 0           # refused
    again = attend4(s)
    assert bool((again[3:5] == 0).all()) and torch.equal(again[:3], out[:3])


@pytest.mark.parametrize("heads,kv,dim,new", [(4, 2, 64, [6, 3]), (8, 1, 128, [2, 1]), (8, 2, 96, [9, 4]), (16, 1, 128, [15, 9]), (8, 1, 256, [7, 5])])
@pytest.mark.parametrize("window", [None, 60])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_nan_reaches_those_who_see_it(heads, kv, dim, new, window, dtype):
    """NaN and infinities in new tokens, in the context, behind the last key and outside a window: their group is NaN for
    the rows that see the token, and nothing else changes, to the bit."""
    s = build([150, 77], new, heads, kv, dim, 16, dtype, seed=dim)
    sinks = 3 if window else 0
    clean4 = in4(s)
    clean = attend4(clean4, window=window, sinks=sinks).cpu()
    vc, kc = s["vc"].clone(), s["kc"].clone()
    table = s["table"].cpu()

    def put(cache, b, x, col, value):
        cache[int(table[b, x // 16]), x % 16, :, col] = value

    put(vc, 0, 151, dim - 1, math.nan)                       # a new token
    put(vc, 0, 150, 0, math.inf)
    put(vc, 0, 150 + new[0], 0, math.nan)                    # behind the last key
    put(kc, 0, 150 + new[0], 0, math.nan)
    put(vc, 1, 5, 0, -math.inf)                              # context: outside the window
    put(vc, 1, 1, dim - 1, math.nan)                         # a sink
    put(vc, 1, 60, 0, math.nan)                              # context
    d = in4(dict(s, kc=kc, vc=vc))
    got = attend4(d, window=window, sinks=sinks).cpu()
    w = window or 10 ** 6
    want = win.reference(d, w, sinks)[0]
    nan = torch.isnan(want)
    assert bool(nan.any()) and bool((~nan).any())
    assert torch.equal(torch.isnan(got), nan)
    assert torch.equal(got[~nan], clean[~nan]) and paged.read_status() == 0
    put(kc, 0, 152 if new[0] > 2 else 150, 3, math.nan)      # a key of NaN: the rows that see it are NaN throughout
    d = in4(dict(s, kc=kc, vc=vc))
    assert torch.equal(torch.isnan(attend4(d, window=window, sinks=sinks).cpu()), torch.isnan(win.reference(d, w, sinks)[0]))


@pytest.mark.parametrize("heads,kv,dim", [(4, 1, 64), (16, 2, 128), (2, 1, 256)])
@pytest.mark.parametrize("window", [None, 70])
def test_nan_within_a_prompt_chunk(heads, kv, dim, window):
    """Without a mask a tile of new tokens is an ordinary one for the row tiles behind it: what is NaN there reaches them, and no
    token before."""
    s = build([90, 0], [310, 130], heads, kv, dim, 16, BF16, seed=dim, tree=False)
    sinks = 2 if window else 0
    clean = attend4(in4(s), window=window, sinks=sinks).cpu()
    vc, table = s["vc"].clone(), s["table"].cpu()
    for b, x, col in ((0, 90, 0), (0, 140, dim - 1), (0, 399, 0), (1, 1, 3), (1, 64, dim - 1)):
        vc[int(table[b, x // 16]), x % 16, :, col] = math.nan
    d = in4(dict(s, vc=vc))
    got = attend4(d, window=window, sinks=sinks).cpu()
    nan = torch.isnan(win.reference(d, window or 10 ** 6, sinks)[0])
    assert bool(nan.any()) and torch.equal(torch.isnan(got), nan) and torch.equal(got[~nan], clean[~nan])


def test_a_cache_without_pages():
    """Every table entry lies outside it: keys and values of zeros."""
    for heads, new in ((4, 1), (4, 30)):
        c = paged.Cache4(0, 16, 2, 64, dtype=F16, device=DEV)
        q = torch.randn(new, heads, 64, device=DEV).half()
        out, lse = paged.tree_attention4(q, c, torch.zeros(1, 4, dtype=torch.int32, device=DEV), torch.tensor([40], dtype=torch.int32, device=DEV),
                                         torch.tensor([0, new], dtype=torch.int32, device=DEV), new, return_lse=True)
        assert not bool(out.any())
        keys = 40 - new + 1 + torch.arange(new)
        assert torch.allclose(lse.cpu(), keys.float().log()[:, None].expand(new, heads), atol=1e-5)
        slots = torch.zeros(new, dtype=torch.int64, device=DEV)
        paged.store_kv4(q[:, :2], q[:, :2], slots, c)
        assert not bool(paged.load_kv4(slots, c)[0].any())
        paged.move_kv4(slots, slots, c)


def test_nan_in_a_split_request():
    s = build([9000, 40], [3, 2], 4, 2, 128, 16, BF16)
    clean = attend4(in4(s)).cpu()
    vc = s["vc"].clone()
    table = s["table"].cpu()
    for x in (100, 9001):
        vc[int(table[0, x // 16]), x % 16, 0, 70] = math.nan
    got = attend4(in4(dict(s, vc=vc))).cpu()
    nan = torch.zeros_like(got, dtype=torch.bool)
    nan[:3, :2, 64:96] = True
    assert torch.equal(torch.isnan(got), nan) and torch.equal(got[~nan], clean[~nan])


def test_slots_past_the_end_may_hold_anything():
    s = in4(build([61, 130, 7], [2, 1, 5], 8, 2, 128, 16, F16))
    want = attend4(s)
    page = 16
    used = torch.zeros(s["cache"].num_pages * page, dtype=torch.bool)
    table = s["table"].cpu()
    for b, (c, n) in enumerate(zip(s["ctx"], s["new"])):
        x = torch.arange(c + n)
        used[table[b].long()[x // page] * page + x % page] = True
    chunks = 4
    back = places(chunks).to(DEV)                           # place p holds token back[p] (the exchange is its own reverse)
    rec = s["cache"].data.view(-1, 2, 2, page // 8, chunks * 160)
    free = (~used).view(-1, page // 8, 8).to(DEV)
    for fill in (0xFF, 0x7C, 0x7F):
        codes = rec[..., :chunks * 128].unflatten(-1, (chunks, 8, 16))
        scales = rec[..., chunks * 128:].unflatten(-1, (chunks, 8, 4))
        at = free[:, None, None, :, None, :, None]
        codes.copy_(torch.where(free[:, :, back][:, None, None, :, :, :, None], torch.full_like(codes, fill), codes))
        scales.copy_(torch.where(at, torch.full_like(scales, fill), scales))
        assert torch.equal(attend4(s), want)


def test_table_entries_outside_the_cache_read_as_zeros():
    s = in4(build([100, 64], [2, 3], 4, 2, 64, 16, F16, tree=False))
    s["table"][0, 2], s["table"][1, 0] = s["cache"].num_pages, -5
    got = attend4(s)
    kc, vc = torch.cat((s["kc"], torch.zeros_like(s["kc"][:1]))), torch.cat((s["vc"], torch.zeros_like(s["vc"][:1])))
    table = s["table"].clone()
    table[1, 0] = s["cache"].num_pages
    d = dict(s, kc=kc, vc=vc, table=table)
    ref, bound, _ = base.reference(d)
    assert bool(((got.cpu().double() - ref).abs() <= bound).all())


def test_offsets_past_32_bits(monkeypatch):
    """5.4 GB of cache, pages at both ends of it."""
    pages, page, kv, dim = 2 ** 18, 16, 8, 128
    s = build([200, 40], [2, 1], 16, kv, dim, page, BF16)
    cache = paged.Cache4(pages, page, kv, dim, dtype=BF16, data=torch.empty(pages * page * kv * dim * 2 * 5 // 8, dtype=torch.uint8, device=DEV))
    assert cache.data.numel() > 2 ** 32
    small = in4(s)
    far = s["table"].long() * 0 + pages - 1 - s["table"].long()
    x = torch.arange(s["kc"].shape[0] * page, device=DEV)
    slots = (pages - 1 - x // page) * page + x % page
    paged.store_kv4(s["kc"].reshape(-1, kv, dim), s["vc"].reshape(-1, kv, dim), slots, cache)
    k, v = paged.load_kv4(slots, cache)
    assert torch.equal(k.view_as(small["kc"]), small["kc"]) and torch.equal(v.view_as(small["vc"]), small["vc"])
    got = attend4(dict(s, cache=cache, table=far.int()))
    assert torch.equal(got, attend4(small))


def test_strided_query_and_output(monkeypatch):
    s = in4(build([50, 9], [4, 2], 6, 2, 64, 16, F16))
    want = attend4(s)
    wide = torch.zeros(6, 9, 96, dtype=F16, device=DEV)
    wide[:, 1:7, 8:72] = s["q"]
    out = torch.full((8, 7, 80), 3.0, dtype=F16, device=DEV)
    attend4(dict(s, q=wide[:, 1:7, 8:72]), out=out[1:7, :6, 8:72])
    assert torch.equal(out[1:7, :6, 8:72], want)
    out[1:7, :6, 8:72] = 3.0
    assert bool((out == 3.0).all())


def test_repeats_in_graphs_and_on_streams():
    s = in4(build([3000, 77, 900, 15], [2, 1, 2, 1], 8, 2, 128, 16, BF16))
    want = attend4(s)
    assert all(torch.equal(attend4(s), want) for _ in range(5))
    side = torch.cuda.Stream()
    paged.reserve_workspace(128, side)
    side.wait_stream(torch.cuda.current_stream())
    g = torch.Generator().manual_seed(9)
    k, v = (torch.randn(6, 2, 128, generator=g).to(BF16).to(DEV) for _ in range(2))
    slots = torch.full((6,), -1, dtype=torch.int64, device=DEV)
    graph = torch.cuda.CUDAGraph()
    out = torch.empty_like(want)
    with torch.cuda.graph(graph, stream=side):
        paged.store_kv4(k, v, slots, s["cache"])
        attend4(s, out=out)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    with torch.cuda.stream(side):
        again = attend4(s)
    torch.cuda.synchronize()
    assert torch.equal(again, want) and paged.read_status() == 0


def test_many_requests(monkeypatch):
    lens = [(i * 37) % 300 for i in range(600)]
    check4(in4(build(lens, [1 + i % 3 for i in range(600)], 2, 1, 32, 16, F16)), monkeypatch)


def test_one_workspace_serves_both_caches():
    s = build([3000, 200], [2, 9], 8, 2, 128, 16, BF16)
    d = in4(s)
    w = paged.attention_workspace(128)
    a, b = base.attend(s), attend4(d)
    for _ in range(2):
        assert torch.equal(base.attend(s, workspace=w), a)
        assert torch.equal(attend4(d, workspace=w), b)
    assert paged.read_status(workspace=w) == 0


def test_refusals():
    s = in4(build([20], [2], 4, 2, 64, 16, F16))
    c = s["cache"]
    k = torch.zeros(2, 2, 64, dtype=F16, device=DEV)
    slots = torch.zeros(2, dtype=torch.int64, device=DEV)
    for bad in (lambda: paged.store_kv4(k[:1], k, slots, c), lambda: paged.store_kv4(k, k, slots.int(), c),
                lambda: paged.store_kv4(k, k[:, :1], slots, c), lambda: paged.load_kv4(slots.cpu(), c), lambda: paged.move_kv4(slots, slots[:1], c),
                lambda: paged.Cache4(2, 16, 1, 64, data=torch.zeros(100, dtype=torch.uint8, device=DEV)),
                lambda: attend4(dict(s, q=s["q"][:, :3])), lambda: attend4(s, sinks=2), lambda: attend4(s, window=0),
                lambda: attend4(s, workspace=torch.zeros(4, device=DEV))):
        with pytest.raises((ValueError, Dsv41Error)):
            bad()
    for bad in (lambda: paged.store_kv4(k.float(), k, slots, c), lambda: attend4(dict(s, q=s["q"].to(BF16)))):
        with pytest.raises(TypeError):
            bad()
