"""Attention through a window with sinks (paged.tree_attention(window=, sinks=)) against its definition in 64 bits: of the keys that
a token sees without a window, the last `window` and those at the first `sinks` positions. The bound is that of
test_gpu_paged.py, over the keys that are left."""
import math

import pytest
import torch

from dsv41_flash_offload_b200 import paged
from test_gpu_paged import DEV, HALF_UNIT, attend, build

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def seen_keys(s, b, i, base, window, sinks):
    c, n = s["ctx"][b], s["new"][b]
    if s["mask"] is None:
        see = list(range(c + i + 1))
    else:
        word = [int(w) & (2 ** 64 - 1) for w in s["mask_host"][base + i]]
        see = list(range(c)) + [c + j for j in range(n) if j // 64 < len(word) and word[j // 64] >> (j % 64) & 1]
    first = len(see) - window
    return [x for at, x in enumerate(see) if at >= first or x < sinks]


def reference(s, window, sinks):
    """(out, bound, lse) in 64 bits; bound without the terms that infinities make meaningless."""
    q, kc, vc = (s[n].cpu().double() for n in ("q", "kc", "vc"))
    s["mask_host"] = None if s["mask"] is None else s["mask"].cpu()
    page, kv, dim = kc.shape[1:]
    heads, scale, u = q.shape[1], dim ** -0.5, HALF_UNIT[s["q"].dtype]
    out, bound, lse = torch.zeros_like(q), torch.zeros_like(q), torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    table, base = s["table"].cpu().long(), 0
    for b, (c, n) in enumerate(zip(s["ctx"], s["new"])):
        pos = torch.arange(c + n)
        k, v = kc[table[b][pos // page], pos % page], vc[table[b][pos // page], pos % page]
        for i in range(n):
            seen = seen_keys(s, b, i, base, window, sinks)
            if not seen:
                continue
            ks, vs = k[seen].repeat_interleave(heads // kv, 1), v[seen].repeat_interleave(heads // kv, 1)
            score = torch.einsum("hd,khd->hk", q[base + i], ks) * scale
            w = torch.softmax(score, 1)
            o, A = (w[:, :, None] * vs.transpose(0, 1)).sum(1), torch.einsum("hk,khd->hd", w, vs.abs())
            e = (dim / 16 + 8) * 2.0 ** -22 * scale * torch.einsum("hd,khd->hk", q[base + i].abs(), ks.abs()).amax(1) + 2.0 ** -21
            lost = len(seen) * 2.0 ** -24 * vs.abs().amax() if s["q"].dtype == F16 else 0.0
            out[base + i], lse[base + i] = o, torch.logsumexp(score, 1)
            bound[base + i] = (2 * u + 2 * e[:, None] + (len(seen) / 16 + 64) * 2.0 ** -22) * A + u * o.abs() + lost + 1e-7
        base += n
    return out, bound, lse


def check(s, window, sinks):
    out, lse = attend(s, window=window, sinks=sinks, return_lse=True)
    assert paged.read_status() == 0
    ref, bound, ref_lse = reference(s, window, sinks)
    over = (out.cpu().double() - ref).abs() - bound
    assert not torch.isnan(out).any() and bool((over <= 0).all()), float(over.max())
    fin = torch.isfinite(ref_lse)
    assert torch.equal(torch.isfinite(lse.cpu()), fin)
    assert float((lse.cpu().double() - ref_lse)[fin].abs().max() if fin.any() else 0) < 2 * HALF_UNIT[s["q"].dtype] + 1e-3
    return out


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 4), (3, 0), (17, 4), (64, 130), (128, 128), (200, 1), (1000, 4), (5000, 7)])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("page", [16, 7])
def test_windows_and_sinks(window, sinks, tree, page):
    check(build([700, 3, 0, 129, 400], [5, 1, 12, 9, 40], 8, 2, 64, page, BF16, seed=window, tree=tree), window, sinks)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,kv,dim,new", [(1, 1, 64, [5, 1]), (8, 2, 128, [9, 4]), (16, 2, 128, [8, 3]), (40, 8, 128, [20, 2]),
                                              (16, 1, 128, [15, 30]), (5, 1, 80, [60, 2]), (4, 2, 256, [7, 20]), (8, 1, 192, [30, 1]),
                                              (8, 1, 256, [5, 2])])
@pytest.mark.parametrize("tree", [False, True])
def test_heads_and_row_tiles(heads, kv, dim, new, dtype, tree):
    check(build([900, 333], new, heads, kv, dim, 32, dtype, seed=heads + dim, tree=tree), 300, 5)


@pytest.mark.parametrize("window,sinks", [(1, 0), (100, 3), (129, 0), (600, 200)])
@pytest.mark.parametrize("heads,kv,dim,page", [(4, 2, 64, 16), (8, 1, 128, 24), (2, 1, 256, 64)])
def test_prompt_chunks(window, sinks, heads, kv, dim, page):
    """Row tiles of one request reach different tiles of keys."""
    check(build([0, 350, 1], [700, 90, 301], heads, kv, dim, page, F16, seed=window, tree=False), window, sinks)


@pytest.mark.parametrize("window", [1, 2, 5, 70, 130])
def test_trees_deeper_than_the_window(window):
    """Ancestors leave the window one by one, also over words of the mask."""
    s = build([3, 0, 40], [150, 100, 7], 4, 2, 64, 16, BF16, words=3, seed=window)
    chain = torch.zeros(257, 3, dtype=torch.int64)
    base = 0
    for n in s["new"]:
        for i in range(n):
            for j in range(i + 1):
                chain[base + i, j // 64] |= (1 << (j % 64)) - (1 << 64 if j % 64 == 63 else 0)
        base += n
    out = check(dict(s, mask=chain.to(DEV)), window, 2)
    plain = attend(dict(s, mask=None), window=window, sinks=2)        # a chain is a sequence
    err = (out.float() - plain.float()).abs().max()
    assert float(err) <= 4 * torch.finfo(BF16).eps * float(plain.float().abs().max())
    check(s, window, 2)


def test_masks_with_holes_and_empty_rows():
    """Any bits: the last `window` of what they leave; a token whose bits leave nothing of an empty context is 0."""
    s = build([0, 30], [40, 40], 4, 2, 64, 16, F16, seed=3)
    g = torch.Generator().manual_seed(5)
    s["mask"] = torch.randint(-2 ** 62, 2 ** 62, (80, 1), generator=g).to(DEV)
    s["mask"][::7] = 0
    out = check(s, 6, 2)
    assert bool((out[0:40:7] == 0).all())


def test_long_windows_are_no_window():
    s = build([700, 3], [5, 30], 8, 2, 128, 16, BF16)
    want = attend(s)
    for window in (2 ** 31 - 1, 2 ** 30, 10 ** 6):
        assert torch.equal(attend(s, window=window), want)
    assert torch.equal(attend(s, window=735, sinks=9), want)


@pytest.mark.parametrize("heads,kv,dim,page,new", [(4, 2, 64, 16, [6, 3]), (16, 2, 128, 32, [8, 3]), (16, 2, 128, 7, [12, 3]),
                                                   (16, 1, 128, 64, [15, 30]), (8, 1, 256, 16, [7, 5])])
@pytest.mark.parametrize("tree", [False, True])
def test_infinities_and_nan_outside_a_window(heads, kv, dim, page, new, tree):
    """What a row does not see does not reach it, whether its tile is read for another row or for the window's edge; what it
    sees does."""
    s = build([650, 300], new, heads, kv, dim, page, F16, seed=dim, tree=tree)
    clean = attend(s, window=200, sinks=3)
    kc, vc = s["kc"].clone(), s["vc"].clone()
    table = s["table"].cpu()

    def put(cache, b, x, value):
        cache[int(table[b, x // page]), x % page, :, ::3] = value

    for x in (3, 4, 100, 449, 440):                 # outside every window
        put(vc, 0, x, math.inf)
        put(kc, 0, x, math.nan)
        put(vc, 0, x + 1, math.nan)
    assert torch.equal(attend(dict(s, kc=kc, vc=vc), window=200, sinks=3), clean)
    put(vc, 0, 450 + 2, math.inf)                   # at the edge: the first tokens' windows reach it
    put(vc, 0, 452, -math.inf if not tree else math.inf)
    put(vc, 1, 1, math.nan)                         # a sink
    d = dict(s, kc=kc, vc=vc)
    got = attend(d, window=200, sinks=3).cpu()
    want = reference(d, 200, 3)[0]
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf].double(), want[inf])
    fin = torch.isfinite(want)
    assert torch.equal(got[fin], clean.cpu()[fin]) and not bool(fin[new[0]:, :, ::3].any())
    assert paged.read_status() == 0


@pytest.mark.parametrize("heads,kv,dim,page", [(4, 1, 64, 16), (16, 2, 128, 64), (8, 1, 128, 7), (2, 1, 256, 24)])
def test_infinities_within_a_prompt_chunk(heads, kv, dim, page):
    """Without a mask a tile of new tokens is an ordinary one for the row tiles behind it: what it holds of infinities reaches
    those whose window does, and no token before."""
    s = build([90, 0], [310, 130], heads, kv, dim, page, F16, seed=dim, tree=False)
    clean = attend(s, window=70, sinks=2).cpu()
    vc, table = s["vc"].clone(), s["table"].cpu()
    for b, x, col, value in ((0, 90, 0, math.inf), (0, 140, dim - 1, math.nan), (0, 399, 0, -math.inf), (1, 1, 3, math.inf), (1, 64, dim - 1, -math.inf)):
        vc[int(table[b, x // page]), x % page, :, col] = value
    d = dict(s, vc=vc)
    got, want = attend(d, window=70, sinks=2).cpu(), reference(d, 70, 2)[0]
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert bool(inf.any()) and torch.equal(torch.isinf(got), inf) and torch.equal(got[inf].double(), want[inf])
    fin = torch.isfinite(want)
    assert torch.equal(got[fin], clean[fin]) and paged.read_status() == 0


def test_windowed_calls_in_a_graph_and_on_another_stream():
    s = build([3000, 77, 900], [9, 4, 1], 8, 2, 128, 16, BF16)
    want = attend(s, window=500, sinks=4)
    side = torch.cuda.Stream()
    paged.reserve_workspace(128, side)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = torch.empty_like(want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            attend(s, window=500, sinks=4, out=out)
    torch.cuda.synchronize()
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    s["seq"].sub_(s["seq"]).add_(torch.tensor([2009, 81, 401], dtype=torch.int32, device=DEV))   # other lengths, same graph
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, attend(s, window=500, sinks=4)) and paged.read_status() == 0


def test_refused_requests_and_requests_without_tokens():
    s = build([100, 50, 0, 70], [3, 4, 2, 0], 4, 2, 64, 16, F16)
    want = attend(s, window=20, sinks=2)
    s["seq"][1] = 0
    got = attend(s, window=20, sinks=2)
    assert bool((got[3:7] == 0).all()) and torch.equal(got[:3], want[:3]) and torch.equal(got[7:], want[7:])
