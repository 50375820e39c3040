"""Page tables, cache store and drafted-tree attention (paged.*) against plain restatements.

Tables and store are whole numbers and copies: exact. Attention is compared with its definition in 64 bits;
the bound per element, with w_j the softmax weights and A = sum_j w_j |v_j|, adds up
  - P rounded to the cache's type (half a unit u, relative) in both sums: 2 u A (fp16 also loses weights
    below 2^-25 of the largest: at most keys * 2^-24 * max |v|),
  - scores in fp32: an absolute error e of the exponent shifts every weight by e relative, in both sums: 2 e A,
    e = (D / 16 + 8) * 2^-22 * scale * max_j sum |q k_j| + 2^-21 (exp2),
  - fp32 sums over the keys: (keys / 16 + 64) * 2^-22 * A,
  - the output's half unit: u |out|."""
import math

import numpy as np
import pytest
import torch

from dsv41_flash_offload_b200 import Dsv41Error, paged

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF_UNIT = {t: torch.finfo(t).eps / 2 for t in (torch.float16, torch.bfloat16)}


# ------------------------------------------------------------------------------------------------
# tables
# ------------------------------------------------------------------------------------------------
def tables_ref(ctx, new, held, table, free, count, page, N, parents=None, words=1):
    """The stack discipline, one request and one page at a time."""
    B, W = table.shape
    table, free = table.copy(), free.copy()
    need = [-(-(c + n) // page) for c, n in zip(ctx, new)]
    stack = free[:count].tolist()
    status = [0] * B
    want = list(need)
    for b in range(B):
        if need[b] > W:
            want[b], status[b] = held[b], paged.TOO_WIDE
        stack += [int(p) for p in table[b, want[b]:held[b]]]
    for i, p in enumerate(stack):
        if count <= i < len(free):
            free[i] = p
    total, served = 0, list(held)
    top = len(stack)
    for b in range(B):
        take = max(want[b] - held[b], 0)
        total += take
        if take and total > top:
            status[b] = paged.NO_PAGES
        elif not status[b]:
            for c in range(held[b], want[b]):
                table[b, c] = stack.pop()
            served[b] = want[b]
    cu = np.concatenate([[0], np.cumsum(new)])
    slots, pos, req = np.full(N, -1, np.int64), np.zeros(N, np.int32), np.full(N, -1, np.int32)
    mask = np.zeros((N, words), np.uint64)
    refused = [s & 3 for s in status]
    for b in range(B):
        for i in range(new[b]):
            t = cu[b] + i
            if t >= N:
                break
            at = ctx[b] + i
            req[t], pos[t] = b, at
            if not refused[b]:
                slots[t] = int(table[b, at // page]) * page + at % page
            if parents is not None:
                chain, cur = [i], i
                while True:
                    up = int(parents[cu[b] + cur])
                    if up < -1 or up >= cur:
                        if cur == i:
                            status[b] |= paged.BAD_PARENT
                        break
                    if up < 0:
                        break
                    chain.append(up)
                    cur = up
                pos[t] = ctx[b] + len(chain) - 1
                for j in chain:
                    if j < 64 * words:
                        mask[t, j // 64] |= np.uint64(1 << (j % 64))
                if i >= 64 * words:
                    status[b] |= paged.BIG_TREE
    seq = [0 if refused[b] else ctx[b] + new[b] for b in range(B)]
    return dict(table=table, free=free, cu=cu, seq=seq, slots=slots, pos=pos, req=req, held=served, count=len(stack),
                status=status, mask=mask.view(np.int64))


def run_tables(ctx, new, held, table, free, count, page, N, parents=None, words=1):
    i32 = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device=DEV)
    tb, fr = i32(table), i32(free)
    t = paged.step_tables(i32(ctx), i32(new), i32(held), tb, fr, i32([count]), page, N,
                          parents=None if parents is None else i32(parents), mask_words=words)
    return t, tb, fr


def check_tables(ctx, new, held, table, free, count, page, N, parents=None, words=1):
    ref = tables_ref(ctx, new, held, table, free, count, page, N, parents, words)
    t, tb, fr = run_tables(ctx, new, held, table, free, count, page, N, parents, words)
    got = dict(table=tb, free=fr, cu=t.cu_lens, seq=t.seq_lens, slots=t.slots, pos=t.positions, req=t.requests,
               held=t.held_pages, count=t.free_count, status=t.status)
    if parents is not None:
        got["mask"] = t.tree_mask
    for key, v in got.items():
        want = np.asarray(ref[key]).reshape(v.shape)
        assert np.array_equal(v.cpu().numpy(), want), key
    return ref


def make_tables(rng, B, page, ctx_hi, new_hi, spare, extra=3, width=None):
    ctx = rng.integers(0, ctx_hi + 1, B).tolist()
    new = rng.integers(0, new_hi + 1, B).tolist()
    held = [-(-c // page) + (int(rng.integers(0, extra + 1)) if rng.random() < 0.3 else 0) for c in ctx]
    W = width or max(max(held), max(-(-(c + n) // page) for c, n in zip(ctx, new))) + 1
    held = [min(h, W) for h in held]
    ids = rng.permutation(sum(held) + spare).astype(np.int32)
    table = np.full((B, W), -7, np.int32)
    at = 0
    for b in range(B):
        table[b, :held[b]] = ids[at:at + held[b]]
        at += held[b]
    free = np.full(len(ids), -9, np.int32)
    free[:spare] = ids[at:]
    return ctx, new, held, table, free, spare


@pytest.mark.parametrize("B,page,ctx_hi,new_hi", [(1, 16, 0, 1), (1, 1, 5, 3), (3, 16, 40, 5), (33, 7, 200, 20), (64, 16, 500, 1),
                                                  (255, 64, 900, 300), (256, 8, 30, 4), (257, 16, 10, 60), (2048, 16, 100, 9)])
@pytest.mark.parametrize("spare", [0, 5, 4000])
def test_step_tables(B, page, ctx_hi, new_hi, spare):
    rng = np.random.default_rng(B * 7 + spare)
    args = make_tables(rng, B, page, ctx_hi, new_hi, spare)
    check_tables(*args, page, sum(args[1]) + int(rng.integers(0, 7)))


@pytest.mark.parametrize("B,page,new_hi,words", [(1, 16, 1, 1), (5, 16, 12, 1), (48, 16, 64, 1), (9, 3, 130, 3), (20, 32, 256, 4)])
def test_step_tables_with_trees(B, page, new_hi, words):
    rng = np.random.default_rng(B)
    args = make_tables(rng, B, page, 300, new_hi, 3000)
    parents = np.concatenate([[rng.integers(-1, i) if i else -1 for i in range(n)] for n in args[1]] + [[-1] * 5])
    check_tables(*args, page, sum(args[1]) + 5, parents.astype(np.int32), words)


def test_step_tables_chain_is_causal():
    ctx, new, held, table, free, count = [5, 0], [64, 33], [1, 0], np.zeros((2, 8), np.int32), np.arange(20, dtype=np.int32), 20
    parents = [i - 1 for i in range(64)] + [i - 1 for i in range(33)]
    t, _, _ = run_tables(ctx, new, held, table, free, count, 16, 97, parents)
    want = [(1 << (i + 1)) - 1 for n in new for i in range(n)]
    assert [int(m) & (2 ** 64 - 1) for m in t.tree_mask[:, 0].cpu()] == want
    assert t.positions.cpu().tolist() == list(range(5, 69)) + list(range(33))


def test_step_tables_refusals_on_the_device():
    # request 1 is too wide, request 2 finds too few pages, request 3 needs none and is served, request 4 waits
    table = np.arange(5 * 4, dtype=np.int32).reshape(5, 4)
    ref = check_tables([10, 60, 16, 3, 16], [6, 20, 40, 2, 16], [1, 4, 1, 1, 1], table, np.arange(100, 110, dtype=np.int32), 1, 16, 84)
    assert ref["status"] == [0, paged.TOO_WIDE, paged.NO_PAGES, 0, paged.NO_PAGES]
    # the same with trees, a parent that is no earlier token, and a tree past its mask
    parents = np.full(84 + 70, -1, np.int32)
    parents[3] = 3
    check_tables([10, 60, 16, 3, 16], [6, 20, 40, 2, 16], [1, 4, 1, 1, 1], table, np.arange(100, 110, dtype=np.int32), 1, 16, 84,
                 parents[:84])
    ref = check_tables([0], [70], [5], np.arange(5, dtype=np.int32)[None], np.zeros(0, np.int32), 0, 16, 70, parents[84:])
    assert ref["status"] == [paged.BIG_TREE]


def test_step_tables_finished_requests_feed_the_others():
    """Pages that come back in a call serve the same call; the stack carries over to the next one."""
    table = np.array([[4, 5, 6, 7], [1, 0, 0, 0]], np.int32)
    ref = check_tables([0, 16], [0, 40], [4, 1], table, np.full(8, -1, np.int32), 0, 16, 40)
    assert ref["table"][1].tolist() == [1, 7, 6, 5] and ref["count"] == 1 and ref["free"][0] == 4


def test_step_tables_over_several_steps():
    """Lifecycle: grow, reject drafts, finish, start; no page is ever held twice or lost."""
    rng = np.random.default_rng(3)
    B, page, W, pages = 12, 4, 10, 90
    i32 = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device=DEV)
    table, free = i32(np.zeros((B, W))), i32(rng.permutation(pages))
    held, count, ctx = i32([0] * B), i32([pages]), [0] * B
    for step in range(30):
        new = rng.integers(0, 9, B).tolist()
        for b in range(B):
            if rng.random() < 0.15 or ctx[b] + new[b] > page * W:
                ctx[b] = 0 if rng.random() < 0.5 else ctx[b]
                new[b] = min(new[b], page * W - ctx[b])
        t = paged.step_tables(i32(ctx), i32(new), held, table, free, count, page, sum(new))
        held, count = t.held_pages, t.free_count
        h, c = held.cpu().tolist(), int(count)
        owned = [int(p) for b in range(B) for p in table[b, :h[b]].cpu()] + free[:c].cpu().tolist()
        assert sorted(owned) == list(range(pages))
        live = [s for s in t.slots.cpu().tolist() if s >= 0]
        assert len(set(live)) == len(live)
        ok = (t.status.cpu().numpy() == 0)
        ctx = [c0 + int(rng.integers(0, n + 1)) if o else c0 for c0, n, o in zip(ctx, new, ok)]


# ------------------------------------------------------------------------------------------------
# store
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("N,heads,dim,page", [(1, 1, 8, 1), (5, 8, 128, 16), (100, 3, 80, 7), (777, 2, 256, 64), (64, 16, 64, 32)])
def test_store_kv(N, heads, dim, page, dtype):
    g = torch.Generator().manual_seed(N)
    pages = N // page + 3
    qkv = torch.randn(N, heads * 4, dim, generator=g).to(dtype).to(DEV)
    k, v = qkv[:, heads:2 * heads], qkv[:, 2 * heads:3 * heads]      # slices of a fused projection
    slots = torch.randperm(pages * page, generator=g)[:N]
    slots[::7] = -1
    if N > 5:
        slots[1] = pages * page                                      # outside the cache: nothing is stored
    for layout in ("slots", "heads", "joint"):
        if layout == "heads":                                        # [pages, heads, page, dim] underneath
            caches = [torch.full((pages, heads, page, dim), float(i), dtype=dtype, device=DEV).transpose(1, 2) for i in range(2)]
        elif layout == "joint":                                      # keys and values of a page side by side
            both = torch.zeros(pages, 2, page, heads, dim, dtype=dtype, device=DEV)
            caches = [both[:, 0], both[:, 1]]
        else:
            caches = [torch.full((pages, page, heads, dim), float(i), dtype=dtype, device=DEV) for i in range(2)]
        want = [c.clone(memory_format=torch.contiguous_format) for c in caches]
        for t, s in enumerate(slots.tolist()):
            if 0 <= s < pages * page:
                want[0][s // page, s % page], want[1][s // page, s % page] = k[t], v[t]
        paged.store_kv(k, v, slots.to(DEV), *caches)
        assert all(torch.equal(c, w) for c, w in zip(caches, want)), layout


def test_store_keeps_bits():
    """Copies, not conversions: NaN payloads, infinities, signed zeros and subnormals arrive as they are."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(64, 8, 128).to(DEV)
    k = bits.view(torch.float16)
    kc, vc = (torch.zeros(4, 16, 8, 128, dtype=torch.float16, device=DEV) for _ in range(2))
    paged.store_kv(k, k.flip(0), torch.arange(64, device=DEV), kc, vc)
    assert torch.equal(kc.view(torch.int16).view(64, 8, 128), bits) and torch.equal(vc.view(torch.int16).view(64, 8, 128), bits.flip(0))


def test_store_nothing():
    kc, vc = (torch.ones(2, 4, 1, 16, dtype=torch.float16, device=DEV) for _ in range(2))
    empty = torch.zeros(0, 1, 16, dtype=torch.float16, device=DEV)
    paged.store_kv(empty, empty, torch.zeros(0, dtype=torch.int64, device=DEV), kc, vc)
    assert float(kc.min()) == 1.0


# ------------------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------------------
def build(ctx, new, heads, kv_heads, dim, page, dtype, seed=0, tree=True, words=1, layout="slots", extra_pages=2, q_scale=1.0):
    g = torch.Generator().manual_seed(seed)
    rng = np.random.default_rng(seed)
    need = [-(-(c + n) // page) for c, n in zip(ctx, new)]
    pages = sum(need) + extra_pages
    shape = (pages, kv_heads, page, dim) if layout == "heads" else (pages, page, kv_heads, dim)
    kc, vc = (torch.randn(shape, generator=g).to(dtype).to(DEV) for _ in range(2))
    if layout == "heads":
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    ids = rng.permutation(pages).astype(np.int32)
    table = np.zeros((len(ctx), max(need + [1])), np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    N = sum(new)
    q = (q_scale * torch.randn(N, heads, dim, generator=g)).to(dtype).to(DEV)
    mask = None
    if tree:
        bits = np.zeros((N, words), np.uint64)
        base = 0
        for n in new:
            for i in range(n):
                up = int(rng.integers(-1, i)) if i else -1
                if up >= 0:
                    bits[base + i] = bits[base + up]
                bits[base + i, i // 64] |= np.uint64(1 << (i % 64))
            base += n
        mask = torch.from_numpy(bits.view(np.int64)).to(DEV)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    return dict(q=q, kc=kc, vc=vc, table=torch.from_numpy(table).to(DEV), seq=i32([c + n for c, n in zip(ctx, new)]),
                cu=i32([0] + np.cumsum(new).tolist()), mask=mask, ctx=ctx, new=new)


def reference(s, scale=None):
    """(out, bound, lse) in 64 bits."""
    q, kc, vc = s["q"].cpu().double(), s["kc"].cpu().double(), s["vc"].cpu().double()
    page, kv, dim = kc.shape[1:]
    heads = q.shape[1]
    scale = dim ** -0.5 if scale is None else scale
    u = HALF_UNIT[s["q"].dtype]
    out, bound, lse = torch.zeros_like(q), torch.zeros_like(q), torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    table, base = s["table"].cpu().long(), 0
    for b, (c, n) in enumerate(zip(s["ctx"], s["new"])):
        pos = torch.arange(c + n)
        k, v = kc[table[b][pos // page], pos % page], vc[table[b][pos // page], pos % page]
        for i in range(n):
            if s["mask"] is None:
                seen = list(range(c + i + 1))
            else:
                word = [int(w) & (2 ** 64 - 1) for w in s["mask"][base + i].cpu()]
                seen = list(range(c)) + [c + j for j in range(n) if j // 64 < len(word) and word[j // 64] >> (j % 64) & 1]
            if not seen:
                continue
            ks, vs = k[seen].repeat_interleave(heads // kv, 1), v[seen].repeat_interleave(heads // kv, 1)
            score = torch.einsum("hd,khd->hk", q[base + i], ks) * scale
            w = torch.softmax(score, 1)
            o, A = torch.einsum("hk,khd->hd", w, vs), torch.einsum("hk,khd->hd", w, vs.abs())
            e = (dim / 16 + 8) * 2.0 ** -22 * abs(scale) * torch.einsum("hd,khd->hk", q[base + i].abs(), ks.abs()).amax(1) + 2.0 ** -21
            lost = len(seen) * 2.0 ** -24 * vs.abs().amax() if s["q"].dtype == torch.float16 else 0.0
            out[base + i], lse[base + i] = o, torch.logsumexp(score, 1)
            bound[base + i] = (2 * u + 2 * e[:, None] + (len(seen) / 16 + 64) * 2.0 ** -22) * A + u * o.abs() + lost + 1e-7
        base += n
    return out, bound, lse


def attend(s, **kw):
    return paged.tree_attention(s["q"], s["kc"], s["vc"], s["table"], s["seq"], s["cu"], max(s["new"] + [0]), tree_mask=s["mask"], **kw)


def check(s, what="", scale=None):
    out, lse = attend(s, return_lse=True, scale=scale)
    assert paged.read_status() == 0, what    # no device wait ran out
    ref, bound, ref_lse = reference(s, scale)
    over = (out.cpu().double() - ref).abs() - bound
    assert not torch.isnan(out).any(), what
    assert bool((over <= 0).all()), f"{what}: over the bound by {float(over.max())}"
    fin = torch.isfinite(ref_lse)
    assert torch.equal(torch.isfinite(lse.cpu()), fin), what
    # the sum is over rounded weights: half a unit relative, plus the scores' error
    assert float((lse.cpu().double() - ref_lse)[fin].abs().max() if fin.any() else 0) < 2 * HALF_UNIT[s["q"].dtype] + 1e-3, what
    return out


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim", [(1, 1, 64), (8, 8, 128), (8, 2, 128), (12, 4, 80), (5, 1, 64), (16, 1, 128), (40, 8, 128),
                                          (4, 2, 256), (6, 3, 192), (8, 1, 256), (2, 2, 8), (3, 1, 96)])
def test_attention_heads(heads, kv, dim, dtype):
    check(build([70, 3, 0, 129], [5, 1, 4, 9], heads, kv, dim, 16, dtype, seed=heads + dim))


@pytest.mark.parametrize("page", [1, 7, 16, 24, 64, 128])
@pytest.mark.parametrize("tree", [True, False])
def test_attention_pages_and_lengths(page, tree):
    """Contexts around tile and page ends, pages that end inside a tile, one token to a whole tree."""
    ctx = [0, 1, 15, 16, 17, 62, 63, 64, 65, 127, 128, 200, 500]
    new = [1, 64, 1, 3, 2, 1, 2, 3, 40, 1, 64, 7, 5]
    check(build(ctx, new, 4, 2, 64, page, torch.bfloat16, seed=page, tree=tree), f"page {page}")


@pytest.mark.parametrize("dim,heads,kv", [(64, 8, 2), (128, 8, 1), (128, 4, 4), (256, 4, 1)])
def test_attention_long_and_split(dim, heads, kv):
    """Few requests with long contexts: every segment is split over many CTAs and joined."""
    check(build([3000, 1777], [3, 1], heads, kv, dim, 32, torch.float16, seed=dim))
    check(build([5000], [1], heads, kv, dim, 16, torch.bfloat16, seed=dim + 1, tree=False))


@pytest.mark.parametrize("new,words", [([130, 1], 3), ([256, 65], 4), ([100], 2)])
def test_attention_trees_past_one_word(new, words):
    check(build([30, 200][:len(new)], new, 4, 2, 64, 16, torch.float16, seed=words, words=words))


def test_attention_causal_chunks():
    """No mask: prompt chunks longer than a tile, and past the first context."""
    check(build([0, 100, 37], [200, 70, 1], 4, 2, 128, 16, torch.bfloat16, tree=False))


def test_attention_large_scores():
    check(build([300], [6], 4, 1, 128, 16, torch.float16, q_scale=20.0))
    check(build([300], [6], 4, 1, 128, 16, torch.bfloat16, q_scale=1.0), scale=0.5)
    check(build([300], [6], 4, 1, 64, 16, torch.bfloat16), scale=-0.2)


def test_rows_that_see_nothing_are_zero():
    s = build([0, 0, 40], [5, 1, 2], 4, 2, 64, 16, torch.float16, seed=4)
    s["mask"][0] = 0
    s["mask"][3] = 0
    s["mask"][5] = 0
    s["mask"][6] = 0
    out = check(s)
    assert float(out[[0, 3, 5]].abs().max()) == 0.0 and float(out[6].abs().min()) > 0.0


def test_mask_bits_past_the_tree_are_ignored():
    s = build([10, 20], [3, 5], 4, 2, 64, 16, torch.float16, seed=5)
    want = attend(s)
    s["mask"][:3] |= ~7
    assert torch.equal(attend(s), want)


@pytest.mark.parametrize("tree", [True, False])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim,new", [(4, 2, 64, [6, 3]), (8, 1, 128, [9, 4]), (2, 1, 256, [7, 1]), (16, 2, 128, [20, 11])])
def test_unseen_infinities_and_nan_do_not_spread(heads, kv, dim, new, dtype, tree):
    """NaN and infinities in unused slots, unused pages and in new tokens: only rows that see them notice."""
    s = build([70, 16], new, heads, kv, dim, 16, dtype, seed=dim, tree=tree)
    clean = attend(s)
    used = torch.zeros(s["kc"].shape[:2], dtype=torch.bool, device=DEV)
    for b, (c, n) in enumerate(zip(s["ctx"], s["new"])):
        pos = torch.arange(c + n, device=DEV)
        used[s["table"][b].long()[pos // 16], pos % 16] = True
    for c in (s["kc"], s["vc"]):
        c[~used] = float("nan")
    assert torch.equal(attend(s), clean)
    # the second new token of request 0: keys NaN, values NaN and infinite
    at = s["ctx"][0] + 1
    page, off = int(s["table"][0, at // 16]), at % 16
    seen = torch.tensor([(i >= 1) if s["mask"] is None else bool(int(s["mask"][i, 0]) >> 1 & 1) for i in range(new[0])] + [False] * new[1])
    for value in (float("nan"), float("inf"), -float("inf")):
        old = s["vc"][page, off].clone()
        s["vc"][page, off, :, 3] = value
        got = attend(s).cpu()
        assert torch.equal(got[~seen], clean.cpu()[~seen])
        hit = got[seen][:, :, 3]
        assert bool((torch.isnan(hit) if math.isnan(value) else hit == value).all())
        same = [d for d in range(dim) if d != 3]
        assert torch.equal(got[seen][:, :, same], clean.cpu()[seen][:, :, same])
        s["vc"][page, off] = old
    s["kc"][page, off] = float("nan")
    got = attend(s).cpu()
    assert torch.equal(got[~seen], clean.cpu()[~seen]) and bool(torch.isnan(got[seen]).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim,page,new", [(4, 2, 64, 16, [6, 3]), (8, 1, 128, 7, [9, 4]), (2, 1, 256, 16, [7, 1]),
                                                   (16, 2, 128, 32, [20, 11]), (4, 4, 128, 64, [3, 2])])
def test_nan_in_the_context_reaches_every_row(heads, kv, dim, page, new, dtype):
    """A value that every row sees: in a whole tile of the context, and in the tile that the new tokens share."""
    s = build([300, 16], new, heads, kv, dim, page, dtype, seed=dim)
    clean = attend(s)
    for at in (5, 290):
        pg, off = int(s["table"][0, at // page]), at % page
        old = s["vc"][pg, off].clone()
        s["vc"][pg, off, :, 3] = float("nan")
        got = attend(s)
        assert bool(torch.isnan(got[:new[0], :, 3]).all()), at
        same = [d for d in range(dim) if d != 3]
        assert torch.equal(got[:, :, same], clean[:, :, same]) and torch.equal(got[new[0]:], clean[new[0]:])
        s["vc"][pg, off] = old


def test_refused_requests_are_zero_and_do_not_disturb():
    s = build([70, 30, 50], [4, 6, 2], 8, 2, 128, 16, torch.bfloat16, seed=6)
    clean = attend(s)
    s["seq"][1] = 0
    got, lse = attend(s, return_lse=True)
    assert float(got[4:10].abs().max()) == 0.0 and bool((lse[4:10] == -math.inf).all())
    assert torch.equal(got[:4], clean[:4]) and torch.equal(got[10:], clean[10:])
    s["seq"][1] = 10 ** 9                       # longer than the table: nothing outside it is read
    assert float(attend(s)[4:10].abs().max()) == 0.0
    s["seq"][1] = 36
    s["table"][1, 0] = 10 ** 6                  # not a page of the cache: read as zeros, no fault
    assert bool(torch.isfinite(attend(s)).all())


def test_requests_without_new_tokens():
    s = build([70, 30, 50, 9, 9], [0, 6, 0, 2, 0], 8, 2, 64, 16, torch.float16, seed=7)
    check(s)
    s = build([7, 8], [0, 0], 8, 2, 64, 16, torch.float16, seed=7)
    assert attend(s).shape == (0, 8, 64)


@pytest.mark.parametrize("page,layout", [(16, "heads"), (128, "heads"), (256, "slots"), (256, "heads"), (24, "heads"), (8, "slots")])
def test_cache_layouts_and_page_sizes(page, layout):
    check(build([70, 300, 0], [5, 9, 20], 8, 2, 128, page, torch.float16, seed=page, layout=layout), f"{page} {layout}")
    check(build([70, 300, 0], [5, 9, 20], 4, 1, 64, page, torch.bfloat16, seed=page, layout=layout), f"{page} {layout}")


@pytest.mark.parametrize("dim", [136, 192, 200, 256])
@pytest.mark.parametrize("page,layout", [(8, "slots"), (64, "heads"), (192, "slots"), (24, "slots"), (1, "heads")])
def test_head_sizes_over_128(dim, page, layout):
    """Up to 32, 64, 128 and more rows to a KV head, whole requests and split ones, tiles of 64 keys that pages end in."""
    dtype = torch.float16 if page == 8 else torch.bfloat16
    check(build([63, 300, 0, 64], [5, 1, 8, 3], 8, 2, dim, page, dtype, seed=dim + page, layout=layout), f"{dim} {page} 32 rows")
    check(build([1000, 127], [30, 33], 2, 1, dim, page, dtype, seed=dim, layout=layout), f"{dim} {page} 66 rows")
    check(build([128, 65], [12, 15], 4, 1, dim, page, dtype, seed=page, layout=layout), f"{dim} {page} 60 rows")
    check(build([190, 1], [64, 40], 5, 1, dim, page, dtype, seed=page, layout=layout), f"{dim} {page} 320 rows")


@pytest.mark.parametrize("requests,ctx,new,heads,dim", [
    (1, 9000, 3, 2, 64), (3, 1500, 10, 5, 128),        # few segments: parts of 4 tiles
    (40, 2500, 1, 4, 64), (44, 1100, 2, 3, 192),       # more: parts of 8
    (50, 3900, 1, 4, 64), (60, 1300, 1, 1, 256),       # runs of the line, several segments to a CTA
    (200, 120, 1, 4, 128), (140, 1000, 1, 2, 64)])     # whole segments, more and fewer than the processors
def test_cuts_of_the_work(requests, ctx, new, heads, dim):
    lens = [max(ctx - 97 * (b % 5) + 13 * (b % 3), 0) for b in range(requests)]
    check(build(lens, [new] * requests, heads, 1, dim, 64, torch.float16, seed=requests), f"{requests} x {ctx}")


def test_keys_and_values_side_by_side():
    """Both caches as slices of one tensor: equal strides, neither contiguous."""
    s = build([70, 200], [5, 9], 8, 2, 128, 16, torch.float16, seed=21)
    want = check(s)
    both = torch.stack((s["kc"], s["vc"]), 1)
    assert torch.equal(attend(dict(s, kc=both[:, 0], vc=both[:, 1])), want)


def test_strided_query_output_and_head_major_cache():
    s = build([70, 200], [5, 9], 8, 2, 128, 16, torch.bfloat16, seed=8, layout="heads")
    want = check(s)
    fused = torch.randn(14, 14, 128, device=DEV).bfloat16()
    fused[:, 2:10] = s["q"]
    buf = torch.zeros(14, 20, 128, dtype=torch.bfloat16, device=DEV)
    s2 = dict(s, q=fused[:, 2:10], kc=s["kc"], vc=s["vc"])
    got = attend(s2, out=buf[:, 4:12])
    assert torch.equal(got, want) and float(buf[:, :4].abs().max()) == 0 and float(buf[:, 12:].abs().max()) == 0
    odd = torch.empty(14 * 8 * 128 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(14, 8, 128)
    odd.copy_(s["q"])
    assert torch.equal(attend(dict(s, q=odd)), want)


def test_offsets_past_32_bits():
    """Pages whose elements lie past 2^31."""
    pages, page, kv, dim = 70000, 64, 4, 128
    if torch.cuda.mem_get_info()[0] < 24e9:
        pytest.skip("needs 24 GB of free device memory")
    s = build([100, 30], [4, 2], 8, kv, dim, page, torch.float16, seed=9)
    want = attend(s)
    big = [torch.empty(pages, page, kv, dim, dtype=torch.float16, device=DEV) for _ in range(2)]
    n = s["kc"].shape[0]
    for b, small in zip(big, (s["kc"], s["vc"])):
        b[-n:] = small
    moved = dict(s, kc=big[0], vc=big[1], table=s["table"] + (pages - n))
    assert torch.equal(attend(moved), want)
    k = torch.randn(2, kv, dim, device=DEV).half()
    paged.store_kv(k, -k, torch.tensor([pages * page - 1, pages * page - 70], device=DEV), *big)
    assert torch.equal(big[0][-1, -1], k[0]) and torch.equal(big[1].view(-1, kv, dim)[-70], -k[1])


def test_repeats_bit_identically_on_other_streams_and_in_a_graph():
    s = build([900, 33, 2000], [5, 9, 1], 8, 2, 128, 16, torch.float16, seed=10)
    want = attend(s)
    for _ in range(5):
        assert torch.equal(attend(s), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = attend(s)
        graph = torch.cuda.CUDAGraph()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    side.synchronize()
    with torch.cuda.graph(graph, stream=side):
        out = attend(s)
    s["q"].mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, attend(s))


def test_many_requests():
    rng = np.random.default_rng(11)
    check(build(rng.integers(0, 90, 300).tolist(), rng.integers(0, 4, 300).tolist(), 2, 1, 64, 16, torch.bfloat16, seed=11))


def test_tables_store_and_attention_run_a_step():
    """step_tables -> store_kv -> tree_attention agrees with attention over the same tokens laid out by hand."""
    B, page, kv, heads, dim = 3, 16, 2, 8, 64
    ctx, new = [40, 0, 17], [6, 3, 1]
    g = torch.Generator().manual_seed(12)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    held = [-(-c // page) for c in ctx]
    table, free = torch.zeros(B, 8, dtype=torch.int32, device=DEV), torch.arange(20, dtype=torch.int32, device=DEV).flip(0).contiguous()
    t0 = paged.step_tables(i32([0] * B), i32(ctx), i32([0] * B), table, free, i32([20]), page, sum(ctx))
    kc, vc = (torch.full((20, page, kv, dim), float("nan"), dtype=torch.float16, device=DEV) for _ in range(2))
    old = torch.randn(2, sum(ctx), kv, dim, generator=g).half().to(DEV)
    paged.store_kv(old[0], old[1], t0.slots, kc, vc)
    parents = i32([-1, 0, 0, 1, 1, 2, -1, -1, 0, -1])
    t = paged.step_tables(i32(ctx), i32(new), t0.held_pages, table, free, t0.free_count, page, 10, parents=parents)
    qkv = torch.randn(10, heads + 2 * kv, dim, generator=g).half().to(DEV)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    paged.store_kv(k, v, t.slots, kc, vc)
    s = dict(q=q, kc=kc, vc=vc, table=table, seq=t.seq_lens, cu=t.cu_lens, mask=t.tree_mask, ctx=ctx, new=new)
    check(s)
    assert t.positions.cpu().tolist() == [40, 41, 41, 42, 42, 42, 0, 0, 1, 17]
    assert t.held_pages.cpu().tolist() == [3, 1, 2] and int(t.free_count) == 14 and held == t0.held_pages.cpu().tolist()


def test_refusals():
    s = build([20], [3], 4, 2, 64, 16, torch.float16)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    att = lambda **kw: attend(dict(s, **kw))
    odd_heads = torch.zeros(3, 5, 64, dtype=torch.float16, device=DEV)
    wide = torch.zeros(9, 16, 2, 264, dtype=torch.float16, device=DEV)
    k = torch.zeros(3, 2, 64, dtype=torch.float16, device=DEV)
    slots = torch.zeros(3, dtype=torch.int64, device=DEV)
    tab = lambda **kw: paged.step_tables(**dict(dict(context_lens=i32([1, 2]), new_lens=i32([1, 1]), held_pages=i32([1, 1]),
                                                     block_table=i32([[0, 1], [1, 2]]), free_pages=i32([3, 4]), free_count=i32([2]),
                                                     page_size=16, num_tokens=2), **kw))
    for bad in (lambda: att(q=odd_heads), lambda: att(q=s["q"].bfloat16()), lambda: att(q=s["q"].float()), lambda: att(q=s["q"][:, :, :56]),
                lambda: att(kc=s["kc"].float(), vc=s["vc"].float()), lambda: att(kc=s["kc"][:-1]), lambda: att(table=s["table"].long()),
                lambda: att(seq=s["seq"].long()), lambda: att(cu=s["cu"][:1]), lambda: att(mask=s["mask"].int()), lambda: att(mask=s["mask"][:2]),
                lambda: att(kc=s["kc"][..., ::2], vc=s["vc"][..., ::2], q=s["q"][..., ::2]), lambda: att(mask=s["mask"].repeat(1, 5)),
                lambda: att(q=torch.zeros(3, 4, 264, dtype=torch.float16, device=DEV), kc=wide, vc=wide),
                lambda: attend(s, scale=float("nan")), lambda: attend(s, out=torch.empty(3, 4, 64, device=DEV)),
                lambda: paged.store_kv(k, k.bfloat16(), slots, s["kc"], s["vc"]), lambda: paged.store_kv(k, k[:2], slots, s["kc"], s["vc"]),
                lambda: paged.store_kv(k, k, slots.int(), s["kc"], s["vc"]), lambda: paged.store_kv(k, k, slots, s["kc"], s["vc"].bfloat16()),
                lambda: tab(new_lens=i32([1])), lambda: tab(context_lens=torch.zeros(2, dtype=torch.int32)), lambda: tab(page_size=0),
                lambda: tab(num_tokens=-1), lambda: tab(parents=i32([0])), lambda: tab(parents=i32([-1, -1]), mask_words=5),
                lambda: tab(block_table=i32([[0, 1]])), lambda: tab(free_count=i32([1, 2])), lambda: tab(context_lens=i32([]))):
        with pytest.raises((ValueError, TypeError, Dsv41Error)):
            bad()
    assert torch.equal(attend(s), attend(s))    # the refusals left everything usable
