"""The paged operators where inputs are at their ends, against plain restatements in 64 bits, with the bounds of
test_gpu_paged.py."""
import math

import numpy as np
import pytest
import torch

from dsv41_flash_offload_b200 import Dsv41Error, paged
from test_gpu_paged import DEV, HALF_UNIT, attend, build, reference, run_tables

pytestmark = pytest.mark.gpu


def nonfinite_reference(s, scale=None):
    """The definition in 64 bits, key by key: what a row sees of infinities and NaN, and nothing else."""
    q, kc, vc = (s[n].cpu().double() for n in ("q", "kc", "vc"))
    page, kv, dim = kc.shape[1:]
    rep, scale = q.shape[1] // kv, dim ** -0.5 if scale is None else scale
    out, table, base = torch.zeros_like(q), s["table"].cpu().long(), 0
    for b, (c, n) in enumerate(zip(s["ctx"], s["new"])):
        pos = torch.arange(c + n)
        k, v = kc[table[b][pos // page], pos % page], vc[table[b][pos // page], pos % page]
        for i in range(n):
            word = (1 << (i + 1)) - 1 if s["mask"] is None else int(s["mask"][base + i, 0])
            seen = list(range(c)) + [c + j for j in range(n) if word >> j & 1]
            for h in range(q.shape[1]):
                w = torch.softmax(k[seen, h // rep] @ q[base + i, h] * scale, 0)
                out[base + i, h] = (w[:, None] * v[seen, h // rep]).sum(0)
        base += n
    return out


def check_nonfinite(s, clean, what=""):
    got, want = attend(s).cpu(), nonfinite_reference(s)
    assert paged.read_status() == 0, what
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf].double(), want[inf]), what
    fin = torch.isfinite(want)
    assert torch.equal(got[fin], clean.cpu()[fin]), what    # nothing else changes, to the bit


ROWS = [(4, 2, 64, 16, [6, 3]), (2, 1, 128, 7, [9, 4]), (4, 1, 256, 16, [7, 1]),     # up to 32 rows
        (16, 2, 128, 32, [8, 3]), (4, 1, 80, 24, [13, 2]), (8, 1, 192, 64, [7, 5]),  # up to 64
        (16, 2, 128, 16, [12, 3]), (8, 1, 256, 8, [16, 2]),                          # up to 128
        (16, 1, 128, 64, [15, 9]), (8, 1, 64, 7, [30, 1]),                           # more
        (4, 2, 72, 16, [5, 3]), (8, 1, 200, 16, [9, 2]), (2, 2, 8, 32, [6, 1])]      # columns that end inside a block


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim,page,new", ROWS)
@pytest.mark.parametrize("tree", [True, False])
def test_infinities_of_the_context(heads, kv, dim, page, new, tree, dtype):
    """In a whole tile of the context and in the tile that the new tokens share; alone, against one of the other sign,
    and with NaN in another column."""
    s = build([300, 16], new, heads, kv, dim, page, dtype, seed=dim + heads, tree=tree)
    clean = attend(s)

    def put(at, column, value):
        s["vc"][int(s["table"][0, at // page]), at % page, :, column] = value

    keep = s["vc"].clone()
    for puts in ([(5, 3, math.inf)], [(290, 3, -math.inf)], [(5, 3, -math.inf), (200, 3, -math.inf), (290, dim - 1, math.inf)],
                 [(17, 3, math.inf), (133, 3, -math.inf), (40, 4, math.nan), (301, 4, math.inf)],
                 [(131, 7, math.inf), (300, 7, -math.inf)], [(131, slice(None, None, 2), math.inf), (300, slice(None), -math.inf)]):
        for p in puts:
            put(*p)
        check_nonfinite(s, clean, str(puts))
        s["vc"].copy_(keep)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim,page,new", ROWS[::3])
def test_infinities_under_vanishing_weights(heads, kv, dim, page, new, dtype):
    """Weights that are zero in 16 bits, or in 32, are not zero: an infinity under them is one in the row. Scores spread
    over some hundreds, within what 64 bits hold."""
    s = build([300, 16], new, heads, kv, dim, page, dtype, seed=dim, q_scale=60.0)
    clean = attend(s)
    for at, value in ((5, math.inf), (255, -math.inf), (299, math.inf), (301, -math.inf)):
        keep = s["vc"].clone()
        s["vc"][int(s["table"][0, at // page]), at % page, :, 2] = value
        check_nonfinite(s, clean, f"{at} {value}")
        s["vc"].copy_(keep)


@pytest.mark.parametrize("heads,dim,new", [(1, 64, 3), (8, 128, 5), (8, 128, 13), (4, 256, 33)])
def test_infinities_in_a_split_request(heads, dim, new):
    """The parts of a request that several processors share: one part's infinities, and parts of which one has all the weight."""
    for q_scale in (1.0, 60.0):
        s = build([6000], [new], heads, 1, dim, 16, torch.bfloat16, seed=dim, q_scale=q_scale)
        clean = attend(s)
        for puts in ([(3, 1, math.inf)], [(2500, 1, -math.inf)], [(700, 0, math.inf), (5400, 0, -math.inf), (5999, 9, math.inf)]):
            keep = s["vc"].clone()
            for at, column, value in puts:
                s["vc"][int(s["table"][0, at // 16]), at % 16, :, column] = value
            check_nonfinite(s, clean, str(puts))
            s["vc"].copy_(keep)


@pytest.mark.parametrize("heads,kv,dim,page,new", ROWS[::3])
def test_infinite_keys(heads, kv, dim, page, new):
    """A key with an infinity has the score +inf (the row is NaN) or -inf (weight zero; its value counts only where it is
    itself infinite, as NaN)."""
    s = build([300, 16], new, heads, kv, dim, page, torch.float16, seed=dim + 1)
    for value_too in (False, True):
        for at in (7, 293):
            keep = s["kc"].clone(), s["vc"].clone()
            page_id = int(s["table"][0, at // page])
            s["kc"][page_id, at % page, :, 1] = math.inf
            if value_too:
                s["vc"][page_id, at % page, :, 5] = math.inf
            got, want = attend(s).cpu(), nonfinite_reference(s)
            assert torch.equal(torch.isnan(got), torch.isnan(want))
            fin = torch.isfinite(want)
            s["kc"].copy_(keep[0])
            s["vc"].copy_(keep[1])
            # finite rows: those without this key, with the bound of one more or less of them
            assert float((got.double() - want)[fin].abs().max()) < 8 * HALF_UNIT[torch.float16] * float(want[fin].abs().max())


@pytest.mark.parametrize("heads,dim,new", [(4, 64, 4), (16, 128, 4), (16, 128, 20)])
def test_a_cache_full_of_infinities(heads, dim, new):
    """Many infinities are no slower than a bounded wait allows."""
    s = build([20000, 100], [new, 2], heads, 1, dim, 64, torch.float16, seed=dim)
    s["vc"][..., 0] = math.inf
    s["vc"][..., 1] = -math.inf
    s["vc"][..., 2] = math.nan
    got = attend(s)
    assert paged.read_status() == 0
    assert bool((got[..., 0] == math.inf).all()) and bool((got[..., 1] == -math.inf).all()) and bool(torch.isnan(got[..., 2]).all())
    assert bool(torch.isfinite(got[..., 3:]).all())


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_two_row_tiles_share_a_cleared_tile(page, dtype):
    """Rows of both row tiles, many times over: what one group of threads clears is cleared for the other's product too."""
    s = build([60, 190], [64, 61], 4, 1, 128, page, dtype, seed=page)
    clean = attend(s)
    hidden = []                                      # tokens that only few others see: leaves of their trees
    for b, base in ((0, 0), (1, 64)):
        bits = [int(w) for w in s["mask"][base:base + s["new"][b], 0]]
        leaves = [j for j in range(s["new"][b]) if sum(w >> j & 1 for w in bits) == 1]
        for j in leaves:
            at = s["ctx"][b] + j
            s["vc"][int(s["table"][b, at // page]), at % page] = math.nan
            hidden.append(base + j)
    rest = [i for i in range(125) if i not in hidden]
    for _ in range(30):
        got = attend(s)
        assert torch.equal(got[rest], clean[rest]) and bool(torch.isnan(got[hidden]).all())


@pytest.mark.parametrize("page", [8, 16, 24, 64, 128])
@pytest.mark.parametrize("dim", [64, 192])
def test_caches_that_repeat_in_memory(page, dim):
    """One KV head read by all, one slot for a whole page, one page for all: expanded views are what they show."""
    s = build([70, 300], [5, 9], 8, 2, dim, page, torch.float16, seed=page)
    pages = s["kc"].shape[0]
    for cut, full in ((lambda c: c[:, :, :1], (pages, page, 2, dim)), (lambda c: c[:, :1], (pages, page, 2, dim)),
                      (lambda c: c[:1], (pages, page, 2, dim))):
        views = {n: cut(s[n]).expand(full) for n in ("kc", "vc")}
        own = dict(s, **{n: v.contiguous() for n, v in views.items()})
        ref, bound, _ = reference(own)
        out = attend(dict(s, **views))
        assert bool(((out.cpu().double() - ref).abs() <= bound).all())


def test_outputs_that_repeat_in_memory_are_refused():
    s = build([20], [3], 4, 2, 64, 16, torch.float16)
    k = torch.zeros(3, 2, 64, dtype=torch.float16, device=DEV)
    slots = torch.arange(3, device=DEV)
    heads = torch.zeros(4, 16, 1, 64, dtype=torch.float16, device=DEV).expand(4, 16, 2, 64)
    tokens = torch.zeros(1, 4, 64, dtype=torch.float16, device=DEV).expand(3, 4, 64)
    for bad in (lambda: paged.store_kv(k, k, slots, heads, heads), lambda: attend(s, out=tokens)):
        with pytest.raises((ValueError, Dsv41Error)):
            bad()


def test_status_of_replays_and_recovery():
    """A wait that ran out is reported wherever its call ran, and the next call starts from clean counters."""
    s = build([900, 2000], [5, 9], 8, 2, 128, 16, torch.float16, seed=10)
    want = attend(s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attend(s)
        graph = torch.cuda.CUDAGraph()
    side.synchronize()
    with torch.cuda.graph(graph, stream=side):
        out = attend(s)
    buf = paged._ws[(torch.cuda.current_device(), side.cuda_stream, 128)][2]
    assert paged.read_status() == 0
    # what a call leaves that gave up: its status, and counters that are not zero
    words = buf[:2048].view(torch.int32)
    words[0] = 1
    words[64:72] = 3
    assert paged.read_status() == 1 and paged.read_status() == 0
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and paged.read_status() == 0


def test_status_of_a_device_by_name():
    s = build([20], [3], 4, 2, 64, 16, torch.float16)
    attend(s)
    words = paged._ws[(torch.cuda.current_device(), torch.cuda.current_stream().cuda_stream, 64)][2][:4].view(torch.int32)
    words[0] = 1
    assert paged.read_status("cuda") == 1 and paged.read_status("cuda:0") == 0 and paged.read_status(torch.device("cuda")) == 0


@pytest.mark.parametrize("dim", [64, 256])
def test_graphs_with_workspaces_of_their_own_replay_at_once(dim):
    """Two graphs captured on one stream that never ran a call, replayed together on two others, each with split requests."""
    cases = [build([3000 + 500 * i, 900], [5, 9], 8, 2, dim, 16, torch.float16, seed=20 + i) for i in range(2)]
    want = [attend(s) for s in cases]
    graphs, outs, spaces = [], [], [paged.attention_workspace(dim) for _ in cases]
    torch.cuda.synchronize()
    capture = torch.cuda.Stream()
    for s, w in zip(cases, spaces):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=capture):
            outs.append([attend(s, workspace=w) for _ in range(4)])
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(25):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for group, w in zip(outs, want) for o in group)
    assert [paged.read_status(workspace=w) for w in spaces] == [0, 0]
    spaces[1][:4].view(torch.int32)[0] = 1
    spaces[1][256:300] = 7
    assert paged.read_status() == 0 and paged.read_status(workspace=spaces[1]) == 1
    graphs[1].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[1]) for o in outs[1]) and paged.read_status(workspace=spaces[1]) == 0


@pytest.mark.filterwarnings("ignore:The CUDA Graph is empty")   # the refused capture
def test_a_reserved_stream_can_capture_at_once():
    s = build([900, 2000], [5, 9], 8, 2, 128, 16, torch.float16, seed=30)
    want = attend(s)
    stream = torch.cuda.Stream()
    paged._ws.pop((torch.cuda.current_device(), stream.cuda_stream, 128), None)   # (streams come from a pool)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="reserve_workspace"):
        with torch.cuda.graph(graph, stream=stream):
            attend(s)
    paged.reserve_workspace(128, stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = attend(s)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_workspaces_that_do_not_fit_are_refused():
    s = build([20], [3], 4, 2, 128, 16, torch.float16)
    full = paged.attention_workspace(128)
    assert torch.equal(attend(s, workspace=full), attend(s))
    for bad in (full[:-256], full[128:], full.view(torch.int32), full.cpu(), full[::2]):
        with pytest.raises((ValueError, Dsv41Error)):
            attend(s, workspace=bad)
    with pytest.raises(Dsv41Error):
        paged.attention_workspace(264)


def test_a_stack_without_room_loses_no_page():
    ctx, new, held = [0, 0, 0, 16], [0, 0, 0, 16], [2, 3, 1, 1]
    table = np.arange(16, dtype=np.int32).reshape(4, 4)
    for parents in (None, [-1] * 16):
        t, tb, fr = run_tables(ctx, new, held, table, np.array([50, 51, -1, -1, -1], np.int32), 2, 16, 16, parents)
        # request 0's two pages fit beside the two there, request 1's three do not, request 2 waits behind it
        assert t.held_pages.cpu().tolist() == [0, 3, 1, 2] and t.status.cpu().tolist() == [0, paged.NO_ROOM, paged.NO_ROOM, 0]
        assert tb[3, :2].cpu().tolist() == [12, 1] and int(t.free_count) == 3 and fr[:4].cpu().tolist() == [50, 51, 0, 1]
        assert t.seq_lens.cpu().tolist() == [0, 0, 0, 32] and t.slots.cpu().tolist() == [16 + i for i in range(16)]
    # more comes back than the stack holds, but the same call takes it again: nothing is kept back
    t, tb, _ = run_tables([0, 16], [0, 48], [4, 1], np.array([[4, 5, 6, 7], [1, 0, 0, 0]], np.int32), np.array([9, -1], np.int32), 1, 16, 48)
    assert t.status.cpu().tolist() == [0, 0] and t.held_pages.cpu().tolist() == [0, 4] and int(t.free_count) == 2
    assert tb[1].cpu().tolist() == [1, 7, 6, 5]


def test_no_page_is_lost_whatever_the_stack_holds():
    rng = np.random.default_rng(7)
    for case in range(60):
        B, page, W = int(rng.integers(1, 40)), int(rng.choice([1, 3, 16])), int(rng.integers(1, 12))
        ctx = rng.integers(0, page * W + 1, B)
        held = np.minimum(W, -(-ctx // page) + rng.integers(0, 4, B) * rng.integers(0, 2, B))
        ctx, new = ctx * (rng.random(B) > 0.3), rng.integers(0, 6, B)
        spare = int(rng.integers(0, 30))
        ids = rng.permutation(int(held.sum()) + spare).astype(np.int32)
        table, at = np.full((B, W), -7, np.int32), 0
        for b in range(B):
            table[b, :held[b]] = ids[at:at + held[b]]
            at += held[b]
        free = np.full(spare + int(rng.choice([0, 1, 5, 20])), -9, np.int32)
        free[:spare] = ids[at:]
        t, tb, fr = run_tables(ctx, new, held, table, free, spare, page, int(new.sum()))
        own = [int(p) for b in range(B) for p in tb[b, :int(t.held_pages[b])].cpu()] + fr[:int(t.free_count)].cpu().tolist()
        assert sorted(own) == list(range(len(ids))), case
        live = [s for s in t.slots.cpu().tolist() if s >= 0]
        assert len(set(live)) == len(live), case


def test_tokens_past_the_batch_are_refused():
    ctx, new, held = [5, 3, 0, 9], [3, 4, 2, 0], [1, 1, 0, 1]
    table = np.arange(16, dtype=np.int32).reshape(4, 4)
    for parents in (None, [-1] * 5):
        t, _, _ = run_tables(ctx, new, held, table, np.arange(90, 99, dtype=np.int32), 9, 16, 5, parents)
        assert t.status.cpu().tolist() == [0, paged.PAST_TOKENS, paged.PAST_TOKENS, 0]
        assert t.seq_lens.cpu().tolist() == [8, 0, 0, 9] and t.slots.cpu().tolist() == [5, 6, 7, -1, -1]
        assert t.held_pages.cpu().tolist() == [1, 1, 1, 1] and int(t.free_count) == 8


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim,ctx,new", [(4, 2, 64, [70, 3, 0, 129], [5, 1, 4, 9]), (16, 1, 128, [3000], [9]),
                                                  (8, 1, 256, [500, 20], [20, 3]), (4, 1, 128, [1500, 64], [64, 40])])
def test_sums_are_of_unrounded_weights(heads, kv, dim, ctx, new, dtype):
    """lse = m + log l: the scores' error e (as in test_gpu_paged.py), the fp32 sum's (keys / 16 + 64) * 2^-22, 2^-21 of the
    exponentials, and the result's own rounding with log2 and the change of base: 4 units of fp32."""
    s = build(ctx, new, heads, kv, dim, 16, dtype, seed=dim)
    _, lse = attend(s, return_lse=True)
    ref = reference(s)[2]
    q, k = s["q"].cpu().double().abs(), s["kc"].cpu().double().abs().amax((0, 1))
    e = (dim / 16 + 8) * 2.0 ** -22 * dim ** -0.5 * torch.einsum("nhd,hd->nh", q, k.repeat_interleave(heads // kv, 0))
    keys = max(c + n for c, n in zip(ctx, new))
    bound = e + (keys / 16 + 64) * 2.0 ** -22 + 2.0 ** -21 + 2.0 ** -21 * ref.abs()
    assert bool(((lse.cpu().double() - ref).abs() <= bound).all())


@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (16, 1, 128), (8, 1, 256)])
def test_a_scale_of_zero_counts_every_key_alike(heads, kv, dim):
    s = build([300, 0], [6, 4], heads, kv, dim, 16, torch.bfloat16, seed=3)
    ref, bound, ref_lse = reference(s, 0.0)
    out, lse = attend(s, scale=0.0, return_lse=True)
    assert bool(((out.cpu().double() - ref).abs() <= bound).all())
    assert float((lse.cpu().double() - ref_lse).abs().max()) <= 2.0 ** -18


@pytest.mark.parametrize("page", [24, 64])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_long_prompt_chunks(page, dtype):
    """No mask, 700 new tokens over an empty and a short context: many row tiles, those past the diagonal left out."""
    s = build([0, 150], [700, 333], 4, 2, 64, page, dtype, seed=page, tree=False)
    out = attend(s)
    ref, bound, _ = reference(s)
    assert paged.read_status() == 0
    assert bool(((out.cpu().double() - ref).abs() <= bound).all())
