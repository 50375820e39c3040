"""The operators together: drafted steps over a cache in 4 bits, through a window, and the scores of what comes out."""
import importlib.util
import os

import pytest
import torch

from conftest import ROOT
from dsv41_flash_offload_b200 import logprobs, paged, w4

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _example():
    spec = importlib.util.spec_from_file_location("draft_step", os.path.join(ROOT, "examples", "draft_step.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def test_steps_over_4_bits_are_steps_over_what_the_codes_stand_for():
    """A prompt, a drafted tree, an accepted path moved to its place, another tree: at each step the attention over the codes is,
    to the tree attention's rounding (P and the output, half a unit each, twice), that over a 16-bit cache that holds what
    load_kv4 reads."""
    ex = _example()
    g = torch.Generator().manual_seed(1)
    pages, page, kv, dim, heads = 40, 16, 2, 64, 8
    c4 = ex.PagedCache(2, pages, page, 10, kv, dim, bits=4)
    context = [0, 0]

    def step(new, parents, window=None, sinks=0):
        n = sum(new)
        t = c4.begin(i32(context), i32(new), n, None if parents is None else i32(parents))
        q, k, v = (torch.randn(n, h, dim, generator=g).half().to(DEV) for h in (heads, kv, kv))
        got = c4.attend(q, k, v, t, max(new), window=window, sinks=sinks)
        kc, vc = (x.view(pages, page, kv, dim) for x in paged.load_kv4(torch.arange(pages * page, device=DEV), c4.packed))
        want = paged.tree_attention(q, kc, vc, c4.block_table, t.seq_lens, t.cu_lens, max(new), tree_mask=t.tree_mask, window=window, sinks=sinks)
        scale = vc.abs().max()
        assert float((got.float() - want.float()).abs().max()) <= 4 * torch.finfo(torch.float16).eps * float(scale)
        return t, kc, vc

    step([33, 70], None)
    context = [33, 70]
    t, kc, vc = step([5, 3], [-1, 0, 0, 1, 3, -1, 0, 1], window=20, sinks=3)
    paths = [[0, 1, 3, 4], [5, 7]]
    src = [int(t.slots[i]) for path in paths for i in path]
    c4.keep(t, paths, i32(context))
    table = c4.block_table.cpu()
    dst = [int(table[b, (context[b] + j) // page]) * page + (context[b] + j) % page for b, path in enumerate(paths) for j in range(len(path))]
    now = paged.load_kv4(torch.tensor(dst, device=DEV), c4.packed)
    for a, b in zip(now, (kc, vc)):
        assert torch.equal(a, b.view(-1, kv, dim)[torch.tensor(src, device=DEV)])
    context = [37, 72]
    step([1, 6], [-1, -1, 0, 1, 2, 3, 4], window=40, sinks=1)
    assert paged.read_status() == 0


def test_a_step_in_a_graph_scores_its_tokens():
    """Store, attention, head and scores captured together, replayed for other lengths and other tokens."""
    kv, dim, heads, vocab, n, hidden = 2, 64, 8, 3001, 6, 512
    g = torch.Generator().manual_seed(2)
    cache = paged.Cache4(24, 16, kv, dim, dtype=torch.float16, device=DEV)
    head = w4.W4Weight.quantize((torch.randn(vocab, heads * dim, generator=g) * 0.05).half().to(DEV), 64)
    table = torch.randperm(24, generator=g).int().view(3, 8).to(DEV)
    draw = lambda *shape: torch.randn(*shape, generator=g).half().to(DEV)
    paged.store_kv4(draw(384, kv, dim), draw(384, kv, dim), torch.arange(384, device=DEV), cache)
    q, k, v = draw(n, heads, dim), draw(n, kv, dim), draw(n, kv, dim)
    tokens = torch.randint(0, vocab, (n, 2), generator=g).to(DEV)
    seq, cu, slots = i32([100, 33, 60]), i32([0, 2, 3, 6]), torch.arange(n, device=DEV) * 3
    assert hidden == heads * dim

    def step():
        paged.store_kv4(k, v, slots, cache)
        a = paged.tree_attention4(q, cache, table, seq, cu, 3, window=50, sinks=4)
        return w4.head_logprobs(a.view(n, -1), head, tokens, top=5)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step()
    for lengths in ([100, 33, 60], [7, 128, 3]):
        seq.copy_(i32(lengths))
        q.copy_(draw(n, heads, dim))
        tokens.copy_(torch.randint(0, vocab, (n, 2), generator=g))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    logits = w4.linear(paged.tree_attention4(q, cache, table, seq, cu, 3, window=50, sinks=4).view(n, -1), head, out_dtype=torch.float32)
    assert torch.equal(out.top_ids, logprobs.token_logprobs(logits, tokens, top=5).top_ids)
    assert bool((out.top_logprobs.diff(dim=1) <= 0).all()) and paged.read_status() == 0


@pytest.mark.parametrize("flags", [["--bits", "4"], ["--window", "24", "--sinks", "4"], ["--bits", "4", "--window", "9", "--sinks", "1"]])
def test_the_example_runs(flags, capsys, monkeypatch):
    monkeypatch.setattr("sys.argv", ["draft_step.py", "--steps", "2", "--requests", "3", *flags])
    _example().main()
    assert "step 1:" in capsys.readouterr().out


def test_two_streams_at_once():
    """Calls of every kind on two streams, each with the workspace of its own stream."""
    g = torch.Generator().manual_seed(3)
    cache = paged.Cache4(300, 16, 2, 128, dtype=torch.bfloat16, device=DEV)
    draw = lambda *shape: torch.randn(*shape, generator=g).bfloat16().to(DEV)
    n = 300 * 16
    k, v = draw(n, 2, 128), draw(n, 2, 128)
    paged.store_kv4(k, v, torch.arange(n, device=DEV), cache)
    kc, vc = (x.view(300, 16, 2, 128) for x in paged.load_kv4(torch.arange(n, device=DEV), cache))
    table = torch.randperm(300, generator=g).int().view(2, 150).to(DEV)
    q, logits, tokens = draw(4, 16, 128), torch.randn(200, 40001, generator=g).to(DEV), torch.randint(0, 40001, (200,), generator=g).to(DEV)
    seq, cu = i32([2400, 1999]), i32([0, 1, 4])
    calls = (lambda: paged.tree_attention4(q, cache, table, seq, cu, 3), lambda: paged.tree_attention4(q, cache, table, seq, cu, 1, window=700, sinks=9),
             lambda: paged.tree_attention(q, kc, vc, table, seq, cu, 3, window=700, sinks=9),
             lambda: logprobs.token_logprobs(logits, tokens, top=7).top_logprobs)
    want = [f() for f in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] += [f() for f in calls]
    torch.cuda.synchronize()
    for out in got:
        for j, x in enumerate(out):
            assert torch.equal(x, want[j % len(calls)])
    assert paged.read_status() == 0
