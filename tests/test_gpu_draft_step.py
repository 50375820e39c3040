"""The operators together (examples/draft_step.py): a drafted step gives every token what it would get if its own path
had been decoded as a plain sequence, and accepted tokens carry over to the next step."""
import importlib.util
import os

import pytest
import torch

from conftest import ROOT
from dsv41_flash_offload_b200 import paged

pytestmark = pytest.mark.gpu


def _example():
    spec = importlib.util.spec_from_file_location("draft_step", os.path.join(ROOT, "examples", "draft_step.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def test_each_path_of_a_tree_is_a_sequence():
    """Same kernels, other batches and masks: the tokens' sums run in another order, so fp32 sums differ in their last
    bits, a fp16 rounding of theirs may fall the other way, and a router may not be asked to decide a near tie
    (the seeds leave every choice clear). Bound: a few units of fp16 at the outputs' size."""
    ex = _example()
    rng = torch.Generator().manual_seed(3)
    layer = ex.DraftLayer(seed=2)
    prompt, parents, hidden = [19, 40], [-1, 0, 0, 1, 3, -1, 0, 1], 512
    new = [5, 3]
    x0 = torch.randn(sum(prompt), hidden, generator=rng).half().cuda()
    x1 = torch.randn(sum(new), hidden, generator=rng).half().cuda()

    def prefill():
        cache = ex.PagedCache(2, 24, 16, 8, layer.kv_heads, layer.head_dim)
        t = cache.begin(i32([0, 0]), i32(prompt), sum(prompt))
        layer.forward(x0, cache, t, max(prompt))
        return cache

    cache = prefill()
    t = cache.begin(i32(prompt), i32(new), sum(new), i32(parents))
    tree = layer.forward(x1, cache, t, max(new))
    for b, token in ((0, 4), (0, 2), (1, 2)):
        base = sum(new[:b])
        path, i = [], token
        while i >= 0:
            path.insert(0, base + i)
            i = parents[base + i]
        lens = [len(path) if r == b else 0 for r in range(2)]
        seq = prefill()
        s = seq.begin(i32(prompt), i32(lens), len(path))
        plain = layer.forward(x1[path].contiguous(), seq, s, len(path))
        err = (plain.float() - tree[path].float()).abs().max()
        assert float(err) <= 8 * torch.finfo(torch.float16).eps * float(tree.float().abs().max()), (b, token, float(err))
    # accept the first request's deepest path: the next step reads it as context
    path = [0, 1, 3, 4]
    cache.keep(t, [path, [5]], i32(prompt))
    nxt = torch.randn(2, hidden, generator=rng).half().cuda()
    t2 = cache.begin(i32([19 + 4, 40 + 1]), i32([1, 1]), 2)
    got = layer.forward(nxt, cache, t2, 1)
    seq = prefill()
    s = seq.begin(i32(prompt), i32([4, 1]), 5)
    layer.forward(x1[[0, 1, 3, 4, 5]].contiguous(), seq, s, 4)
    s = seq.begin(i32([23, 41]), i32([1, 1]), 2)
    want = layer.forward(nxt, seq, s, 1)
    assert float((got.float() - want.float()).abs().max()) <= 8 * torch.finfo(torch.float16).eps * float(want.float().abs().max())
    assert paged.read_status() == 0 and not bool(t2.status.any())


def test_the_example_runs(capsys, monkeypatch):
    monkeypatch.setattr("sys.argv", ["draft_step.py", "--steps", "2", "--requests", "3"])
    _example().main()
    assert "step 1:" in capsys.readouterr().out
