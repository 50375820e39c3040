"""The cut of a call's key tiles into runs: many requests of very unequal lengths, with and without lists of tiles of their own, so that
a thread sums several requests, warps sum one request's row tiles together, and runs end inside requests, heads and row tiles."""
import numpy as np
import pytest
import torch

import test_gpu_kv4 as kv4
import test_gpu_paged as base
import test_gpu_window as win
from test_gpu_paged import build

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def lengths(count, seed, long_new):
    """One token each, some without any, a few prompts of many row tiles among them."""
    rng = np.random.default_rng(seed)
    new = rng.integers(0, 3, count)
    new[rng.integers(0, count, 5)] = rng.integers(long_new // 2, long_new, 5)
    ctx = np.exp(rng.uniform(0, np.log(400), count)).astype(int) - 1
    ctx[rng.integers(0, count, 3)] = 2500
    return ctx.tolist(), new.tolist()


@pytest.mark.parametrize("count", [37, 500, 1300])
@pytest.mark.parametrize("tree", [False, True])
def test_without_a_window(count, tree):
    ctx, new = lengths(count, count, 250 if not tree else 60)
    base.check(build(ctx, new, 4, 2, 64, 16, F16, seed=count, tree=tree))


@pytest.mark.parametrize("count", [37, 500, 1300])
@pytest.mark.parametrize("window,sinks", [(150, 3), (2000, 0)])
def test_prompts_among_single_tokens_through_a_window(count, window, sinks):
    ctx, new = lengths(count, count + 1, 250)
    win.check(build(ctx, new, 4, 2, 64, 16, BF16, seed=count, tree=False), window, sinks)


@pytest.mark.parametrize("count", [37, 700, 2048])
@pytest.mark.parametrize("heads,kv,new", [(2, 2, 60), (8, 1, 60)])
@pytest.mark.parametrize("window", [None, 100])
@pytest.mark.parametrize("tree", [False, True])
def test_over_4_bits(count, heads, kv, new, window, tree, monkeypatch):
    ctx, lens = lengths(count, count + 2, new)
    s = kv4.in4(build(ctx, lens, heads, kv, 32, 8, F16, seed=count, tree=tree))
    kv4.check4(s, monkeypatch, window, 2 if window else 0)


def test_bounds_on_new_tokens_only_pick_the_kernel():
    """max_new of 1 for requests that bring more: slower, the same."""
    from dsv41_flash_offload_b200 import paged
    ctx, new = lengths(200, 9, 100)
    for tree in (False, True):
        new = [min(n, 60) for n in new]
        s = kv4.in4(build(ctx, new, 4, 2, 64, 16, F16, seed=5, tree=tree))
        ref, bound, _ = base.reference(s)
        for few in (1, 5, 60):
            out = paged.tree_attention4(s["q"], s["cache"], s["table"], s["seq"], s["cu"], few, tree_mask=s["mask"])
            assert bool(((out.cpu().double() - ref).abs() <= bound).all()) and paged.read_status() == 0
