"""The paged operators where inputs are at their ends, against plain restatements in 64 bits, with the bounds of
test_gpu_paged.py."""
import math

import pytest
import torch

from dsv41_flash_offload_b200 import Dsv41Error, paged
from test_gpu_paged import DEV, attend, build, reference

pytestmark = pytest.mark.gpu


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
