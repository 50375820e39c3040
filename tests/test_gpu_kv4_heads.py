"""Attention of more than 16 rows over a cache in 4 bits (decoding warps in front of the tensor cores) at every head size that is not a whole
tile of columns: groups of decoding threads then get unequal numbers of chunks, some of them none. Against the definitions and to the
bounds of test_gpu_paged.py and test_gpu_window.py, over what the codes stand for."""
import pytest
import torch

import test_gpu_kv4 as kv4
from dsv41_flash_offload_b200 import paged
from test_gpu_paged import DEV, build

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
ROWS = [(8, 1, [4, 3]), (8, 1, [5, 8]), (16, 2, [9, 16]), (8, 1, [20, 37])]   # up to 32, 64, 128 rows a KV head, and more


@pytest.mark.parametrize("dim", [32, 96, 160, 192, 224])
@pytest.mark.parametrize("heads,kv,new", ROWS)
@pytest.mark.parametrize("window,sinks", [(None, 0), (60, 3)])
@pytest.mark.parametrize("tree", [False, True])
def test_heads_and_rows(heads, kv, new, dim, window, sinks, tree, monkeypatch):
    dtype = F16 if (dim // 32 + len(new) + new[0]) % 2 else BF16
    kv4.check4(kv4.in4(build([150, 300], new, heads, kv, dim, 24, dtype, seed=dim + new[1], tree=tree)), monkeypatch, window, sinks)


@pytest.mark.parametrize("dim", [32, 160, 224])
@pytest.mark.parametrize("heads,kv,new", ROWS)
def test_split_requests(heads, kv, new, dim, monkeypatch):
    kv4.check4(kv4.in4(build([5000, 1300], new, heads, kv, dim, 16, BF16, seed=dim)), monkeypatch)


@pytest.mark.parametrize("dim", [32, 96, 160, 192, 224])
@pytest.mark.parametrize("heads,kv,new", [(5, 1, [6, 4]), (8, 1, [6, 4]), (8, 1, [9, 7]), (16, 1, [9, 12])])
@pytest.mark.parametrize("window", [None, 60])
def test_nan_reaches_those_who_see_it(heads, kv, new, dim, window):
    kv4.test_nan_reaches_those_who_see_it(heads, kv, dim, new, window, F16 if dim % 64 else BF16)


@pytest.mark.parametrize("dim", [32, 160])
@pytest.mark.parametrize("heads,kv", [(8, 1), (3, 1)])
def test_tokens_behind_the_last_request_stay(heads, kv, dim):
    """A padded batch: rows that belong to no request keep what they held, in both kernels."""
    for new in ([1, 2], [9, 5], [30, 40]):
        s = kv4.in4(build([100, 33], new, heads, kv, dim, 16, F16, seed=dim))
        n, pad = sum(new), 5
        want = kv4.attend4(s)
        wide = lambda t: torch.cat((t, torch.zeros(pad, *t.shape[1:], dtype=t.dtype, device=DEV)))
        out = torch.full((n + pad, heads, dim), 7.0, dtype=F16, device=DEV)
        kv4.attend4(dict(s, q=wide(s["q"]), mask=wide(s["mask"])), out=out)
        assert torch.equal(out[:n], want) and bool((out[n:] == 7.0).all()) and paged.read_status() == 0
