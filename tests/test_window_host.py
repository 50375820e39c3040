"""Windowed attention: what the library refuses, and the list of key tiles that it visits, restated."""
import ctypes as C
import random

import pytest

from dsv41_flash_offload_b200 import _lib, paged
from test_step_host import FAKE, _err


def test_window_refusals():
    a = dict(dtype=0, batch=1, num_tokens=2, max_new=2, q_heads=4, kv_heads=2, head_dim=64, page_size=16, num_pages=4, max_keys=64,
             q=FAKE, q_stride_token=256, q_stride_head=64, k_cache=FAKE, v_cache=FAKE, stride_page=2048, stride_slot=128,
             stride_head=64, block_table=FAKE, table_stride=4, seq_lens=FAKE, cu_lens=FAKE, tree_mask=None, mask_words=1, scale=0.1,
             out=FAKE, out_stride_token=256, out_stride_head=64, lse=None)

    def call(window, sinks, **kw):
        return _lib.load().dsv41_tree_attention_window(C.byref(_lib.TreeAttentionArgs(**{**a, **kw})), window, sinks, FAKE, 1 << 40, None)

    _err(call(-1, 0), b"window")
    _err(call(8, -1), b"window")
    _err(call(0, 4), b"without a window")
    _err(call(8, 0, q=None), b"NULL")
    assert call(8, 4, num_tokens=0) == 0
    for window, sinks in ((0, 0), (-3, 0), (1 << 31, 0), (5, -1), (None, 2)):
        with pytest.raises(ValueError):
            paged._window(window, sinks)
    assert paged._window(None, 0) == (0, 0) and paged._window(7, 3) == (7, 3)


def key_tiles(seq, n, group, window, sinks, tree, RT, KT):
    """Tiles of each row tile, as KeyTiles lists them."""
    ctx, lists = seq - n, []
    for rt in range(-(-n * group // RT)):
        before, last = 0, seq - 1
        if not tree:
            before, last = rt * RT // group + 1, ctx + (min(rt * RT + RT, n * group) - 1) // group
        end, first = last // KT + 1, max(ctx + before - window, 0) // KT
        ns = min(-(-min(sinks, seq) // KT), end)
        skip = max(first - ns, 0)
        lists.append([x if x < ns else x + skip for x in range(end - skip)])
    return lists, max(-(-seq // KT), 1)


def test_every_visible_key_is_in_the_list_once():
    rng = random.Random(1)
    for _ in range(4000):
        n, ctx = rng.randint(1, 40), rng.choice((0, 1, rng.randint(0, 60), rng.randint(0, 600)))
        group, KT, RT = rng.choice((1, 2, 3, 5, 8, 16)), rng.choice((4, 8, 16)), rng.choice((8, 16, 32))
        window, sinks = rng.choice((1, 2, rng.randint(1, 40), rng.randint(1, 700))), rng.choice((0, 1, 4, rng.randint(0, 90)))
        tree = rng.random() < 0.5
        seq = ctx + n
        lists, total = key_tiles(seq, n, group, window, sinks, tree, RT, KT)
        for rt, tiles in enumerate(lists):
            assert len(set(tiles)) == len(tiles) and 0 <= min(tiles) and max(tiles) < total
            seen = set()
            for row in range(rt * RT, min(rt * RT + RT, n * group)):
                i = row // group
                if tree:    # any set of new tokens
                    see = list(range(ctx)) + [ctx + j for j in range(n) if rng.random() < 0.7]
                else:
                    see = list(range(ctx + i + 1))
                seen |= set(see[-window:]) | {x for x in see if x < sinks}
            assert {x // KT for x in seen} <= set(tiles), (n, ctx, group, window, sinks, tree, rt)
