"""The cache in 4 bits: what the C side and the Python side refuse, sizes, and the layout and the rounding restated."""
import ctypes as C

import pytest
import torch

from dsv41_flash_offload_b200 import Dsv41Error, _lib, paged
from test_step_host import FAKE, _err


def _cache(**kw):
    return _lib.Kv4Cache(**{**dict(num_pages=4, page_size=16, kv_heads=2, head_dim=64, data=FAKE), **kw})


def _tokens(**kw):
    a = dict(dtype=0, num_tokens=2, k=FAKE, v=FAKE, k_stride_token=128, k_stride_head=64, v_stride_token=128, v_stride_head=64, slots=FAKE)
    return C.byref(_lib.Kv4Tokens(**{**a, **kw}))


def test_sizes():
    n = C.c_size_t()
    size = _lib.load().dsv41_kv4_cache_size
    for pages, page, heads, dim in ((1, 8, 1, 32), (7, 24, 3, 96), (5, 128, 8, 256), (0, 16, 2, 64), (1 << 20, 64, 8, 128)):
        assert size(pages, page, heads, dim, C.byref(n)) == 0
        assert n.value == pages * page * heads * 2 * dim * 5 // 8
    _err(size(1, 8, 1, 32, None), b"NULL")


def test_cache_refusals():
    L = _lib.load()
    for kw, text in ((dict(page_size=12), b"page_size"), (dict(page_size=0), b"page_size"), (dict(page_size=4), b"page_size"),
                     (dict(head_dim=40), b"head_dim"), (dict(head_dim=288), b"head_dim"), (dict(head_dim=0), b"head_dim"),
                     (dict(kv_heads=0), b"kv_heads"), (dict(num_pages=-1), b"num_pages"), (dict(data=None), b"data"),
                     (dict(data=FAKE + 8), b"data"), (dict(page_size=1 << 24), b"pages of")):
        c = C.byref(_cache(**kw))
        _err(L.dsv41_kv4_store(c, _tokens(), None), text)
        _err(L.dsv41_kv4_load(c, _tokens(), None), text)
        _err(L.dsv41_kv4_move(c, FAKE, FAKE, 1, FAKE, 1 << 20, None), text)
    _err(L.dsv41_kv4_store(None, _tokens(), None), b"NULL")


def test_token_refusals():
    L, c = _lib.load(), C.byref(_cache())
    for fn in (L.dsv41_kv4_store, L.dsv41_kv4_load):
        for kw, text in ((dict(dtype=2), b"dtype"), (dict(num_tokens=-1), b"num_tokens"), (dict(k=None), b"NULL"), (dict(slots=None), b"NULL"),
                         (dict(v=FAKE + 8), b"16-byte"), (dict(k_stride_token=132), b"stride"), (dict(v_stride_head=-8), b"stride")):
            _err(fn(c, _tokens(**kw), None), text)
        assert fn(c, _tokens(num_tokens=0), None) == 0
        _err(fn(c, None, None), b"NULL")
    _err(L.dsv41_kv4_load(c, _tokens(k_stride_token=0), None), b"repeats")
    _err(L.dsv41_kv4_move(c, FAKE, FAKE, -1, FAKE, 100, None), b"num_tokens")
    _err(L.dsv41_kv4_move(c, FAKE, None, 1, FAKE, 1 << 20, None), b"NULL")
    _err(L.dsv41_kv4_move(c, FAKE, FAKE, 1, FAKE + 8, 1 << 20, None), b"16-byte")
    assert L.dsv41_kv4_move(c, FAKE, FAKE, 1, FAKE, 2 * 2 * 2 * 20 - 1, None) == _lib.E_WORKSPACE
    assert L.dsv41_kv4_move(c, FAKE, FAKE, 0, FAKE, 0, None) == 0


def test_attention_refusals():
    a = dict(dtype=0, batch=1, num_tokens=2, max_new=2, q_heads=4, kv_heads=2, head_dim=64, page_size=16, num_pages=4, max_keys=64,
             q=FAKE, q_stride_token=256, q_stride_head=64, k_cache=None, v_cache=None, stride_page=0, stride_slot=0,
             stride_head=0, block_table=FAKE, table_stride=4, seq_lens=FAKE, cu_lens=FAKE, tree_mask=None, mask_words=1, scale=0.1,
             out=FAKE, out_stride_token=256, out_stride_head=64, lse=None)

    def call(window=0, sinks=0, ws=FAKE, nbytes=1 << 40, cache=None, **kw):
        args = C.byref(_lib.TreeAttentionArgs(**{**a, **kw}))
        return _lib.load().dsv41_tree_attention4(args, C.byref(cache or _cache()), window, sinks, ws, nbytes, None)

    for kw, text in ((dict(dtype=2), b"dtype"), (dict(q_heads=5), b"q_heads"), (dict(head_dim=32), b"cache's"), (dict(page_size=8), b"cache's"),
                     (dict(num_pages=3), b"cache's"), (dict(kv_heads=1), b"cache's"), (dict(q=None), b"NULL"), (dict(out=FAKE + 8), b"16-byte"),
                     (dict(window=-1), b"window"), (dict(sinks=2), b"without a window"), (dict(cache=_cache(data=None)), b"data"),
                     (dict(out_stride_token=0), b"repeats"), (dict(ws=None), b"NULL"), (dict(scale=float("nan")), b"scale")):
        _err(call(**kw), text)
    assert call(nbytes=1000) == _lib.E_WORKSPACE
    assert call(num_tokens=0) == 0


def test_python_refuses_without_a_gpu():
    for bad in (lambda: paged.Cache4(2, 12, 1, 64, data=torch.zeros(1)), lambda: paged.Cache4(2, 16, 1, 40, data=torch.zeros(1))):
        with pytest.raises(Dsv41Error):
            bad()
    with pytest.raises(ValueError):
        paged.Cache4(2, 16, 1, 64, data=torch.zeros(2 * 16 * 64 * 2 * 5 // 8, dtype=torch.uint8))
    with pytest.raises(TypeError):
        paged.Cache4(2, 16, 1, 64, dtype=torch.float32)
