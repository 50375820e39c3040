"""CPU-only tests of the decode-step operators: C ABI refusals (before any device work), sizes, and a
restatement of the unsigned division by a constant the attention kernel uses for page lookups."""
import ctypes as C
import random

import pytest
import torch

from dsv41_flash_offload_b200 import _lib, paged, w4

FAKE = 1 << 20   # never dereferenced: the checks run before any device work


def _err(rc, text):
    assert rc == _lib.E_INVALID and text in _lib.load().dsv41_last_error(), (rc, _lib.load().dsv41_last_error())


def test_w4_layout_sizes_and_refusals():
    L = _lib.load()
    n = C.c_size_t()
    # 2 row tiles x 2 chunks of 512 bytes, then 2 x 4 groups x 32 bytes, then 2 x 4 x 16 bytes of zero points
    assert L.dsv41_w4_layout_size(17, 96, 32, 0, C.byref(n)) == 0 and n.value == 2 * 2 * 512 + 256
    assert L.dsv41_w4_layout_size(17, 96, 32, 1, C.byref(n)) == 0 and n.value == 2 * 2 * 512 + 256 + 256
    for bad in ((0, 64, 64), (16, 96, 64), (16, 64, 48), (16, 0, 32)):
        _err(L.dsv41_w4_layout_size(*bad, 0, C.byref(n)), b"multiple")
    _err(L.dsv41_w4_pack(None, None, None, 16, 64, 64, None, 1 << 20, None), b"NULL")
    assert L.dsv41_w4_pack(FAKE, FAKE, None, 16, 64, 64, FAKE, 100, None) == _lib.E_WORKSPACE


def test_w4_product_refusals():
    L = _lib.load()
    w = _lib.W4WeightC(64, 128, 64, 0, 0, FAKE)

    def lin(w=w, x=FAKE, xd=0, xs=128, t=2, out=FAKE, od=2, os=64, acc=0):
        return L.dsv41_w4_linear(None if w is None else C.byref(w), x, xd, xs, t, out, od, os, acc, None)

    _err(lin(w=None), b"weight is NULL")
    _err(lin(w=_lib.W4WeightC(64, 100, 64, 0, 0, FAKE)), b"multiple of its group")
    _err(lin(w=_lib.W4WeightC(64, 128, 16, 0, 0, FAKE)), b"group 16")
    _err(lin(w=_lib.W4WeightC(64, 128, 64, 0, 2, FAKE)), b"scales")
    _err(lin(w=_lib.W4WeightC(64, 128, 64, 0, 0, FAKE + 16)), b"256-byte")
    _err(lin(xd=2), b"x dtype")
    _err(lin(od=3), b"out dtype")
    _err(lin(od=0, acc=1), b"fp32 out")
    _err(lin(x=None), b"NULL")
    _err(lin(x=FAKE + 8), b"16-byte")
    _err(lin(xs=127), b"x_stride")
    _err(lin(xs=132), b"x_stride")
    _err(lin(os=63), b"out_stride")
    _err(lin(t=-1), b"tokens")
    assert lin(t=0) == 0
    up = _lib.W4WeightC(64, 128, 32, 0, 0, FAKE)
    _err(L.dsv41_w4_gated(C.byref(w), C.byref(up), FAKE, 0, 128, 1, 10.0, FAKE, 0, 64, None), b"gate and up differ")
    _err(L.dsv41_w4_gated(C.byref(w), None, FAKE, 0, 128, 1, 10.0, FAKE, 0, 64, None), b"up weight is NULL")
    _err(L.dsv41_w4_gated(C.byref(w), C.byref(w), FAKE, 0, 128, 1, float("nan"), FAKE, 0, 64, None), b"limit")


def _tables(**kw):
    a = dict(batch=2, width=4, page_size=16, num_tokens=8, context_lens=FAKE, new_lens=FAKE, held_pages=FAKE, block_table=FAKE,
             table_stride=4, free_pages=FAKE, free_count=FAKE, free_capacity=8, mask_words=1, parents=None, cu_lens=FAKE,
             seq_lens=FAKE, slots=FAKE, positions=FAKE, requests=FAKE, held_out=FAKE + 64, free_count_out=FAKE + 64, status=FAKE,
             tree_mask=None)
    a.update(kw)
    return _lib.load().dsv41_step_tables(C.byref(_lib.StepTablesArgs(**a)), None)


def test_step_tables_refusals():
    for kw, text in ((dict(batch=0), b"batch"), (dict(batch=2049), b"batch"), (dict(table_stride=3), b"block table"),
                     (dict(batch=2048, width=1 << 20, table_stride=1 << 20), b"block table"), (dict(page_size=0), b"page_size"),
                     (dict(num_tokens=-1), b"num_tokens"), (dict(free_capacity=-1), b"free_capacity"), (dict(cu_lens=None), b"NULL"),
                     (dict(free_pages=None), b"NULL"), (dict(slots=None), b"NULL"), (dict(held_out=FAKE), b"overlaps"),
                     (dict(free_count_out=FAKE), b"overlaps"), (dict(slots=FAKE + 4), b"misaligned"),
                     (dict(parents=FAKE, tree_mask=FAKE, mask_words=0), b"mask_words"), (dict(parents=FAKE), b"tree_mask")):
        _err(_tables(**kw), text)
    _err(_lib.load().dsv41_step_tables(None, None), b"NULL")


def _store(**kw):
    a = dict(num_tokens=4, kv_heads=2, head_dim=64, num_pages=4, page_size=16, k=FAKE, v=FAKE, k_stride_token=128, k_stride_head=64,
             v_stride_token=128, v_stride_head=64, slots=FAKE, k_cache=FAKE, v_cache=FAKE, stride_page=2048, stride_slot=128,
             stride_head=64)
    a.update(kw)
    return _lib.load().dsv41_store_kv(C.byref(_lib.StoreKvArgs(**a)), None)


def test_store_refusals():
    for kw, text in ((dict(head_dim=60), b"head_dim"), (dict(kv_heads=0), b"kv_heads"), (dict(num_tokens=-1), b"num_tokens"),
                     (dict(page_size=0), b"page_size"), (dict(k=None), b"NULL"), (dict(v=FAKE + 8), b"16-byte"),
                     (dict(stride_slot=130), b"stride"), (dict(k_stride_head=4), b"stride")):
        _err(_store(**kw), text)
    assert _store(num_tokens=0) == 0


def _attn(ws=FAKE, nbytes=1 << 40, **kw):
    a = dict(dtype=0, batch=1, num_tokens=2, max_new=2, q_heads=4, kv_heads=2, head_dim=64, page_size=16, num_pages=4, max_keys=64,
             q=FAKE, q_stride_token=256, q_stride_head=64, k_cache=FAKE, v_cache=FAKE, stride_page=2048, stride_slot=128,
             stride_head=64, block_table=FAKE, table_stride=4, seq_lens=FAKE, cu_lens=FAKE, tree_mask=None, mask_words=1, scale=0.1,
             out=FAKE, out_stride_token=256, out_stride_head=64, lse=None)
    a.update(kw)
    return _lib.load().dsv41_tree_attention(C.byref(_lib.TreeAttentionArgs(**a)), ws, nbytes, None)


def test_attention_refusals():
    for kw, text in ((dict(dtype=2), b"dtype"), (dict(batch=0), b"batch"), (dict(batch=2049), b"batch"), (dict(q_heads=5), b"q_heads"),
                     (dict(head_dim=264), b"head_dim"), (dict(head_dim=60), b"head_dim"), (dict(page_size=0), b"page_size"),
                     (dict(max_new=-1), b"max_new"), (dict(q=None), b"NULL"), (dict(ws=None), b"NULL"), (dict(q=FAKE + 8), b"16-byte"),
                     (dict(k_cache=FAKE + 8), b"16-byte"), (dict(ws=FAKE + 64), b"256-byte"), (dict(q_stride_head=68), b"stride"),
                     (dict(stride_slot=132), b"stride"), (dict(scale=float("inf")), b"scale"), (dict(max_keys=-1), b"max_keys"),
                     (dict(tree_mask=FAKE, mask_words=5), b"mask_words"), (dict(num_tokens=1 << 30), b"2^31")):
        _err(_attn(**kw), text)
    assert _attn(nbytes=1000) == _lib.E_WORKSPACE
    assert _attn(num_tokens=0) == 0
    n = C.c_size_t()
    sizes = []
    for d in (8, 64, 128, 256):
        assert _lib.load().dsv41_tree_attention_workspace_size(d, C.byref(n)) == 0
        sizes.append(n.value)
    assert sizes[0] == sizes[1] < sizes[2] and all(s > 0 and s % 256 == 0 for s in sizes)


def test_python_refuses_cpu_tensors():
    with pytest.raises(ValueError):
        w4.W4Weight(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.float16))
    z = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        paged.step_tables(z, z, z, torch.zeros(2, 2, dtype=torch.int32), z, z[:1], 16, 2)
    c = torch.zeros(1, 16, 1, 64, dtype=torch.float16)
    with pytest.raises(ValueError):
        paged.tree_attention(torch.zeros(1, 1, 64, dtype=torch.float16), c, c, torch.zeros(1, 1, dtype=torch.int32), z[:1], z, 1)


def test_page_division_restatement():
    """m = ceil(2^(31 + l) / d), l = ceil(log2 d): (n * m >> 32) >> (l - 1) is n // d for every n < 2^31."""
    rng = random.Random(0)
    for d in list(range(2, 400)) + [1000, 4097, 65537, (1 << 30) - 1, (1 << 31) - 1]:
        l = (d - 1).bit_length()
        m = -(-(1 << (31 + l)) // d)
        assert m < 1 << 32
        for n in [0, 1, d - 1, d, min(d + 1, 2 ** 31 - 1), 2 ** 31 - 1] + [rng.randrange(1 << 31) for _ in range(50)]:
            assert ((n * m) >> 32) >> (l - 1) == n // d
