"""A paged key/value cache for decode steps with drafted tokens: the step's page tables and slot maps, the
store of new keys and values, and the attention of drafted trees over the cache.

A cache is a pair of tensors [num_pages, page_size, kv_heads, head_dim]; slot s is token s % page_size of page
s // page_size, and row b of a block table lists the pages of request b. One step of a layer stack is

    t = step_tables(context_lens, new_lens, held_pages, block_table, free_pages, free_count, page_size, N, parents=...)
    per layer:  store_kv(k, v, t.slots, k_cache, v_cache)
                out = tree_attention(q, k_cache, v_cache, block_table, t.seq_lens, t.cu_lens, max_new, tree_mask=t.tree_mask)

All lengths stay on the GPU, nothing synchronises the host, and after the first tree_attention on a stream
(whose workspace is kept per device, stream and head size) only outputs are allocated, so a step can be
captured in a CUDA graph. A graph uses the workspace that its capture took: the capture stream's own (made there by an
eager call or by reserve_workspace), or one given as `workspace=`. Replays that share a workspace, and eager calls on
that stream, have to follow one another; graphs that run at the same time need one each (attention_workspace).
"""
from __future__ import annotations

import ctypes as C
import threading
from typing import NamedTuple

import torch

from . import _lib

_DTYPES = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}
MAX_REQUESTS = 2048
MAX_MASK_WORDS = 4
NO_PAGES, TOO_WIDE, BAD_PARENT, BIG_TREE, NO_ROOM, PAST_TOKENS = 1, 2, 4, 8, 16, 32   # status bits of a request


class StepTables(NamedTuple):
    """What one step of the layer stack reads (all on the GPU)."""
    cu_lens: torch.Tensor            # int32 [B + 1] running sums of the new tokens
    seq_lens: torch.Tensor           # int32 [B] context + new tokens (0: the request was refused)
    slots: torch.Tensor              # int64 [N] cache slot of each new token (-1: none)
    positions: torch.Tensor          # int32 [N] position of each new token (context + depth in its tree)
    requests: torch.Tensor           # int32 [N] request of each new token (-1: padding)
    held_pages: torch.Tensor         # int32 [B] pages held after the step's exchange
    free_count: torch.Tensor         # int32 [1] height of the stack of free pages after it
    status: torch.Tensor             # int32 [B] 0, or why a request was refused / its tree is broken
    tree_mask: torch.Tensor | None   # int64 [N, mask_words] ancestors of each drafted token


def _vector(t: torch.Tensor, name: str, n: int, dtype: torch.dtype, dev: torch.device) -> torch.Tensor:
    if t.dtype is not dtype or t.shape != (n,) or t.device != dev:
        raise ValueError(f"{name} must be {str(dtype)[6:]} [{n}] on {dev}")
    return t if t.is_contiguous() else t.contiguous()


def _table(t: torch.Tensor, batch: int, dev: torch.device) -> tuple[int, int, int]:
    """Address, width and row stride of a block table."""
    if t.dtype is torch.int32 and t.dim() == 2 and t.device == dev:
        rows, width = t.shape
        if rows == batch:
            if t.is_contiguous():
                return t.data_ptr(), width, width
            if t.stride(1) == 1 and t.stride(0) >= width:
                return t.data_ptr(), width, t.stride(0)
    raise ValueError(f"block_table must be int32 [{batch}, width] with contiguous rows on {dev}")


def step_tables(context_lens: torch.Tensor, new_lens: torch.Tensor, held_pages: torch.Tensor, block_table: torch.Tensor,
                free_pages: torch.Tensor, free_count: torch.Tensor, page_size: int, num_tokens: int, *,
                parents: torch.Tensor | None = None, mask_words: int = 1) -> StepTables:
    """Bring every request's pages in line with its length and build the step's maps, in one launch.

    Request b holds held_pages[b] pages (row b of block_table) for context_lens[b] tokens and brings new_lens[b]
    (all int32 [B]); surplus pages go back on the stack free_pages[:free_count], missing ones come off it, in
    request order. block_table [B, W] and free_pages are updated in place; held_pages and free_count come back
    as new tensors for the next step. A finished request has lengths 0: its pages go back. Rejected drafts:
    pass the accepted context length and the surplus goes back. num_tokens is the length of the step's token
    batch, >= sum(new_lens); requests whose tokens pass it get seq_lens 0 and slots -1 (status PAST_TOKENS). parents
    (int32 [num_tokens]): index within its request of each drafted token's parent, which must lie before it, -1 for
    the context; then positions are context + depth and tree_mask is built, for trees of up to 64 * mask_words tokens. A request that finds no pages is refused: status bit,
    seq_lens 0, slots -1. free_pages should have room for every page of the pool: a request whose surplus does not fit, and
    those behind it, keep theirs (status NO_ROOM) and are served all the same."""
    dev = context_lens.device
    if not context_lens.is_cuda or context_lens.dim() != 1 or not 1 <= context_lens.shape[0] <= MAX_REQUESTS:
        raise ValueError(f"context_lens must be a CUDA int32 [B] with B in 1..{MAX_REQUESTS}")
    B, N = context_lens.shape[0], int(num_tokens)
    context_lens = _vector(context_lens, "context_lens", B, torch.int32, dev)
    new_lens = _vector(new_lens, "new_lens", B, torch.int32, dev)
    held_pages = _vector(held_pages, "held_pages", B, torch.int32, dev)
    free_count = _vector(free_count, "free_count", 1, torch.int32, dev)
    table, width, table_stride = _table(block_table, B, dev)
    if free_pages.dtype != torch.int32 or free_pages.dim() != 1 or not free_pages.is_contiguous() or free_pages.device != dev:
        raise ValueError(f"free_pages must be a contiguous int32 vector on {dev}")
    if N < 0:
        raise ValueError("num_tokens is negative")
    mask = None
    if parents is not None:
        if not 1 <= mask_words <= MAX_MASK_WORDS:
            raise ValueError(f"mask_words must be 1..{MAX_MASK_WORDS}")
        parents = _vector(parents, "parents", N, torch.int32, dev)
        mask = parents.new_empty((N, mask_words), dtype=torch.int64)
    ints = context_lens.new_empty(2 * N + 4 * B + 2)
    positions, requests, cu, seq, held, count, status = ints.split_with_sizes((N, N, B + 1, B, B, 1, B))
    slots = context_lens.new_empty(N, dtype=torch.int64)
    base = ints.data_ptr()
    at = base + 8 * N
    args = _lib.StepTablesArgs(
        B, width, int(page_size), N, context_lens.data_ptr(), new_lens.data_ptr(), held_pages.data_ptr(), table,
        table_stride, free_pages.data_ptr(), free_count.data_ptr(), free_pages.shape[0], int(mask_words), parents.data_ptr() if parents is not None else None,
        at, at + 4 * B + 4, slots.data_ptr(), base, base + 4 * N, at + 8 * B + 4, at + 12 * B + 4, at + 12 * B + 8,
        mask.data_ptr() if mask is not None else None)
    _lib.call(dev, _lib.load().dsv41_step_tables, C.byref(args), _lib.current_stream(dev))
    return StepTables(cu, seq, slots, positions, requests, held, count, status, mask)


def _cache(k_cache: torch.Tensor, v_cache: torch.Tensor) -> tuple[torch.Size, tuple, torch.device]:
    """Shape, strides and device of a pair of caches, checked."""
    shape, strides, dev = k_cache.shape, k_cache.stride(), k_cache.device
    if len(shape) != 4 or shape != v_cache.shape or strides != v_cache.stride() or k_cache.dtype is not v_cache.dtype:
        raise ValueError("the caches must be [num_pages, page_size, kv_heads, head_dim], alike in shape, dtype and strides")
    if not k_cache.is_cuda or v_cache.device != dev:
        raise ValueError("the caches must live on one CUDA device")
    if k_cache.dtype not in _DTYPES:
        raise TypeError(f"unsupported cache dtype {k_cache.dtype} (fp16 or bf16)")
    if shape[3] % 8 or shape[3] == 0:
        raise ValueError("head_dim must be a multiple of 8")
    if (strides[3] != 1 or strides[0] % 8 or strides[1] % 8 or strides[2] % 8 or k_cache.data_ptr() % 16
            or v_cache.data_ptr() % 16):
        raise ValueError("the caches must have contiguous, 16-byte aligned heads")
    return shape, strides, dev


def _heads(t: torch.Tensor, name: str, shape: tuple, like: torch.Tensor) -> torch.Tensor:
    """t of this shape with contiguous, 16-byte aligned heads (copied if they are not)."""
    if t.shape != shape or t.device != like.device:
        raise ValueError(f"{name} must be {list(shape)} on {like.device}")
    if t.dtype is not like.dtype:
        raise TypeError(f"{name} is {t.dtype}, the cache {like.dtype}")
    s = t.stride()
    if s[2] != 1 or s[0] % 8 or s[1] % 8 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def store_kv(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor) -> None:
    """k_cache[slots[t]] = k[t] and v_cache[slots[t]] = v[t] for new keys and values [N, kv_heads, head_dim] (any
    strides with contiguous heads, e.g. slices of a fused projection); slots int64 [N], -1 stores nothing."""
    (pages, page_size, heads, dim), cs, dev = _cache(k_cache, v_cache)
    N = slots.shape[0] if slots.dim() else 0
    slots = _vector(slots, "slots", N, torch.int64, dev)
    k = _heads(k, "k", (N, heads, dim), k_cache)
    v = _heads(v, "v", (N, heads, dim), k_cache)
    ks, vs = k.stride(), v.stride()
    args = _lib.StoreKvArgs(N, heads, dim, pages, page_size, k.data_ptr(), v.data_ptr(), ks[0], ks[1], vs[0], vs[1],
                            slots.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), cs[0], cs[1], cs[2])
    _lib.call(dev, _lib.load().dsv41_store_kv, C.byref(args), _lib.current_stream(dev))


# one zeroed workspace per (device, stream, padded head size): its counters are zero between calls. Eager calls that
# overlap on several streams get one each; a replayed graph uses the one of its capture, whatever stream it runs on.
_ws_lock = threading.Lock()
_ws: dict = {}


def attention_workspace(head_dim: int, device=None) -> torch.Tensor:
    """A workspace of its own for tree_attention calls of this head size (or one padded alike: up to 64, 128, 256), zeroed
    on the current stream. For graphs that are replayed at the same time; not for two calls at once."""
    dev = _device(device)
    size = C.c_size_t()
    with torch.cuda.device(dev):
        _lib.check(_lib.load().dsv41_tree_attention_workspace_size(int(head_dim), C.byref(size)), "workspace_size")
        return torch.zeros(size.value, dtype=torch.uint8, device=dev)


def reserve_workspace(head_dim: int, stream: torch.cuda.Stream | None = None, device=None) -> None:
    """Make the workspace that tree_attention calls on `stream` (default: the current one) use, before a capture."""
    dev = stream.device if stream is not None else _device(device)
    with torch.cuda.stream(stream if stream is not None else torch.cuda.current_stream(dev)):
        _workspace(dev, _lib.current_stream(dev), head_dim)


def _device(device) -> torch.device:
    dev = torch.device(device if device is not None else "cuda")
    return dev if dev.index is not None else torch.device("cuda", torch.cuda.current_device())


def _workspace(dev: torch.device, stream: int, head_dim: int) -> tuple[int, int]:
    """Address and size of the stream's workspace."""
    key = (dev.index, stream, 64 if head_dim <= 64 else 128 if head_dim <= 128 else 256)
    got = _ws.get(key)
    if got is None:
        with _ws_lock, torch.cuda.device(dev):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("dsv41: workspace must be allocated before CUDA-graph capture (run once eagerly on the capture "
                                   "stream, call paged.reserve_workspace for it, or pass workspace=)")
            buf = attention_workspace(head_dim, dev)
            got = _ws.setdefault(key, (buf.data_ptr(), buf.numel(), buf))
    return got[:2]


def read_status(device=None, workspace: torch.Tensor | None = None) -> int:
    """Synchronise the current stream; return (then clear) the status of the device's tree_attention calls, on whichever
    stream they ran or were captured, or of those that were given `workspace`: 0 = ok, 1 = a bounded device-side wait ran
    out (results since the last read are invalid). Calls that other streams have still to finish report in a later read."""
    if workspace is not None:
        return _read_and_clear(workspace.device, workspace, _lib.current_stream(workspace.device))
    dev = _device(device)
    stream, worst = _lib.current_stream(dev), 0
    for (index, _, _), (_, _, buf) in list(_ws.items()):
        if index == dev.index:
            worst = max(worst, _read_and_clear(dev, buf, stream))
    return worst


def _read_and_clear(dev: torch.device, buf: torch.Tensor, stream: int) -> int:
    st = C.c_int32()
    _lib.call(dev, _lib.load().dsv41_read_status, buf.data_ptr(), stream, C.byref(st))
    if st.value:
        # the counters of a call that gave up are not back at zero; its stream may be another than this one
        torch.cuda.synchronize(dev)
        buf.zero_()
        torch.cuda.synchronize(dev)
    return st.value


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                   seq_lens: torch.Tensor, cu_lens: torch.Tensor, max_new: int, *, tree_mask: torch.Tensor | None = None,
                   scale: float | None = None, out: torch.Tensor | None = None, return_lse: bool = False,
                   workspace: torch.Tensor | None = None):
    """Attention of the step's new tokens over the paged cache that already holds their keys and values.

    q [N, q_heads, head_dim] (the caches' dtype, head_dim up to 256); request b owns rows cu_lens[b]:cu_lens[b + 1]
    and the first seq_lens[b] slots of its pages, the last of them its new tokens. With tree_mask (int64 [N, words],
    step_tables) a token sees the context and the new tokens of its bits, without it the context and the new tokens
    up to itself. max_new is an upper bound on a request's new tokens, scale defaults to head_dim ** -0.5. Query head
    h reads KV head h // (q_heads / kv_heads). A row that sees nothing is 0 with lse -inf. Returns out [N, q_heads,
    head_dim] in q's dtype, or (out, lse fp32 [N, q_heads]); rows past cu_lens[B] are not written. workspace: one of
    attention_workspace's, which no other call may use at the same time (default: the stream's own)."""
    (pages, page_size, kv_heads, dim), cs, dev = _cache(k_cache, v_cache)
    if q.dim() != 3 or q.shape[1] == 0 or q.shape[1] % kv_heads:
        raise ValueError(f"q must be [N, q_heads, {dim}] with q_heads a multiple of {kv_heads}")
    N, q_heads, _ = q.shape
    q = _heads(q, "q", (N, q_heads, dim), k_cache)
    if seq_lens.dim() != 1:
        raise ValueError("seq_lens must be int32 [B]")
    B = seq_lens.shape[0]
    seq_lens = _vector(seq_lens, "seq_lens", B, torch.int32, dev)
    cu_lens = _vector(cu_lens, "cu_lens", B + 1, torch.int32, dev)
    table, width, table_stride = _table(block_table, B, dev)
    words, mask = 1, None
    if tree_mask is not None:
        if tree_mask.dtype is not torch.int64 or tree_mask.dim() != 2 or tree_mask.shape[0] != N or tree_mask.device != dev:
            raise ValueError(f"tree_mask must be int64 [{N}, words] on {dev}")
        words = tree_mask.shape[1]
        tree_mask = tree_mask.contiguous()
        mask = tree_mask.data_ptr()
    if out is None:
        out = q.new_empty((N, q_heads, dim))
        os = (q_heads * dim, dim)
    else:
        os = out.stride()
        if (out.shape != (N, q_heads, dim) or out.dtype is not q.dtype or out.device != dev or os[2] != 1 or os[0] % 8
                or os[1] % 8 or out.data_ptr() % 16):
            raise ValueError("out must be like q, with contiguous, 16-byte aligned heads")
    lse = q.new_empty((N, q_heads), dtype=torch.float32) if return_lse else None
    stream = _lib.current_stream(dev)
    if workspace is None:
        ws, ws_bytes = _workspace(dev, stream, dim)
    else:
        if workspace.dtype is not torch.uint8 or not workspace.is_contiguous() or workspace.device != dev:
            raise ValueError(f"workspace must be one of attention_workspace's on {dev}")
        ws, ws_bytes = workspace.data_ptr(), workspace.numel()
    qs = q.stride()
    args = _lib.TreeAttentionArgs(
        _DTYPES[q.dtype], B, N, int(max_new), q_heads, kv_heads, dim, page_size, pages, min(width * page_size, 0x7fffff00),
        q.data_ptr(), qs[0], qs[1], k_cache.data_ptr(), v_cache.data_ptr(), cs[0], cs[1], cs[2], table, table_stride,
        seq_lens.data_ptr(), cu_lens.data_ptr(), mask, words, dim ** -0.5 if scale is None else float(scale), out.data_ptr(),
        os[0], os[1], lse.data_ptr() if lse is not None else None)
    _lib.call(dev, _lib.load().dsv41_tree_attention, C.byref(args), ws, ws_bytes, stream)
    return (out, lse) if return_lse else out
