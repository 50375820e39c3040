"""Scores of a step's logits: log probabilities of given tokens, entropy, and the likeliest alternatives of every row, in one
pass over the logits.

`token_logprobs` takes logits as they are (a head's output, a slice of a padded one, any type); `w4.head_logprobs` goes from
hidden states through a 4-bit head. All work runs on the current CUDA stream and nothing synchronises the host, so the calls can
be captured in a CUDA graph. Beside the outputs, token_logprobs allocates a copy of tokens that are not contiguous int64 and of
logits whose columns do not lie together; head_logprobs allocates its logits, fp32, of up to 256 rows at a time, and what it joins
the results of more rows from. A captured graph keeps these in its pool.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch

from . import _lib

_DTYPES = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16, torch.float32: _lib.DTYPE_F32}
MAX_TOP, MAX_GIVEN = 32, 1024


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor        # fp32, shaped like the given tokens
    entropy: torch.Tensor         # fp32 [N], in nats
    lse: torch.Tensor             # fp32 [N] log of the sum of exponentials
    top_ids: torch.Tensor         # int64 [N, top]
    top_logprobs: torch.Tensor    # fp32 [N, top]


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0) -> TokenLogprobs:
    """log softmax of logits [N, V] (fp16, bf16 or fp32, contiguous rows of any stride) at the given tokens [N] or [N, m] (int64
    or int32), the rows' entropies, and the `top` (up to 32) tokens with the largest logits in descending order, equal ones by the
    lowest index. A token outside 0..V - 1 has log probability -inf. A logit of -inf is no alternative: places that find
    none hold id -1 and -inf. A row of -inf alone has entropy 0 and lse -inf; a row that holds NaN or +inf is NaN
    throughout, with ids -1."""
    if logits.dim() != 2 or not logits.is_cuda or logits.shape[1] == 0:
        raise ValueError("logits must be a CUDA tensor [N, V]")
    if logits.dtype not in _DTYPES:
        raise TypeError(f"unsupported logits dtype {logits.dtype} (fp16, bf16 or fp32)")
    (n, vocab), dev = logits.shape, logits.device
    if tokens.dim() not in (1, 2) or tokens.shape[0] != n or tokens.device != dev:
        raise ValueError(f"tokens must be [{n}] or [{n}, m] on {dev}")
    if tokens.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"unsupported tokens dtype {tokens.dtype} (int64 or int32)")
    given = tokens.shape[1] if tokens.dim() == 2 else 1
    if given > MAX_GIVEN:
        raise ValueError(f"up to {MAX_GIVEN} tokens a row")
    if not 0 <= top <= MAX_TOP:
        raise ValueError(f"top must be 0..{MAX_TOP}")
    top = int(top)
    if logits.stride(1) != 1 and vocab > 1:
        logits = logits.contiguous()
    if tokens.dtype is not torch.int64 or not tokens.is_contiguous():
        tokens = tokens.to(torch.int64).contiguous()
    # one allocation for all that is fp32
    floats = logits.new_empty(n * (given + 2 + top), dtype=torch.float32)
    logprobs, entropy, lse, top_logprobs = floats.split_with_sizes((n * given, n, n, n * top))
    ids = tokens.new_empty((n, top))
    base = floats.data_ptr()
    at = base + 4 * n * given
    args = _lib.TokenLogprobsArgs(_DTYPES[logits.dtype], n, vocab, given, top, logits.data_ptr(), logits.stride(0), tokens.data_ptr(),
                                  base, at, at + 4 * n, ids.data_ptr(), at + 8 * n)
    _lib.call(dev, _lib.load().dsv41_token_logprobs, C.byref(args), _lib.current_stream(dev))
    return TokenLogprobs(logprobs if tokens.dim() == 1 else logprobs.view(n, given), entropy, lse, ids, top_logprobs.view(n, top))
