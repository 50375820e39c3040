"""Scores of logits: what the C side and the Python side refuse, without a GPU."""
import ctypes as C

import pytest
import torch

from dsv41_flash_offload_b200 import _lib, logprobs
from test_step_host import FAKE, _err


def _call(**kw):
    a = dict(dtype=2, rows=2, vocab=100, given=1, top=4, logits=FAKE, row_stride=100, tokens=FAKE, logprobs=FAKE, entropy=FAKE, lse=FAKE,
             top_ids=FAKE, top_logprobs=FAKE)
    return _lib.load().dsv41_token_logprobs(C.byref(_lib.TokenLogprobsArgs(**{**a, **kw})), None)


def test_refusals():
    for kw, text in ((dict(dtype=3), b"dtype"), (dict(rows=-1), b"rows"), (dict(rows=1 << 28), b"rows"), (dict(vocab=0), b"vocab"),
                     (dict(vocab=0x7fffffff), b"vocab"), (dict(given=-1), b"given"), (dict(given=1025), b"given"), (dict(top=33), b"top"),
                     (dict(top=-1), b"top"), (dict(row_stride=-4), b"row_stride"), (dict(logits=None), b"NULL"), (dict(tokens=None), b"NULL"),
                     (dict(entropy=None), b"NULL"), (dict(top_ids=None), b"NULL"), (dict(logits=FAKE + 2), b"misaligned"),
                     (dict(tokens=FAKE + 4), b"misaligned")):
        _err(_call(**kw), text)
    assert _lib.load().dsv41_token_logprobs(None, None) == _lib.E_INVALID
    assert _call(rows=0) == 0


def test_python_refuses_cpu_tensors():
    with pytest.raises(ValueError):
        logprobs.token_logprobs(torch.zeros(2, 10), torch.zeros(2, dtype=torch.int64))
