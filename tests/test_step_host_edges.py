"""CPU-only tests of what the decode-step operators refuse before any device work."""
from test_step_host import FAKE, _attn, _err, _store  # noqa: F401


def test_outputs_that_repeat_in_memory_are_refused():
    for kw in (dict(stride_page=0), dict(stride_slot=0), dict(stride_head=0)):
        _err(_store(**kw), b"repeat")
    for kw in (dict(out_stride_token=0), dict(out_stride_head=0)):
        _err(_attn(**kw), b"repeats")
