"""CPU-only tests of what the decode-step operators refuse before any device work."""
from test_step_host import _attn, _err, _store


def test_outputs_that_repeat_in_memory_are_refused():
    for kw in (dict(stride_page=0), dict(stride_slot=0), dict(stride_head=0)):
        _err(_store(**kw), b"repeat")
    for kw in (dict(out_stride_token=0), dict(out_stride_head=0)):
        _err(_attn(**kw), b"repeats")


def test_rows_that_pass_32_bits_when_rounded_to_tiles_are_refused():
    for tokens, heads in (((1 << 31) // 4 - 1, 4), ((1 << 31) - 1, 1), ((1 << 31) - 255, 1)):
        _err(_attn(num_tokens=tokens, q_heads=heads, kv_heads=1), b"2^31")
