"""The end of bf16's range in a cache in 4 bits: groups whose hi - lo is just below what fp32 holds are stored as any other, groups where it
passes fp32 stand for NaN, and neither touches the groups beside them."""
import pytest
import torch

from dsv41_flash_offload_b200 import paged
from test_gpu_kv4 import check_store, stored
from test_gpu_paged import DEV

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
HALF = 2.0 ** 127
BELOW = HALF * (1 - 2.0 ** -8)      # the number before it


def group(lo, hi, seed):
    """32 values of [lo, hi] in bf16, both ends among them."""
    g = torch.Generator().manual_seed(seed)
    x = (torch.rand(32, generator=g, dtype=torch.float64) * (hi / 2 - lo / 2) * 2 + lo).clamp(lo, hi)
    x[3], x[20] = lo, hi
    return x.to(BF16)


@pytest.mark.parametrize("lo,hi", [(-HALF, BELOW), (-BELOW, HALF), (-1.5 * HALF, 0.49 * HALF), (0.0, torch.finfo(BF16).max), (-torch.finfo(BF16).max, 0.0),
                                   (-BELOW, BELOW)])
def test_ranges_that_fp32_holds(lo, hi):
    assert torch.isfinite(torch.tensor(hi - lo, dtype=torch.float64).float())
    other = torch.randn(9, 32, generator=torch.Generator().manual_seed(2)).to(BF16)
    x = torch.stack([torch.cat((group(lo, hi, i), other[i])) for i in range(9)])[:, None].contiguous()
    check_store(x, -x.flip(0), 8, BF16)
    cache, slots = stored(x, x, 8, BF16)
    assert bool(torch.isfinite(paged.load_kv4(slots.to(DEV), cache)[0].float()).all())


@pytest.mark.parametrize("lo,hi", [(-HALF, HALF), (-1.25 * HALF, 1.25 * HALF), (-torch.finfo(BF16).max, torch.finfo(BF16).max), (-1.75 * HALF, 0.25 * HALF)])
def test_ranges_past_fp32_are_nan(lo, hi):
    small = torch.randn(9, 32, generator=torch.Generator().manual_seed(1)).to(BF16)
    x = torch.stack([torch.cat((small[i], group(lo, hi, i), small[i])) for i in range(9)])[:, None].contiguous()
    assert bool(torch.isfinite(x.float()).all())
    plain = torch.cat((small, small, small), 1)[:, None].contiguous()
    (cache, slots), (other, _) = stored(x, x, 8, BF16), stored(plain, plain, 8, BF16)
    for got, want in zip(paged.load_kv4(slots.to(DEV), cache), paged.load_kv4(slots.to(DEV), other)):
        assert bool(torch.isnan(got[..., 32:64]).all())
        for at in (slice(0, 32), slice(64, 96)):
            assert torch.equal(got[..., at], want[..., at])
