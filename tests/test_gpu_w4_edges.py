"""4-bit products of infinities and NaN, and SwiGLU far from zero."""
import math

import pytest
import torch

from dsv41_flash_offload_b200 import w4
from test_gpu_w4 import DEV, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("limit", [None, 10.0])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens", [4, 12, 30])
def test_gated_keeps_nan(tokens, dtype, limit):
    """min(silu(g), L) * clamp(u, -L, L) of the products' infinities and NaN, as the definition has it: silu(-inf) is
    -inf / inf, and a clamp keeps NaN."""
    wg, dg = make(40, 128, 64, True, dtype, 3)
    wu, du = make(40, 128, 64, True, dtype, 4)
    x = torch.randn(tokens, 128, generator=torch.Generator().manual_seed(5)).to(dtype).to(DEV)
    for out_dtype in (torch.float32, dtype):
        clean = w4.gated(x, wg, wu, limit, out_dtype=out_dtype)
        for value in (math.nan, math.inf, -math.inf):
            bad = x.clone()
            bad[2, 7] = value
            got = w4.gated(bad, wg, wu, limit, out_dtype=out_dtype).cpu()
            xd = bad[2].cpu().double()
            g, u = (dg * xd).sum(1), (du * xd).sum(1)
            s = g / (1.0 + torch.exp(-g))
            if limit:
                s, u = s.clamp(max=limit), u.clamp(-limit, limit)
            want = s * u
            assert torch.equal(torch.isnan(got[2]), torch.isnan(want)), (value, out_dtype)
            inf = torch.isinf(want)
            assert torch.equal(got[2][inf].double(), want[inf])
            rest = [t for t in range(tokens) if t != 2]
            assert torch.equal(got[rest], clean.cpu()[rest])
