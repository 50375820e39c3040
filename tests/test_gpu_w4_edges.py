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


def test_silu_of_large_gates():
    """Gates that are one input each (code 9, zero point 8, scale 1) against an up product of 1. fp32 exp, sum and divide:
    at most 8 units of the result; below 2^-126 a result may be 0."""
    gate, up = torch.full((31, 32), 8, dtype=torch.uint8), torch.full((31, 32), 8, dtype=torch.uint8)
    gate[torch.arange(31), torch.arange(31)] = 9
    up[:, 31] = 9
    pack = lambda c: w4.W4Weight((c[:, 0::2] | c[:, 1::2] << 4).to(DEV), torch.ones(31, 1, dtype=torch.float16, device=DEV))
    for base in (-85.0, -60.0, -30.0, -8.0, 0.0, 25.0):
        x = torch.cat((base + torch.arange(31) * 0.34375, torch.ones(1))).half()[None]
        got = w4.gated(x.to(DEV), pack(gate), pack(up), None, out_dtype=torch.float32).cpu().double()[0]
        g = x[0, :31].double()
        want = g / (1.0 + torch.exp(-g))
        assert bool(((got - want).abs() <= 8 * 2.0 ** -23 * want.abs() + 2.0 ** -126).all()), base


@pytest.mark.parametrize("n,k,group,zeros", [(40000, 256, 64, True), (60001, 128, 128, False), (38000, 1024, 32, False), (700, 8192, 128, True)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_tiles_of_one_warp_and_of_many(n, k, group, zeros, dtype):
    """Warps that hold whole row tiles, and tiles that 16 warps share. fp32 sums: group / 16 matrix instructions a group,
    one addition a group, one a warp, each off by at most 2^-22 of S = sum |w x| (tensor cores may truncate)."""
    w, dense = make(n, k, group, zeros, dtype, n)
    dense = dense.to(DEV)
    for tokens in (1, 11, 25):
        x = torch.randn(tokens, k, generator=torch.Generator().manual_seed(tokens)).to(dtype).to(DEV)
        got = w4.linear(x, w, out_dtype=torch.float32).double()
        bound = (group / 16 + k / group + 16) * 2.0 ** -22 * (x.double().abs() @ dense.abs().t())
        assert bool(((got - x.double() @ dense.t()).abs() <= bound).all()), tokens
