"""Products with 4-bit weights (w4.linear, w4.gated, w4.shared_expert) against the definition in 64 bits.

Tolerance: all products are exact in fp32 inputs of a fp32 sum, so an output is off by at most the sum's
rounding. An element passes through at most K/128 + 32 roundings (K/16 matrix instructions shared by 8 warps,
the groups' scales, the join of the warps), each at most 2^-22 of S = sum |w x| (two units of fp32, as tensor
cores may truncate), plus half a unit of the output type. SwiGLU carries those errors with its derivatives
(|silu'| <= 1.1)."""
import numpy as np
import pytest
import torch

from dsv41_flash_offload_b200 import Dsv41Error, exl3, w4

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF_UNIT = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.float16, torch.bfloat16)}


def make(n, k, group, zeros, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16, (n, k), generator=g)
    scales = ((torch.rand(n, k // group, generator=g) - 0.3) * 0.05).to(dtype)
    z = torch.randint(0, 16, (n, k // group), generator=g).to(torch.uint8) if zeros else None
    packed = (codes[:, 0::2] | codes[:, 1::2] << 4).to(torch.uint8)
    off = torch.full((n, k // group), 8.0) if z is None else z.double()
    dense = ((codes.view(n, -1, group).double() - off.double()[:, :, None]) * scales.double()[:, :, None]).view(n, k)
    return w4.W4Weight(packed.to(DEV), scales.to(DEV), None if z is None else z.to(DEV)), dense


def ref_and_bound(x, dense):
    xd = x.detach().cpu().double()
    k = dense.shape[1]
    return xd @ dense.t(), (k / 128 + 32) * 2.0 ** -22 * (xd.abs() @ dense.abs().t())


def check(got, ref, bound, what=""):
    bad = (got.detach().cpu().double() - ref).abs() - bound - HALF_UNIT[got.dtype] * ref.abs() - 2.0 ** -25
    assert bool((bad <= 0).all()), f"{what}: over the bound by {float(bad.max())}"


@pytest.mark.parametrize("tokens", [1, 2, 7, 8, 9, 16, 17, 32, 33, 70])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_linear_tokens(tokens, dtype):
    w, dense = make(80, 512, 64, True, dtype, tokens)
    x = torch.randn(tokens, 512, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    ref, bound = ref_and_bound(x, dense)
    for out_dtype in (torch.float32, torch.float16, torch.bfloat16):
        got = w4.linear(x, w, out_dtype=out_dtype)
        assert got.dtype == out_dtype and got.shape == (tokens, 80)
        check(got, ref, bound, f"{tokens} {out_dtype}")


@pytest.mark.parametrize("n,k,group,zeros", [
    (1, 32, 32, False), (1, 128, 128, True), (15, 96, 32, True), (17, 64, 64, False), (33, 2304, 128, False),
    (48, 1056, 32, False), (1000, 640, 128, True), (16, 16384, 64, False), (4096, 2048, 128, False), (129, 320, 64, True),
])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_linear_sizes(n, k, group, zeros, dtype):
    w, dense = make(n, k, group, zeros, dtype, n + k)
    for tokens in (1, 5, 20):
        x = torch.randn(tokens, k, generator=torch.Generator().manual_seed(2)).to(dtype).to(DEV)
        check(w4.linear(x, w, out_dtype=torch.float32), *ref_and_bound(x, dense), f"{n}x{k}")


def test_layout_is_exact():
    """Every code, scale and zero point reaches its place: unit inputs pick single weights, exactly."""
    for dtype in (torch.float16, torch.bfloat16):
        w, dense = make(37, 160, 32, True, dtype, 7)
        got = w4.linear(torch.eye(160, dtype=dtype, device=DEV), w, out_dtype=torch.float32)
        assert torch.equal(got.cpu().double(), dense.t())


@pytest.mark.parametrize("limit", [None, 10.0, 0.5])
@pytest.mark.parametrize("n,k,group,zeros,dtype", [(24, 256, 32, True, torch.float16), (130, 640, 64, False, torch.bfloat16),
                                                    (2304, 512, 128, True, torch.bfloat16)])
def test_gated(n, k, group, zeros, dtype, limit):
    wg, dg = make(n, k, group, zeros, dtype, 3)
    wu, du = make(n, k, group, zeros, dtype, 4)
    for tokens in (1, 6, 32, 40):
        x = (3 * torch.randn(tokens, k, generator=torch.Generator().manual_seed(5))).to(dtype).to(DEV)
        (g, eg), (u, eu) = ref_and_bound(x, dg), ref_and_bound(x, du)
        s = g * torch.sigmoid(g)
        if limit:
            s, u = s.clamp(max=limit), u.clamp(-limit, limit)
        # fp32 exp and divide: 8 units of the silu
        es = 1.1 * eg + 8 * 2.0 ** -23 * s.abs()
        bound = es * u.abs() + eu * s.abs() + es * eu + 2.0 ** -23 * (s * u).abs()
        check(w4.gated(x, wg, wu, limit), s * u, bound, f"gated {tokens}")
        check(w4.gated(x, wg, wu, limit, out_dtype=torch.float32), s * u, bound, f"gated fp32 {tokens}")


def test_gated_extremes():
    """Gates far below zero give 0 (silu(-inf) is a limit, not NaN with -large), far above the clamp."""
    codes = torch.full((16, 16), 0xFF, dtype=torch.uint8, device=DEV)   # 15 - 8 = 7 everywhere
    w = w4.W4Weight(codes, torch.ones(16, 1, dtype=torch.float16, device=DEV))
    x = torch.full((1, 32), 4.0, dtype=torch.float16, device=DEV)       # products 896
    assert torch.equal(w4.gated(x, w, w, 10.0).cpu(), torch.full((1, 16), 100.0, dtype=torch.float16))
    assert torch.equal(w4.gated(-x, w, w, 10.0).cpu().abs(), torch.zeros(1, 16, dtype=torch.float16))


def test_inputs_with_strides_offsets_and_leading_dims():
    w, dense = make(40, 256, 64, False, torch.float16, 8)
    big = torch.randn(6, 3, 600, generator=torch.Generator().manual_seed(6)).half().to(DEV)
    for x in (big[:, 0, 8:264], big[:, 1, 3:259], big[:, :, :256], big[:, :, 1:257].transpose(0, 1), big[0, 0, :256],
              big[:0, 0, :256], big[:1, 0, :256].expand(5, 256)):
        got = w4.linear(x, w, out_dtype=torch.float32)
        assert got.shape == (*x.shape[:-1], 40)
        ref, bound = ref_and_bound(x.reshape(-1, 256), dense)
        check(got.reshape(-1, 40), ref, bound)


def test_out_views_and_accumulate():
    w, dense = make(40, 256, 64, False, torch.bfloat16, 9)
    x = torch.randn(5, 256, generator=torch.Generator().manual_seed(7)).bfloat16().to(DEV)
    ref, bound = ref_and_bound(x, dense)
    buf = torch.full((5, 100), 2.0, device=DEV)
    view = buf[:, 30:70]
    assert w4.linear(x, w, out=view, accumulate=True) is view
    check(view, ref + 2.0, bound + 2.0 ** -23 * (ref.abs() + 2))
    assert float((buf[:, :30] - 2).abs().max()) == 0 and float((buf[:, 70:] - 2).abs().max()) == 0
    check(w4.linear(x, w, out=view), ref, bound)


def test_padding_does_not_read_nan():
    """Tokens and inputs beyond the call's are never multiplied: rows of NaN behind x leave no trace."""
    w, dense = make(20, 96, 32, True, torch.float16, 10)
    buf = torch.full((64, 128), float("nan"), dtype=torch.float16, device=DEV)
    buf[:3, :96] = torch.randn(3, 96, generator=torch.Generator().manual_seed(8)).half().to(DEV)
    check(w4.linear(buf[:3, :96], w, out_dtype=torch.float32), *ref_and_bound(buf[:3, :96], dense))


def test_non_finite_inputs_stay_in_their_row():
    w, dense = make(20, 128, 64, False, torch.float16, 11)
    x = torch.randn(4, 128, generator=torch.Generator().manual_seed(9)).half().to(DEV)
    clean = w4.linear(x, w, out_dtype=torch.float32)
    x[2, 5] = float("nan")
    got = w4.linear(x, w, out_dtype=torch.float32)
    assert bool(torch.isnan(got[2]).all()) and torch.equal(got[[0, 1, 3]], clean[[0, 1, 3]])


def test_repeats_bit_identically_on_other_streams_and_in_a_graph():
    w, _ = make(300, 1024, 128, False, torch.bfloat16, 12)
    x = torch.randn(4, 1024, generator=torch.Generator().manual_seed(10)).bfloat16().to(DEV)
    ref = w4.linear(x, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = w4.linear(x, w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = w4.linear(x, w)
    x.copy_(torch.randn(4, 1024, generator=torch.Generator().manual_seed(11)).bfloat16())
    graph.replay()
    assert torch.equal(out, w4.linear(x, w))


@pytest.mark.parametrize("symmetric", [True, False])
def test_quantize(symmetric):
    dense = torch.randn(48, 256, generator=torch.Generator().manual_seed(12)).half().to(DEV)
    w = w4.W4Weight.quantize(dense, 64, symmetric)
    back = w4.linear(torch.eye(256, dtype=torch.float16, device=DEV), w, out_dtype=torch.float32).t()
    groups = dense.float().view(48, -1, 64)
    step = groups.abs().amax(2) / 7 if symmetric else (groups.amax(2) - groups.amin(2)) / 15
    # half a step of rounding; asymmetric zero points are whole codes, which may shift a group by half a step more
    limit = step * (0.5 if symmetric else 1.0) * 1.01 + 1e-6
    assert bool(((back - dense.float()).view(48, -1, 64).abs().amax(2) <= limit).all())


def test_shared_expert_joins_the_routed_layer():
    H, I, T = 512, 256, 6
    layer = exl3.Exl3MoELayer.synthetic(8, H, I, seed=5, device=DEV)
    g = torch.Generator().manual_seed(13)
    x = torch.randn(T, H, generator=g).half().to(DEV)
    logits = torch.randn(T, 8, generator=g).to(DEV)
    routed = exl3.apply_exl3_fused_moe_logits(x, logits, layer, 2, 10.0)
    (wg, dg), (wu, du), (wd, dd) = make(I, H, 64, False, torch.float16, 14), make(I, H, 64, False, torch.float16, 15), \
        make(H, I, 64, True, torch.float16, 16)
    act = w4.gated(x, wg, wu, 10.0)
    ref, bound = ref_and_bound(act, dd)
    out = w4.shared_expert(x, wg, wu, wd, 10.0, out=routed.clone())
    check(out, ref + routed.cpu().double(), bound + 2.0 ** -23 * (ref.abs() + routed.cpu().double().abs()))


def test_refusals():
    w, _ = make(32, 128, 64, False, torch.float16, 17)
    w2, _ = make(48, 128, 64, False, torch.float16, 17)
    w3, _ = make(32, 128, 32, False, torch.float16, 17)
    x = torch.zeros(2, 128, dtype=torch.float16, device=DEV)
    codes = torch.zeros(4, 64, dtype=torch.uint8, device=DEV)
    scales = torch.zeros(4, 2, dtype=torch.float16, device=DEV)
    for bad in (lambda: w4.linear(x.float(), w), lambda: w4.linear(x[:, :64], w), lambda: w4.linear(x.cpu(), w),
                lambda: w4.linear(x, w, accumulate=True), lambda: w4.linear(x, w, out=torch.empty(2, 31, device=DEV)),
                lambda: w4.linear(x, w, out=torch.empty(2, 32, dtype=torch.float16, device=DEV), accumulate=True),
                lambda: w4.linear(x, w, out_dtype=torch.int32), lambda: w4.gated(x, w, w2), lambda: w4.gated(x, w, w3),
                lambda: w4.W4Weight(codes.int(), scales), lambda: w4.W4Weight(codes, scales.float()),
                lambda: w4.W4Weight(codes, scales[:, :0]), lambda: w4.W4Weight(codes.cpu(), scales),
                lambda: w4.W4Weight(codes, torch.zeros(4, 3, dtype=torch.float16, device=DEV)),
                lambda: w4.W4Weight(codes, torch.zeros(4, 8, dtype=torch.float16, device=DEV)),
                lambda: w4.W4Weight(codes, scales, torch.full((4, 2), 16, dtype=torch.uint8, device=DEV)),
                lambda: w4.W4Weight(codes, scales, torch.zeros(4, 1, dtype=torch.uint8, device=DEV))):
        with pytest.raises((ValueError, TypeError, Dsv41Error)):
            bad()
