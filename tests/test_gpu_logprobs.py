"""Scores of logits (logprobs.token_logprobs, w4.head_logprobs) against log softmax in 64 bits; ids against a stable sort.

Bounds, all absolute: L sums V positive fp32 terms, some V / 512 of them one after another and 64 more in trees: relative error
(V / 512 + 64) 2^-24; each term is off by 2^-22 (ex2) and by its argument's rounding, two roundings of |z| 2^-24 relative each and
log2(e) in fp32, weighted by p: at most 2^-22 times the mean of |z| = |x - m|. With Z that mean,
    e = (V / 512 + 64) 2^-24 + 2^-22 (1 + Z)
is the error of log L; a log probability adds its own roundings, 2^-22 (|x - m| + |log L|); the entropy's second sum is off by e
and two roundings, relative to Z."""
import math

import pytest
import torch

from dsv41_flash_offload_b200 import Dsv41Error, logprobs, w4

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def make(rows, vocab, given, dtype, seed=0, scale=2.5):
    g = torch.Generator().manual_seed(seed)
    x = (scale * torch.randn(rows, vocab, generator=g)).to(dtype)
    t = torch.randint(0, vocab, (rows, given) if given != 1 else (rows,), generator=g)
    return x.to(DEV), t.to(DEV)


def check(x, tokens, top, got=None):
    got = got or logprobs.token_logprobs(x, tokens, top)
    n, vocab = x.shape
    d = x.cpu().double()
    t = tokens.cpu().view(n, -1)
    m = d.amax(1, keepdim=True)
    z = d - m
    p = z.exp()
    L = p.sum(1, keepdim=True)
    logL, Z = L.log(), (torch.where(p > 0, p * -z, torch.zeros_like(p)).sum(1, keepdim=True) / L)
    e = (vocab / 512 + 64) * 2.0 ** -24 + 2.0 ** -22 * (1 + Z)
    inside = (t >= 0) & (t < vocab)
    zt = z.gather(1, t.clamp(0, vocab - 1))
    want = torch.where(inside, zt - logL, torch.full_like(zt, -math.inf))
    lp = got.logprobs.cpu().double().view(n, -1)
    fin = torch.isfinite(want)
    assert got.logprobs.shape == tokens.shape and torch.equal(torch.isfinite(lp), fin) and torch.equal(lp[~fin], want[~fin])
    assert bool(((lp - want).abs() <= e + 2.0 ** -22 * (zt.abs() + logL))[fin].all())
    H = (logL + Z)[:, 0]
    assert bool(((got.entropy.cpu().double() - H).abs() <= (e * (1 + Z) + 2.0 ** -22 * (logL + Z))[:, 0]).all())
    lse = (m + logL)[:, 0]
    assert bool(((got.lse.cpu().double() - lse).abs() <= e[:, 0] + 2.0 ** -23 * (lse.abs() + m[:, 0].abs())).all())
    ids, tlp = got.top_ids.cpu(), got.top_logprobs.cpu().double()
    assert ids.shape == tlp.shape == (n, top)
    if top:
        val, order = torch.sort(d, dim=1, descending=True, stable=True)
        k = min(top, vocab)
        val, order = val[:, :k], order[:, :k]
        none = val == -math.inf
        assert torch.equal(ids[:, :k], torch.where(none, torch.full_like(order, -1), order))
        assert bool((ids[:, k:] == -1).all()) and bool((tlp[:, k:] == -math.inf).all())
        want = torch.where(none, val, val - m - logL)
        fin = torch.isfinite(want)
        assert torch.equal(tlp[:, :k][~fin], want[~fin])
        assert bool(((tlp[:, :k] - want).abs() <= e + 2.0 ** -22 * ((val - m).abs() + logL))[fin].all())
    return got


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows,vocab,given,top", [(1, 1, 1, 1), (3, 2, 1, 5), (2, 7, 3, 7), (5, 31, 1, 32), (1, 513, 2, 0), (4, 4097, 1, 20),
                                                  (1, 100001, 1, 5), (2, 65536, 4, 32), (40, 9999, 1, 1), (100, 32768, 4, 20),
                                                  (300, 20001, 1, 32), (7, 163840, 1, 8)])
def test_rows(rows, vocab, given, top, dtype):
    check(*make(rows, vocab, given, dtype, seed=vocab + rows), top)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("rows", [1, 30, 400])
def test_orders_and_ties(rows, dtype):
    """Rows in ascending, descending, constant and coarse order: every way the candidates can fall."""
    v = 30011
    ramp = torch.linspace(-9, 9, v).expand(rows, v)
    t = torch.arange(rows, device=DEV) % v
    for x in (ramp, ramp.flip(1), torch.full((rows, v), 1.25), torch.round(ramp), torch.full((rows, v), -0.0), ramp * 0,
              torch.where(torch.arange(v) % 1000 < 3, 5.0, -5.0).expand(rows, v)):
        check(x.to(dtype).to(DEV).contiguous(), t, 32)
    zeros = torch.zeros(rows, v)
    zeros[:, ::2] = -0.0
    check(zeros.to(dtype).to(DEV), t, 9)


def test_more_candidates_than_the_list_holds():
    """The largest logits all lie with 31 of a row's 512 threads, thousands of them above the 32nd thread's largest."""
    v, rows = 200000, 300
    g = torch.Generator().manual_seed(1)
    owner = (torch.arange(v) // 4) % 512
    x = torch.randn(rows, v, generator=g) - 4.0
    x[:, owner < 31] = torch.rand(rows, int((owner < 31).sum()), generator=g) + 8.0
    check(x.to(DEV), torch.arange(rows, device=DEV), 32)
    x[:, owner < 31] = 9.0
    check(x.to(DEV), torch.arange(rows, device=DEV), 32)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_masked_rows(dtype):
    x, t = make(64, 5003, 2, dtype, seed=3)
    low = torch.finfo(dtype).min
    x[0] = -math.inf
    x[1] = -math.inf
    x[1, 77] = 3.0
    x[2, :] = low                              # uniform, at the type's lowest value
    x[3, 5:] = low
    x[4] = -math.inf
    x[4, 100:110] = low
    x[5, ::2] = -math.inf
    x[6] = torch.finfo(dtype).max
    x[7, :] = torch.finfo(dtype).max
    x[7, 4000] = low
    x[8, 1:] = -math.inf
    t[1, 0], t[9, 0], t[9, 1], t[10, 1] = 77, -1, 5003, 2 ** 40
    t[0] = 5
    got = logprobs.token_logprobs(x, t, 12)
    keep = [i for i in range(64) if i != 0]
    check(x[keep], t[keep], 12, logprobs.TokenLogprobs(*(f[keep] for f in got)))
    assert bool((got.logprobs[0] == -math.inf).all()) and float(got.entropy[0]) == 0 and float(got.lse[0]) == -math.inf
    assert bool((got.top_ids[0] == -1).all()) and bool((got.top_logprobs[0] == -math.inf).all())


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("vocab", [50, 20000])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_without_a_distribution(bad, vocab, dtype):
    x, t = make(6, vocab, 2, dtype, seed=4)
    t[1, 1] = -1
    want = logprobs.token_logprobs(x, t, 6)
    y = x.clone()
    y[1, vocab // 3] = bad
    y[4, 0] = bad
    y[4, 1:] = -math.inf
    got = logprobs.token_logprobs(y, t, 6)
    for i in range(6):
        for a, b in zip(got, want):
            if i not in (1, 4):
                assert torch.equal(a[i], b[i])
            elif a.dtype == torch.int64:
                assert bool((a[i] == -1).all())
            else:
                assert bool(torch.isnan(a[i]).all())


@pytest.mark.parametrize("dtype", [F16, F32])
def test_strides_and_alignment(dtype):
    """Slices of a padded head, odd strides, rows that repeat, columns that do not lie together; int32 tokens."""
    x, t = make(37, 8211, 1, dtype, seed=5)
    want = logprobs.token_logprobs(x, t, 11)
    for off in (1, 2, 3, 5, 7):
        wide = torch.full((37, 8211 + 9 + off), math.nan, dtype=dtype, device=DEV)
        wide[:, off:off + 8211] = x
        for a, b in zip(logprobs.token_logprobs(wide[:, off:off + 8211], t.int(), 11), want):
            # (a row's place in memory decides which thread sums what)
            assert torch.equal(a, b) if a.dtype == torch.int64 else torch.allclose(a, b, rtol=1e-5, atol=1e-5)
        check(wide[:, off:off + 8211], t, 11)
    check(x[3:4].expand(37, 8211), t, 4)
    check(x.t().contiguous().t(), t, 4)
    assert logprobs.token_logprobs(x[:0], t[:0], 3).top_ids.shape == (0, 3)
    assert logprobs.token_logprobs(x, t[:, None][:, :0], 0).logprobs.shape == (37, 0)


def test_offsets_past_32_bits():
    rows, vocab = 33, 131
    big = torch.empty(32 * (1 << 27) + vocab, dtype=BF16, device=DEV)
    x = big.as_strided((rows, vocab), (1 << 27, 1))
    src, t = make(rows, vocab, 1, BF16, seed=6)
    x.copy_(src)
    for a, b in zip(logprobs.token_logprobs(x, t, 5), logprobs.token_logprobs(src, t, 5)):
        assert torch.equal(a, b) if a.dtype == torch.int64 else torch.allclose(a, b, rtol=1e-5, atol=1e-5)


def test_graphs_and_streams():
    x, t = make(12, 50001, 3, F32, seed=7)
    want = logprobs.token_logprobs(x, t, 8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = logprobs.token_logprobs(x, t, 8)
    for _ in range(2):
        for f in got:
            f.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    x.copy_(x.flip(1))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, logprobs.token_logprobs(x, t, 8)))
    with torch.cuda.stream(side):
        again = logprobs.token_logprobs(x, t, 8)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, got))


@pytest.mark.parametrize("n", [0, 1, 30, 600])
def test_head(n):
    g = torch.Generator().manual_seed(8)
    head = w4.W4Weight.quantize((torch.randn(5001, 256, generator=g) * 0.1).half().to(DEV), 64)
    x = torch.randn(n, 256, generator=g).half().to(DEV)
    t = torch.randint(0, 5001, (n, 2), generator=g).to(DEV)
    got = w4.head_logprobs(x, head, t, 6)
    if n:
        check(torch.cat([w4.linear(x[r:r + 256], head, out_dtype=F32) for r in range(0, n, 256)]), t, 6, got)
    assert got.logprobs.shape == (n, 2) and got.top_ids.shape == (n, 6) and got.entropy.shape == (n,)


def test_refusals():
    x, t = make(4, 50, 1, F32)
    for bad in (lambda: logprobs.token_logprobs(x[0], t), lambda: logprobs.token_logprobs(x, t[:3]), lambda: logprobs.token_logprobs(x, t, 33),
                lambda: logprobs.token_logprobs(x, t, -1), lambda: logprobs.token_logprobs(x, t.cpu()),
                lambda: logprobs.token_logprobs(x[:, :0], t), lambda: logprobs.token_logprobs(x, t[:, None].expand(4, 1025))):
        with pytest.raises((ValueError, Dsv41Error)):
            bad()
    for bad in (lambda: logprobs.token_logprobs(x.double(), t), lambda: logprobs.token_logprobs(x, t.float())):
        with pytest.raises(TypeError):
            bad()
