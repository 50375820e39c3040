"""The step of examples/draft_step.py against a restatement of it that shares none of its kernels: 4-bit weights
dequantised from their codes, attention token by token over lists of keys and values, SwiGLU and all products in 64
bits, rounded to fp16 where the step stores fp16; the routed experts by the CPU oracle. Bound: the layer's parity bar
(max-abs 2e-2, cosine 0.9999)."""
import numpy as np
import pytest
import torch

from conftest import assert_close_layer
from dsv41_flash_offload_b200 import exl3, paged, w4
from moe_ref import oracle_out
from test_gpu_draft_step import _example, i32

pytestmark = pytest.mark.gpu


class PlainStep:
    def __init__(self, layer, codes, oracle):
        self.layer, self.oracle = layer, oracle
        self.w = {name: self.dense(*codes[getattr(layer, name)]) for name in ("qkv", "out", "gate", "up", "down")}
        self.router = layer.router.cpu().double()

    @staticmethod
    def dense(codes, scales):
        q = torch.stack((codes & 15, codes >> 4), 2).view(codes.shape[0], scales.shape[1], -1).double()
        return ((q - 8) * scales.double()[:, :, None]).view(codes.shape[0], -1)

    def forward(self, x, keys, values, new, sees):
        """x fp16 [N, hidden]; keys, values: a list of a request's [kv_heads, dim] each, which grows by the new tokens;
        sees[t]: new tokens of its request that token t sees. Also the router's margin at each token."""
        lay, n, r16 = self.layer, x.shape[0], lambda v: v.half().double()
        x = x.cpu().double()
        qkv = r16(x @ self.w["qkv"].t()).view(n, -1, lay.head_dim)
        q, k, v = qkv.split((lay.q_heads, lay.kv_heads, lay.kv_heads), 1)
        att, base = torch.zeros(n, lay.q_heads, lay.head_dim, dtype=torch.float64), 0
        for b, count in enumerate(new):
            ctx = len(keys[b])
            keys[b] += [k[base + i] for i in range(count)]
            values[b] += [v[base + i] for i in range(count)]
            for i in range(count):
                at = list(range(ctx)) + [ctx + j for j in sees[base + i]]
                for h in range(lay.q_heads):
                    g = h // (lay.q_heads // lay.kv_heads)
                    p = torch.softmax(torch.stack([keys[b][j][g] for j in at]) @ q[base + i, h] * lay.head_dim ** -0.5, 0)
                    att[base + i, h] = p @ torch.stack([values[b][j][g] for j in at])
            base += count
        h = x + r16(att).view(n, -1) @ self.w["out"].t()
        h16 = r16(h)
        logits = r16(h16 @ self.router.t())
        top = logits.topk(lay.topk + 1, 1)
        ids, weights = top.indices[:, :lay.topk], torch.softmax(top.values[:, :lay.topk], 1)
        y = torch.from_numpy(np.asarray(oracle_out(self.oracle, lay.experts, h16.half(), ids, weights, exl3.SWIGLU_LIMIT_DEFAULT))).double()
        gate, up, lim = h16 @ self.w["gate"].t(), h16 @ self.w["up"].t(), exl3.SWIGLU_LIMIT_DEFAULT
        act = r16((gate * torch.sigmoid(gate)).clamp(max=lim) * up.clamp(-lim, lim))
        return r16(h + y + act @ self.w["down"].t()), top.values[:, lay.topk - 1] - top.values[:, lay.topk]


def test_a_drafted_step_is_the_plain_one(oracle, monkeypatch):
    codes, init = {}, w4.W4Weight.__init__

    def keep(self, c, scales, zeros=None):
        init(self, c, scales, zeros)
        codes[self] = (c.cpu(), scales.cpu())

    monkeypatch.setattr(w4.W4Weight, "__init__", keep)
    ex = _example()
    layer = ex.DraftLayer(seed=4)
    plain = PlainStep(layer, codes, oracle)
    rng = torch.Generator().manual_seed(6)
    prompt, new, parents = [19, 40, 1], [5, 3, 7], [-1, 0, 0, 1, 3, -1, 0, 1, -1, 0, 1, 1, 0, 4, -1]
    cache = ex.PagedCache(3, 24, 16, 8, layer.kv_heads, layer.head_dim)
    keys, values = [[] for _ in prompt], [[] for _ in prompt]

    def compare(x, got, want, margin):
        clear = margin > 2.0 ** -7              # a router is not asked to decide a near tie
        assert int(clear.sum()) >= x.shape[0] // 2
        assert_close_layer(got.cpu()[clear].numpy(), want[clear].numpy(), "drafted step")

    x = torch.randn(sum(prompt), 512, generator=rng).half().cuda()
    t = cache.begin(i32([0, 0, 0]), i32(prompt), sum(prompt))
    compare(x, layer.forward(x, cache, t, max(prompt)), *plain.forward(x, keys, values, prompt, [range(i + 1) for n in prompt for i in range(n)]))

    sees, base = [], 0
    for n in new:
        for i in range(n):
            path, at = [], i
            while at >= 0:
                path.insert(0, at)
                at = parents[base + at]
            sees.append(path)
        base += n
    x = torch.randn(sum(new), 512, generator=rng).half().cuda()
    t = cache.begin(i32(prompt), i32(new), sum(new), i32(parents))
    compare(x, layer.forward(x, cache, t, max(new)), *plain.forward(x, keys, values, new, sees))
    assert paged.read_status() == 0 and not bool(t.status.any())
