"""One decode step with drafted tokens through a layer: page tables, 4-bit projections, cache store, tree attention,
router, routed experts and a shared expert, then the scores of the drafted tokens, every product and every piece of
bookkeeping on the GPU.

    python examples/draft_step.py [--steps 4] [--requests 6] [--bits 4] [--window 24 --sinks 4]

`DraftLayer.forward` is the step as a serving engine would run it (positional encoding and normalisation, which this
framework leaves to the engine, are left out); `main` drafts random trees, accepts a path of each and goes on, as a
speculative decoder does. All weights are random.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from dsv41_flash_offload_b200 import exl3, paged, w4  # noqa: E402


class PagedCache:
    """A layer's keys and values, and the tables all layers share."""

    def __init__(self, requests, pages, page_size, width, kv_heads, head_dim, device="cuda", bits=16):
        shape = (pages, page_size, kv_heads, head_dim)
        self.page_size, self.bits = page_size, bits
        if bits == 4:
            self.packed = paged.Cache4(*shape, dtype=torch.float16, device=device)
        else:
            self.k, self.v = (torch.empty(shape, dtype=torch.float16, device=device) for _ in range(2))
        self.block_table = torch.zeros(requests, width, dtype=torch.int32, device=device)
        self.free_pages = torch.arange(pages, dtype=torch.int32, device=device)
        self.free_count = torch.full((1,), pages, dtype=torch.int32, device=device)
        self.held_pages = torch.zeros(requests, dtype=torch.int32, device=device)

    def begin(self, context_lens, new_lens, tokens, parents=None):
        t = paged.step_tables(context_lens, new_lens, self.held_pages, self.block_table, self.free_pages, self.free_count,
                              self.page_size, tokens, parents=parents)
        self.held_pages, self.free_count = t.held_pages, t.free_count
        return t

    def keep(self, tables, accepted, context_lens):
        """Move the accepted tokens of each drafted tree (indices into the step's batch, in path order, one list per
        request) to the positions right after the context. The pages they leave go back at the next begin()."""
        src = [i for path in accepted for i in path]
        if not src:
            return
        dev = self.block_table.device
        req = torch.tensor([b for b, path in enumerate(accepted) for _ in path], device=dev)
        pos = torch.tensor([j for path in accepted for j in range(len(path))], device=dev) + context_lens.long()[req]
        dst = self.block_table[req, pos // self.page_size].long() * self.page_size + pos % self.page_size
        slots = tables.slots[torch.tensor(src, device=dev)]
        if self.bits == 4:
            return paged.move_kv4(slots, dst, self.packed)
        for cache in (self.k, self.v):
            flat = cache.view(-1, *cache.shape[2:])
            flat[dst] = flat[slots]

    def attend(self, q, k, v, t, max_new, **kw):
        """Store the step's keys and values, then attend to what its tokens see."""
        lists = (self.block_table, t.seq_lens, t.cu_lens, max_new)
        if self.bits == 4:
            paged.store_kv4(k, v, t.slots, self.packed)
            return paged.tree_attention4(q, self.packed, *lists, tree_mask=t.tree_mask, **kw)
        paged.store_kv(k, v, t.slots, self.k, self.v)
        return paged.tree_attention(q, self.k, self.v, *lists, tree_mask=t.tree_mask, **kw)


class DraftLayer:
    """Attention and MoE of one layer, dense weights in 4 bits, experts in the trellis format."""

    def __init__(self, hidden=512, intermediate=256, experts=8, topk=2, q_heads=8, kv_heads=2, head_dim=64, seed=0, device="cuda",
                 window=None, sinks=0):
        self.window, self.sinks = window, sinks
        g = torch.Generator().manual_seed(seed)
        rand = lambda n, k: (torch.randn(n, k, generator=g) * k ** -0.5).half().to(device)
        self.q_heads, self.kv_heads, self.head_dim, self.topk = q_heads, kv_heads, head_dim, topk
        dense = dict(qkv=rand((q_heads + 2 * kv_heads) * head_dim, hidden), out=rand(hidden, q_heads * head_dim),
                     gate=rand(intermediate, hidden), up=rand(intermediate, hidden), down=rand(hidden, intermediate))
        for name, weight in dense.items():
            setattr(self, name, w4.W4Weight.quantize(weight, 64))
        self.router = rand(experts, hidden)
        self.experts = exl3.Exl3MoELayer.synthetic(experts, hidden, intermediate, seed=seed, device=device)

    def forward(self, x, cache, t, max_new):
        """x fp16 [N, hidden], the step's token batch -> fp16 [N, hidden]."""
        n = x.shape[0]
        qkv = w4.linear(x, self.qkv).view(n, -1, self.head_dim)
        q, k, v = qkv.split((self.q_heads, self.kv_heads, self.kv_heads), 1)
        a = cache.attend(q, k, v, t, max_new, window=self.window, sinks=self.sinks)
        h = w4.linear(a.view(n, -1), self.out, out=x.float(), accumulate=True)          # residual
        h16 = h.half()
        y = exl3.apply_exl3_fused_moe_logits(h16, h16 @ self.router.t(), self.experts, self.topk, exl3.SWIGLU_LIMIT_DEFAULT)
        w4.shared_expert(h16, self.gate, self.up, self.down, exl3.SWIGLU_LIMIT_DEFAULT, out=y)
        return (h + y).half()


def draft_trees(rng, requests, most):
    """Random trees: sizes, and each token's parent (an earlier token of its request, or -1)."""
    new = torch.randint(1, most + 1, (requests,), generator=rng).tolist()
    parents = [int(torch.randint(-1, i, (1,), generator=rng)) if i else -1 for n in new for i in range(n)]
    return new, parents


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=4)
    ap.add_argument("--requests", type=int, default=6)
    ap.add_argument("--bits", type=int, default=16, choices=(16, 4), help="of the cache")
    ap.add_argument("--window", type=int, default=None, help="keys that a token sees, and the first --sinks")
    ap.add_argument("--sinks", type=int, default=0)
    args = ap.parse_args()
    rng = torch.Generator().manual_seed(1)
    layer, hidden, vocab = DraftLayer(window=args.window, sinks=args.sinks), 512, 1000
    head = w4.W4Weight.quantize((torch.randn(vocab, hidden, generator=rng) * hidden ** -0.5).half().cuda(), 64)
    cache = PagedCache(args.requests, 64, 16, 16, layer.kv_heads, layer.head_dim, bits=args.bits)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")

    context = [0] * args.requests
    prompt = torch.randint(1, 40, (args.requests,), generator=rng).tolist()
    t = cache.begin(i32(context), i32(prompt), sum(prompt))                             # prompts: causal, no tree
    layer.forward(torch.randn(sum(prompt), hidden, generator=rng).half().cuda(), cache, t, max(prompt))
    context = prompt
    for step in range(args.steps):
        new, parents = draft_trees(rng, args.requests, 8)
        t = cache.begin(i32(context), i32(new), sum(new), i32(parents))
        y = layer.forward(torch.randn(sum(new), hidden, generator=rng).half().cuda(), cache, t, max(new))
        # what the model says of the drafted tokens: each one's log probability after its parent (a verifier compares these with the
        # draft's), the entropy there and the likeliest tokens
        drafted = torch.randint(0, vocab, (sum(new),), generator=rng).cuda()
        scores = w4.head_logprobs(y, head, drafted, top=4)
        # here the path to each request's last token is accepted
        accepted, base = [], 0
        for n in new:
            path, i = [], n - 1
            while i >= 0:
                path.insert(0, base + i)
                i = parents[base + i]
            accepted.append(path)
            base += n
        cache.keep(t, accepted, i32(context))
        context = [c + len(path) for c, path in zip(context, accepted)]
        assert not bool(t.status.any()) and paged.read_status() == 0
        print(f"step {step}: {sum(new)} drafted tokens, {sum(map(len, accepted))} accepted, lengths {context}, "
              f"|y| {float(y.float().abs().mean()):.4f}, mean log probability {float(scores.logprobs.mean()):.3f}, free pages {int(t.free_count)}")


if __name__ == "__main__":
    main()
