"""What the operators around the routed experts cost, case by case.

A decode step with drafted tokens runs, around the routed-expert layer: the block tables and slot maps of
the step, the 4-bit products of the dense weights (projections, shared expert, head), the store of the new
keys and values into the paged cache, and the attention of each drafted tree over that cache. `listed()`
holds one case for each of the sizes such a program meets, `draw()` makes more of the same ranges,
`run()` is one pass through an operator: in plain torch where `own` is false, through the framework's
entry points (`w4`, `paged`) where it is true. `exact()` gives the same outputs from the operators'
definitions in 64 bits.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
_DT = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def listed():
    return [
        # the down product of a shared expert for one token: the latency of the smallest 4-bit product
        _linear("w4-down-one", tokens=1, n=4096, k=2048, group=128, zeros=False, dtype="float16", out="float32"),
        # gate and up of a shared expert with SwiGLU for a few drafted tokens, at the 5120/2304 layer shape
        _gated("w4-gated-draft", tokens=6, n=2304, k=5120, group=64, zeros=True, dtype="bfloat16"),
        # the same for a full decode batch at the 4096/2048 shape, finest groups
        _gated("w4-gated-batch", tokens=32, n=2048, k=4096, group=32, zeros=False, dtype="float16"),
        # an output head over an odd vocabulary for four tokens: the bandwidth of the weight stream
        _linear("w4-head", tokens=4, n=100001, k=4096, group=128, zeros=False, dtype="bfloat16", out="float32"),
        # the tables of a decode step with drafted trees: a few dozen requests, latency only
        _tables("tables-draft", batch=48, new=(1, 16), ctx=(1, 8000), page=16, tree=True),
        # the tables of a step that prefills many prompts of uneven lengths, some requests finished
        _tables("tables-prefill", batch=512, new=(0, 2048), ctx=(0, 6000), page=64, tree=False),
        # keys and values of a decode step's drafted tokens into their slots
        _store("store-draft", tokens=100, kv_heads=8, dim=128, page=16, dtype="bfloat16"),
        # keys and values of a prefill chunk into their slots
        _store("store-prefill", tokens=16384, kv_heads=8, dim=128, page=64, dtype="float16"),
        # one request, one token, no tree: the latency of the smallest attention call
        _tree("attn-one", batch=1, new=(1, 1), ctx=(2047, 2047), q_heads=32, kv_heads=8, dim=128, page=16,
              tree=False, dtype="bfloat16"),
        # a decode batch with small drafted trees of uneven sizes over uneven contexts
        _tree("attn-draft", batch=16, new=(5, 13), ctx=(100, 4000), q_heads=32, kv_heads=8, dim=128, page=16,
              tree=True, dtype="float16"),
        # few requests with very long contexts: the bandwidth of the cache
        _tree("attn-long", batch=4, new=(16, 16), ctx=(65536, 131056), q_heads=64, kv_heads=8, dim=128, page=64,
              tree=True, dtype="bfloat16"),
        # wide trees: many rows for each key, products and exponentials bound it
        _tree("attn-wide", batch=32, new=(61, 64), ctx=(1000, 8192), q_heads=32, kv_heads=8, dim=128, page=32,
              tree=True, dtype="bfloat16"),
    ]


def _linear(name, **kw):
    return dict(kw, name=name, op="linear")


def _gated(name, **kw):
    return dict(kw, name=name, op="gated")


def _ranged(kw):
    kw = dict(kw)
    for key in ("new", "ctx"):
        lo, hi = kw.pop(key)
        kw[key + "_min"], kw[key + "_max"] = lo, hi
    return kw


def _tables(name, **kw):
    return dict(_ranged(kw), name=name, op="tables")


def _store(name, **kw):
    return dict(kw, name=name, op="store")


def _tree(name, **kw):
    return dict(_ranged(kw), name=name, op="tree")


def _log_int(rng, lo, hi):
    """A whole number of lo..hi, spread evenly over its logarithm."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    while True:
        case = _draw(rng)
        w = work(case)
        if w["bytes"] <= 1.5e9 and w["flops"] <= 1.5e11:
            return case


def _draw(rng):
    op = rng.choice(("linear", "gated", "tables", "store", "tree", "tree"))
    if op in ("linear", "gated"):
        group = rng.choice((32, 64, 128))
        case = dict(op=op, tokens=_log_int(rng, 1, 32), group=group, zeros=rng.random() < 0.5,
                    k=group * _log_int(rng, 2, 16384 // group), dtype=rng.choice(("float16", "bfloat16")))
        case["n"] = _log_int(rng, 48, min(100001, 200_000_000 // case["k"]))
        if op == "linear":
            case["out"] = rng.choice(("float32", case["dtype"]))
        return case
    if op == "tables":
        tree = rng.random() < 0.6
        new = (rng.randint(0, 1), _log_int(rng, 1, 64)) if tree else (0, _log_int(rng, 1, 2048))
        return _strip(_tables("", batch=_log_int(rng, 1, 512), new=new, ctx=(0, _log_int(rng, 1, 16000)),
                              page=rng.choice((1, 8, 16, 24, 32, 64, 128)), tree=tree))
    dtype = rng.choice(("float16", "bfloat16"))
    if op == "store":
        return _strip(_store("", tokens=_log_int(rng, 1, 16384), kv_heads=rng.choice((1, 2, 3, 4, 8)),
                             dim=rng.choice((64, 80, 96, 128, 256)), page=rng.choice((1, 8, 16, 24, 32, 64)),
                             dtype=dtype))
    kv = rng.choice((1, 2, 3, 4, 8))
    hi = _log_int(rng, 1, 64)
    ctx = _log_int(rng, 1, 65536)
    return _strip(_tree("", batch=_log_int(rng, 1, 64), new=(rng.randint(1, hi), hi), ctx=(rng.randint(0, ctx), ctx),
                        q_heads=kv * rng.choice((1, 2, 3, 4, 5, 8, 16)), kv_heads=kv,
                        dim=rng.choice((64, 80, 96, 128, 128, 256)), page=rng.choice((1, 8, 16, 24, 32, 64, 128)),
                        tree=rng.random() < 0.7, dtype=dtype))


def _strip(case):
    case.pop("name")
    return case


# ------------------------------------------------------------------------------------------------
# lengths (plain numbers that follow from the case alone) and work
# ------------------------------------------------------------------------------------------------
def _spread(lo, hi, count, step):
    """`count` lengths of lo..hi: both ends, and a low-discrepancy sequence between them."""
    out = [int(lo + (hi - lo) * ((0.5 + step * i) % 1.0) + 0.5) for i in range(count)]
    if count > 1:
        out[0], out[-1] = hi, lo
    return out


def _lens(case):
    ctx = _spread(case["ctx_min"], case["ctx_max"], case["batch"], 0.6180339887)
    new = _spread(case["new_min"], case["new_max"], case["batch"], 0.7548776662)
    return ctx, new


def _pages(tokens, page):
    return (tokens + page - 1) // page


def work(case):
    op = case["op"]
    if op in ("linear", "gated"):
        t, n, k, g = case["tokens"], case["n"], case["k"], case["group"]
        mats = 2 if op == "gated" else 1
        weights = mats * (n * k // 2 + n * (k // g) * (3 if case["zeros"] else 2))
        out = t * n * (4 if op == "linear" and case["out"] == "float32" else 2)
        return {"bytes": weights + t * k * 2 + out, "flops": 2 * t * n * k * mats}
    if op == "store":
        row = case["kv_heads"] * case["dim"] * 2
        return {"bytes": case["tokens"] * (4 * row + 8), "flops": 0}
    ctx, new = _lens(case)
    page = case["page"]
    if op == "tables":
        held = _held(case, ctx, new)
        moved = sum(abs(_pages(c + n, page) - h) for c, n, h in zip(ctx, new, held))
        per_token = 8 + 4 + 4 + (8 + 4 if case["tree"] else 0)
        return {"bytes": sum(new) * per_token + moved * 8 + case["batch"] * 24, "flops": 0}
    hq, hk, d = case["q_heads"], case["kv_heads"], case["dim"]
    keys = sum(c + n for c, n in zip(ctx, new))
    pairs = sum(n * c + n for c, n in zip(ctx, new))
    pages = sum(_pages(c + n, page) for c, n in zip(ctx, new))
    return {"bytes": keys * hk * d * 4 + sum(new) * (hq * d * 4 + 8) + pages * 4 + case["batch"] * 8,
            "flops": pairs * hq * d * 4}


def _held(case, ctx, new):
    """Pages each request holds before the step: those of its context, and for every seventh request the
    pages of a longer past (drafts that were not accepted, a request that has ended)."""
    held = [_pages(c, case["page"]) for c in ctx]
    for i in range(3, len(held), 7):
        held[i] += 1 + i % 5
    return held


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def _parents(new, seed):
    """Random drafted trees, each token's parent before it; -1 hangs a token on the context."""
    rng = np.random.default_rng(seed)
    return np.concatenate([np.array([int(rng.integers(-1, i)) if i else -1 for i in range(n)], np.int32)
                           for n in new] or [np.zeros(0, np.int32)])


def _mask_bits(parents, new):
    """Bit j of token i's word: i is j or descends from it (up to 64 tokens a tree)."""
    bits = np.zeros(len(parents), np.uint64)
    base = 0
    for n in new:
        for i in range(n):
            p = int(parents[base + i])
            bits[base + i] = np.uint64(1 << i) | (bits[base + p] if p >= 0 else np.uint64(0))
        base += n
    return bits.view(np.int64).reshape(-1, 1)


def _weights(case, gen):
    n, k, g = case["n"], case["k"], case["group"]
    w = {"q": torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device=DEV, generator=gen),
         "s": ((torch.rand((n, k // g), device=DEV, generator=gen) + 0.5) * (0.2 / math.sqrt(k))).to(_DT[case["dtype"]]),
         "z": None}
    if case["zeros"]:
        w["z"] = torch.randint(4, 12, (n, k // g), dtype=torch.uint8, device=DEV, generator=gen)
    return w


def _inputs(case, seed):
    gen = _gen(seed)
    op = case["op"]
    s = {"case": case}
    if op in ("linear", "gated"):
        s["w"] = [_weights(case, gen) for _ in range(2 if op == "gated" else 1)]
        s["x"] = torch.randn((case["tokens"], case["k"]), device=DEV, generator=gen).to(_DT[case["dtype"]])
        return s
    if op == "store":
        t, h, d, page = case["tokens"], case["kv_heads"], case["dim"], case["page"]
        dt = _DT[case["dtype"]]
        pages = _pages(t, page) + 4
        s["k"] = torch.randn((t, h, d), device=DEV, generator=gen).to(dt)
        s["v"] = torch.randn((t, h, d), device=DEV, generator=gen).to(dt)
        s["kc"] = torch.zeros((pages, page, h, d), dtype=dt, device=DEV)
        s["vc"] = torch.zeros((pages, page, h, d), dtype=dt, device=DEV)
        slots = torch.randperm(pages, device=DEV, generator=gen)[:, None] * page + torch.arange(page, device=DEV)
        slots = slots.reshape(-1)[:t].clone()
        slots[3::50] = -1                      # tokens without a slot (a refused request, padding)
        s["slots"] = slots
        return s
    ctx, new = _lens(case)
    page, batch = case["page"], case["batch"]
    if op == "tables":
        held = _held(case, ctx, new)
        width = max(max(held), max(_pages(c + n, page) for c, n in zip(ctx, new))) + 2
        spare = sum(_pages(n, page) + 1 for n in new) + 8
        ids = torch.randperm(sum(held) + spare, device=DEV, generator=gen).to(torch.int32)
        col = torch.arange(width, device=DEV)[None, :]
        h = _ints(held)
        first = torch.cumsum(h, 0) - h
        index = (first[:, None] + col).clamp(max=ids.numel() - 1)
        s["table"] = torch.where(col < h[:, None], ids[index], torch.full_like(index, -1, dtype=torch.int32))
        s["free"] = torch.full((ids.numel(),), -1, dtype=torch.int32, device=DEV)
        s["free"][:spare] = ids[sum(held):]
        s["count"] = _ints([spare])
        s["ctx"], s["new"], s["held"], s["total"] = _ints(ctx), _ints(new), h, sum(new)
        s["parents"] = _ints(_parents(new, seed).tolist()) if case["tree"] else None
        return s
    hq, hk, d, dt = case["q_heads"], case["kv_heads"], case["dim"], _DT[case["dtype"]]
    need = [_pages(c + n, page) for c, n in zip(ctx, new)]
    total = sum(need) + 3
    s["kc"] = torch.randn((total, page, hk, d), dtype=dt, device=DEV, generator=gen)
    s["vc"] = torch.randn((total, page, hk, d), dtype=dt, device=DEV, generator=gen)
    s["q"] = (1.5 * torch.randn((sum(new), hq, d), device=DEV, generator=gen)).to(dt)
    ids = torch.randperm(total, device=DEV, generator=gen).to(torch.int32)
    table = torch.zeros((batch, max(need)), dtype=torch.int32, device=DEV)
    at = 0
    for b, p in enumerate(need):
        table[b, :p] = ids[at:at + p]
        at += p
    s["table"] = table
    s["ctx_host"], s["new_host"] = ctx, new
    s["seq"] = _ints([c + n for c, n in zip(ctx, new)])
    s["cu"] = _ints([0] + np.cumsum(new).tolist())
    s["mask"] = None
    if case["tree"]:
        s["mask"] = torch.from_numpy(_mask_bits(_parents(new, seed), new)).to(DEV)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and case["op"] in ("linear", "gated"):
        from dsv41_flash_offload_b200 import w4
        s["packed"] = [w4.W4Weight(w["q"], w["s"], w["z"]) for w in s["w"]]
    return s


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from dsv41_flash_offload_b200 import paged, w4
    case = s["case"]
    op = case["op"]
    if op == "linear":
        return w4.linear(s["x"], s["packed"][0], out_dtype=_DT[case["out"]])
    if op == "gated":
        return w4.gated(s["x"], s["packed"][0], s["packed"][1], limit=10.0)
    if op == "tables":
        t = paged.step_tables(s["ctx"], s["new"], s["held"], s["table"], s["free"], s["count"], case["page"],
                              s["total"], parents=s["parents"])
        out = [s["table"], s["free"], t.cu_lens, t.seq_lens, t.slots, t.positions, t.requests, t.held_pages,
               t.free_count, t.status]
        return out + [t.tree_mask] if case["tree"] else out
    if op == "store":
        paged.store_kv(s["k"], s["v"], s["slots"], s["kc"], s["vc"])
        return [s["kc"], s["vc"]]
    return paged.tree_attention(s["q"], s["kc"], s["vc"], s["table"], s["seq"], s["cu"], case["new_max"],
                                tree_mask=s["mask"])


def _dense(w, group):
    n = w["q"].shape[0]
    q = torch.stack((w["q"] & 15, w["q"] >> 4), 2).view(n, -1, group).float()
    z = 8.0 if w["z"] is None else w["z"].float()[:, :, None]
    return ((q - z) * w["s"].float()[:, :, None]).view(n, -1)


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op == "linear":
        return (s["x"].float() @ _dense(s["w"][0], case["group"]).t()).to(_DT[case["out"]])
    if op == "gated":
        g = s["x"].float() @ _dense(s["w"][0], case["group"]).t()
        u = s["x"].float() @ _dense(s["w"][1], case["group"]).t()
        a = (g / (1.0 + torch.exp(-g))).clamp(max=10.0)
        return (a * u.clamp(-10.0, 10.0)).to(_DT[case["dtype"]])
    if op == "tables":
        return _tables_plain(s)
    if op == "store":
        keep = s["slots"] >= 0
        at = s["slots"][keep]
        for src, dst in ((s["k"], s["kc"]), (s["v"], s["vc"])):
            dst.view(-1, *src.shape[1:])[at] = src[keep]
        return [s["kc"], s["vc"]]
    return _tree_plain(s)


def _tables_plain(s):
    page, total, table, free, batch = s["case"]["page"], s["total"], s["table"], s["free"], s["case"]["batch"]
    width = table.shape[1]
    ctx, new, held = s["ctx"].long(), s["new"].long(), s["held"].long()
    count = s["count"].long()
    need = (ctx + new + page - 1) // page
    fits = need <= width
    want = torch.where(fits, need, held)
    give, take = (held - want).clamp(min=0), (want - held).clamp(min=0)
    given, taken = torch.cumsum(give, 0), torch.cumsum(take, 0)
    top = count + given[-1]                                        # stack height after the returns
    admitted = fits & ((take == 0) | (taken <= top))
    col = torch.arange(width, device=table.device)[None, :]
    # returned pages go on the stack in request order
    ids = torch.arange(free.numel(), device=free.device)
    slot = torch.searchsorted(given, (ids - count).clamp(min=0), right=True).clamp(max=batch - 1)
    page_at = (want[slot] + ids - count - (given - give)[slot]).clamp(0, width - 1)
    pushed = (ids >= count) & (ids < top)
    free.copy_(torch.where(pushed, table[slot, page_at], free))
    # taken pages come off its top in request order
    fresh = (col >= held[:, None]) & (col < want[:, None]) & admitted[:, None]
    pop = (top - 1 - (taken - take)[:, None] - (col - held[:, None])).clamp(0, free.numel() - 1)
    table.copy_(torch.where(fresh, free[pop], table))
    cu = torch.cumsum(new, 0)
    req = torch.searchsorted(cu, torch.arange(total, device=table.device), right=True)
    at = torch.arange(total, device=table.device) - (cu - new)[req]
    pos = ctx[req] + at
    slots = table[req, (pos // page).clamp(max=width - 1)].long() * page + pos % page
    slots = torch.where(admitted[req], slots, torch.full_like(slots, -1))
    status = (fits & ~admitted).int() + 2 * (~fits).int()          # of each request: 0, or why it was refused
    out_take = torch.where(admitted, take, torch.zeros_like(take)).sum()
    out = [table, free, torch.cat((torch.zeros_like(cu[:1]), cu)).int(),
           torch.where(admitted, ctx + new, torch.zeros_like(ctx)).int(), slots, pos.int(), req.int(),
           torch.where(admitted, want, held).int(), (top - out_take).int(), status]
    if s["parents"] is not None:
        # ancestors: step every token's pointer to its parent until all have left their tree
        first = (cu - new)[req]
        mask = torch.ones_like(slots) << at
        up = s["parents"].long()
        for _ in range(s["case"]["new_max"] - 1):
            live = up >= 0
            mask = mask | torch.where(live, torch.ones_like(mask) << up.clamp(min=0), torch.zeros_like(mask))
            up = torch.where(live, s["parents"].long()[first + up.clamp(min=0)], up)
        bits = (mask[:, None] >> torch.arange(64, device=mask.device)[None, :]) & 1
        out[5] = (ctx[req] + bits.sum(1) - 1).int()
        out.append(mask[:, None])
    return out


def _tree_plain(s):
    case = s["case"]
    hk, d, page = case["kv_heads"], case["dim"], case["page"]
    rep = case["q_heads"] // hk
    scale = 1.0 / math.sqrt(d)
    out = torch.empty_like(s["q"])
    at = 0
    for b, (c, n) in enumerate(zip(s["ctx_host"], s["new_host"])):
        pages = s["table"][b, :_pages(c + n, page)].long()
        visible = torch.ones((n, c + n), dtype=torch.bool, device=DEV)
        if s["mask"] is None:
            visible[:, c:] = torch.tril(visible[:, c:])
        else:
            visible[:, c:] = (s["mask"][at:at + n] >> torch.arange(n, device=DEV)[None, :]) & 1 != 0
        for h in range(hk):
            k = s["kc"][pages, :, h].reshape(-1, d)[:c + n].float()
            v = s["vc"][pages, :, h].reshape(-1, d)[:c + n].float()
            q = s["q"][at:at + n, h * rep:(h + 1) * rep].float().reshape(n * rep, d)
            score = (q @ k.t()).view(n, rep, -1) * scale
            score = torch.where(visible[:, None, :], score, torch.full_like(score, -math.inf))
            p = torch.exp(score - score.amax(2, keepdim=True))
            p = (p / p.sum(2, keepdim=True)).view(n * rep, -1)
            out[at:at + n, h * rep:(h + 1) * rep] = (p @ v).view(n, rep, d).to(out.dtype)
        at += n
    return out


# ------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op in ("linear", "gated"):
        prods = []
        for w in s["w"]:
            acc = torch.zeros((case["tokens"], case["n"]), dtype=torch.float64, device=DEV)
            x = s["x"].double()
            for j in range(case["k"] // case["group"]):            # group by group: s * (sum q x - z sum x)
                lo = j * case["group"]
                q = w["q"][:, lo // 2:(lo + case["group"]) // 2].to(torch.int64)
                even, odd = (q % 16).double(), (q // 16).double()
                xs = x[:, lo:lo + case["group"]]
                z = torch.full((case["n"],), 8.0, dtype=torch.float64, device=DEV) if w["z"] is None else w["z"][:, j].double()
                dot = xs[:, 0::2] @ even.t() + xs[:, 1::2] @ odd.t()
                acc += (dot - xs.sum(1)[:, None] * z[None, :]) * w["s"][:, j].double()[None, :]
            prods.append(acc)
        if op == "linear":
            return prods[0]
        g, u = prods
        silu = torch.minimum(g * torch.sigmoid(g), torch.full_like(g, 10.0))
        return silu * torch.maximum(torch.minimum(u, torch.full_like(u, 10.0)), torch.full_like(u, -10.0))
    if op == "tables":
        return None                                                # whole numbers throughout
    if op == "store":
        row = case["kv_heads"] * case["dim"]
        outs = []
        for src, dst in ((s["k"], s["kc"]), (s["v"], s["vc"])):
            buf = dst.double().view(-1, row)
            at = s["slots"].tolist()
            rows = [t for t, slot in enumerate(at) if slot >= 0]
            buf[[at[t] for t in rows]] = src.double().view(-1, row)[rows]
            outs.append(buf.view(dst.shape))
        return outs
    return _tree_exact(s)


def _tree_exact(s):
    case = s["case"]
    hk, hq, d, page = case["kv_heads"], case["q_heads"], case["dim"], case["page"]
    rep = hq // hk
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    flat_k, flat_v = s["kc"].view(-1, hk, d), s["vc"].view(-1, hk, d)
    mask = None if s["mask"] is None else s["mask"].view(-1).tolist()
    row = 0
    for b, (c, n) in enumerate(zip(s["ctx_host"], s["new_host"])):
        pos = torch.arange(c + n, device=DEV)
        slot = s["table"][b].long()[pos // page] * page + pos % page
        for i0 in range(0, n, 16):
            ni = min(16, n - i0)
            bias = torch.zeros((ni, c + n), dtype=torch.float64, device=DEV)
            for i in range(ni):
                for j in range(n):
                    word = mask[row + i0 + i] if mask is not None else (1 << (i0 + i + 1)) - 1
                    if not (word >> j) & 1:
                        bias[i, c + j] = -math.inf
            for h in range(hk):
                k, v = flat_k[slot, h].double(), flat_v[slot, h].double()
                q = s["q"][row + i0:row + i0 + ni, h * rep:(h + 1) * rep].double()
                score = torch.einsum("nrd,kd->rnk", q, k) / math.sqrt(d) + bias
                weight = torch.softmax(score, 2)
                out[row + i0:row + i0 + ni, h * rep:(h + 1) * rep] = torch.einsum("rnk,kd->nrd", weight, v)
        row += n
    return out

