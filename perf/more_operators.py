"""What long contexts and scored answers cost, case by case.

Requests with long contexts are served from a cache in 4 bits (the store of new keys and values, their reading back,
the attention of drafted tokens over it) or through a window with a few first tokens that stay visible; what a
step answers with is scored: log probabilities of given tokens, entropy and the likeliest alternatives of every row of
logits. `listed()` holds the sizes such a program meets, `draw()` makes more of the same ranges, `run()` is one pass
through an operator: in plain torch where `own` is false, through the framework's entry points (`paged`, `logprobs`)
where it is true. `exact()` gives the same outputs from the operators' definitions in 64 bits.

4 bits: a token's head is cut into groups of 32 columns. With lo and hi the smallest and largest value of a group,
s = (hi - lo) / 15 in the cache's type and code = round((x - lo) / s) in 0..15, a code stands for lo + s * code in the
cache's type.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
GROUP = 32
_DT = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def listed():
    return [
        # keys and values of a decode step's drafted tokens into a cache in 4 bits, and back: latency only
        _store("store4-draft", tokens=100, kv_heads=8, dim=128, page=16, dtype="bfloat16"),
        # a prompt chunk, some tokens without a slot
        _store("store4-prefill", tokens=16384, kv_heads=8, dim=128, page=64, dtype="float16"),
        # one request, one token: the latency of the smallest attention over 4 bits
        _attn("attn4-one", batch=1, new=(1, 1), ctx=(2047, 2047), q_heads=32, kv_heads=8, dim=128, page=16,
              tree=False, window=0, sinks=0, bits=4, dtype="bfloat16"),
        # few requests with very long contexts, one token each: the bandwidth of the cache
        _attn("attn4-long", batch=4, new=(1, 1), ctx=(65536, 131056), q_heads=64, kv_heads=8, dim=128, page=64,
              tree=False, window=0, sinks=0, bits=4, dtype="bfloat16"),
        # a decode batch with small drafted trees of uneven sizes over uneven contexts
        _attn("attn4-draft", batch=16, new=(5, 13), ctx=(100, 16000), q_heads=32, kv_heads=8, dim=128, page=16,
              tree=True, window=0, sinks=0, bits=4, dtype="float16"),
        # wide trees: many rows for each key
        _attn("attn4-wide", batch=32, new=(61, 64), ctx=(1000, 8192), q_heads=32, kv_heads=8, dim=128, page=32,
              tree=True, window=0, sinks=0, bits=4, dtype="bfloat16"),
        # a drafted step through a window over long contexts, odd window and pages
        _attn("window-draft", batch=32, new=(1, 9), ctx=(500, 32000), q_heads=32, kv_heads=4, dim=128, page=24,
              tree=True, window=1000, sinks=4, bits=16, dtype="bfloat16"),
        # long prompt chunks through a window
        _attn("window-prefill", batch=2, new=(6000, 8192), ctx=(0, 4000), q_heads=32, kv_heads=8, dim=128, page=64,
              tree=False, window=2048, sinks=16, bits=16, dtype="float16"),
        # one row of the head's logits: the latency of the smallest call
        _score("score-one", rows=1, vocab=100001, given=1, top=5, masked=False, dtype="float32"),
        # the rows of a drafted step, each with its drafted children, a grammar masking some of the rows
        _score("score-draft", rows=100, vocab=32768, given=4, top=20, masked=True, dtype="bfloat16"),
        # the tokens of a prompt, no alternatives: the bandwidth of the logits
        _score("score-prompt", rows=2048, vocab=100001, given=1, top=0, masked=False, dtype="float32"),
        # a batch of answers with many alternatives out of 16-bit logits (ties are common)
        _score("score-batch", rows=512, vocab=128000, given=1, top=32, masked=False, dtype="bfloat16"),
    ]


def _store(name, **kw):
    return dict(kw, name=name, op="store")


def _score(name, **kw):
    return dict(kw, name=name, op="score")


def _attn(name, **kw):
    for key in ("new", "ctx"):
        lo, hi = kw.pop(key)
        kw[key + "_min"], kw[key + "_max"] = lo, hi
    return dict(kw, name=name, op="attn")


def _log_int(rng, lo, hi):
    """A whole number of lo..hi, spread evenly over its logarithm."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    while True:
        case = _draw(rng)
        w = work(case)
        if w["bytes"] <= 8e8 and w["flops"] <= 3e11:
            case.pop("name")
            return case


def _draw(rng):
    op = rng.choice(("store", "attn", "attn", "attn", "score", "score"))
    dtype = rng.choice(("float16", "bfloat16"))
    if op == "store":
        return _store("", tokens=_log_int(rng, 1, 16384), kv_heads=rng.choice((1, 2, 3, 4, 8)),
                      dim=rng.choice((32, 64, 96, 128, 192, 256)), page=rng.choice((8, 16, 24, 32, 64)), dtype=dtype)
    if op == "score":
        return _score("", rows=_log_int(rng, 1, 2048), vocab=_log_int(rng, 1000, 160000), given=rng.choice((1, 1, 2, 5)),
                      top=rng.choice((0, 1, 5, 20, 32)), masked=rng.random() < 0.4, dtype=rng.choice(("float32", dtype)))
    kv = rng.choice((1, 2, 3, 4, 8))
    bits = rng.choice((4, 4, 16))
    windowed = bits == 16 or rng.random() < 0.3
    common = dict(q_heads=kv * rng.choice((1, 2, 3, 4, 5, 8, 16)), kv_heads=kv,
                  dim=rng.choice((32, 64, 96, 128, 128, 256) if bits == 4 else (64, 80, 96, 128, 128, 256)),
                  page=rng.choice((8, 16, 24, 32, 64, 128) if bits == 4 else (1, 8, 16, 24, 32, 64, 128)), bits=bits, dtype=dtype,
                  window=_log_int(rng, 1, 8192) if windowed else 0, sinks=rng.choice((0, 1, 4, 16, 130)) if windowed else 0)
    if windowed and rng.random() < 0.3:          # prompt chunks
        new = _log_int(rng, 65, 8192)
        ctx = _log_int(rng, 1, 8192)
        return _attn("", batch=rng.randint(1, 4), new=(rng.randint(1, new), new), ctx=(0, ctx), tree=False, **common)
    new = _log_int(rng, 1, 64)
    ctx = _log_int(rng, 1, 65536)
    return _attn("", batch=_log_int(rng, 1, 64), new=(rng.randint(1, new), new), ctx=(rng.randint(0, ctx), ctx),
                 tree=rng.random() < 0.7, **common)


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


def _sums(lo, hi):
    """Sum of the whole numbers lo..hi."""
    return (lo + hi) * (hi - lo + 1) // 2 if hi >= lo else 0


def work(case):
    op = case["op"]
    if op == "store":
        head = case["dim"] * 2
        packed = case["dim"] // 2 + case["dim"] // GROUP * 4
        return {"bytes": case["tokens"] * case["kv_heads"] * 2 * (2 * head + 2 * packed) + case["tokens"] * 16, "flops": 0}
    if op == "score":
        size = 4 if case["dtype"] == "float32" else 2
        return {"bytes": case["rows"] * (case["vocab"] * size + case["given"] * 12 + case["top"] * 12 + 8), "flops": 0}
    ctx, new = _lens(case)
    hq, hk, d, win, sinks = case["q_heads"], case["kv_heads"], case["dim"], case["window"], case["sinks"]
    keys = pairs = 0
    for c, n in zip(ctx, new):
        if not win:
            keys += c + n
            pairs += n * c + (n if case["tree"] else _sums(1, n))
            continue
        first = max(0, c - win + 1)                                  # what the first token's window reaches
        keys += c + n - first + min(sinks, first)
        full = max(0, min(n, win - c))                               # tokens that see everything (a tree: about)
        pairs += (_sums(c + 1, c + full)) + (n - full) * win + sum(min(sinks, c + i + 1 - win) for i in range(full, n))
    row = d * 4 if case["bits"] == 16 else 2 * (d // 2 + d // GROUP * 4)
    pages = sum(_pages(c + n, case["page"]) for c, n in zip(ctx, new))
    return {"bytes": keys * hk * row + sum(new) * (hq * d * 4 + 8) + min(pages, keys) * 4 + case["batch"] * 8,
            "flops": pairs * hq * d * 4}


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def _parents(new, seed):
    """Random drafted trees, each token's parent before it; -1 hangs a token on the context."""
    rng = np.random.default_rng(seed)
    return [[int(rng.integers(-1, i)) if i else -1 for i in range(n)] for n in new]


def _mask_bits(parents):
    """Bit j of token i's word: i is j or descends from it (up to 64 tokens a tree)."""
    bits = []
    for tree in parents:
        own_bits = []
        for i, p in enumerate(tree):
            own_bits.append((1 << i) | (own_bits[p] if p >= 0 else 0))
        bits += own_bits
    return np.array(bits, np.uint64).view(np.int64).reshape(-1, 1)


def _inputs(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    op, dt = case["op"], _DT[case["dtype"]]
    randn = lambda *shape: torch.randn(shape, device=DEV, generator=gen)
    s = {"case": case}
    if op == "score":
        n, v = case["rows"], case["vocab"]
        logits = (2.5 * randn(n, v)).to(dt)
        s["tokens"] = torch.randint(0, v, (n, case["given"]), device=DEV, generator=gen)
        if case["masked"]:                       # every third row may only answer with some of the tokens
            keep = torch.rand((n, v), device=DEV, generator=gen) < 0.1
            keep.scatter_(1, s["tokens"][:, :1], True)
            keep[torch.arange(n, device=DEV) % 3 != 0] = True
            logits.masked_fill_(~keep, -math.inf)
        s["logits"] = logits
        if case["given"] == 1:
            s["tokens"] = s["tokens"].view(n)
        return s
    h, d, page = case["kv_heads"], case["dim"], case["page"]
    if op == "store":
        t = case["tokens"]
        s["pages"] = _pages(t, page) + 4
        s["k"], s["v"] = (1.3 * randn(t, h, d)).to(dt), randn(t, h, d).to(dt)
        slots = torch.randperm(s["pages"], device=DEV, generator=gen)[:, None] * page + torch.arange(page, device=DEV)
        slots = slots.reshape(-1)[:t].clone()
        slots[3::50] = -1                        # tokens without a slot (a refused request, padding)
        s["slots"] = slots
        return s
    ctx, new = _lens(case)
    hq, batch = case["q_heads"], case["batch"]
    need = [_pages(c + n, page) for c, n in zip(ctx, new)]
    total = sum(need) + 3
    s["kc"], s["vc"] = (torch.randn((total, page, h, d), dtype=dt, device=DEV, generator=gen) for _ in range(2))
    s["q"] = (1.5 * randn(sum(new), hq, d)).to(dt)
    ids = torch.randperm(total, device=DEV, generator=gen).to(torch.int32)
    table = torch.zeros((batch, max(need)), dtype=torch.int32, device=DEV)
    at = 0
    for b, p in enumerate(need):
        table[b, :p] = ids[at:at + p]
        at += p
    s["table"], s["ctx_host"], s["new_host"] = table, ctx, new
    s["seq"] = _ints([c + n for c, n in zip(ctx, new)])
    s["cu"] = _ints([0] + np.cumsum(new).tolist())
    s["mask"] = torch.from_numpy(_mask_bits(_parents(new, seed))).to(DEV) if case["tree"] else None
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "score" or case.get("bits") == 16:
        return s
    dt = _DT[case["dtype"]]
    pages = s["pages"] if case["op"] == "store" else s["kc"].shape[0]
    if own:
        from dsv41_flash_offload_b200 import paged
        s["cache"] = paged.Cache4(pages, case["page"], case["kv_heads"], case["dim"], dtype=dt, device=DEV)
    elif case["op"] == "store":
        shape = (2, pages * case["page"], case["kv_heads"], case["dim"] // GROUP)
        s["packed"] = (torch.zeros((*shape, GROUP // 2), dtype=torch.uint8, device=DEV),
                       *(torch.zeros(shape, dtype=dt, device=DEV) for _ in range(2)))
    if case["op"] == "attn":                     # the cache in hand: what earlier steps have stored
        kc, vc = (s.pop(n).flatten(0, 1) for n in ("kc", "vc"))
        if own:
            paged.store_kv4(kc, vc, torch.arange(kc.shape[0], device=DEV), s["cache"])
        else:
            s["packed"] = [_quantize(x) for x in (kc, vc)]
    return s


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from dsv41_flash_offload_b200 import logprobs, paged
    case = s["case"]
    if case["op"] == "store":
        paged.store_kv4(s["k"], s["v"], s["slots"], s["cache"])
        return list(paged.load_kv4(s["slots"], s["cache"]))
    if case["op"] == "score":
        r = logprobs.token_logprobs(s["logits"], s["tokens"], top=case["top"])
        return [r.logprobs, r.entropy] + ([r.top_ids, r.top_logprobs] if case["top"] else [])
    if case["bits"] == 4:
        return paged.tree_attention4(s["q"], s["cache"], s["table"], s["seq"], s["cu"], case["new_max"], tree_mask=s["mask"],
                                     window=case["window"] or None, sinks=case["sinks"])
    return paged.tree_attention(s["q"], s["kc"], s["vc"], s["table"], s["seq"], s["cu"], case["new_max"],
                                tree_mask=s["mask"], window=case["window"] or None, sinks=case["sinks"])


def _run_plain(s):
    op = s["case"]["op"]
    return _store_plain(s) if op == "store" else _score_plain(s) if op == "score" else _attn_plain(s)


def _quantize(x):
    """[N, heads, dim] -> codes (two a byte), scales and smallest values of each group of 32 columns."""
    g = x.unflatten(2, (-1, GROUP)).float()
    lo, hi = g.amin(3), g.amax(3)
    scale = ((hi - lo) / 15.0).to(x.dtype)
    top = torch.finfo(x.dtype).max
    over = (lo.double() + 15.0 * scale.double()).to(x.dtype).double().abs() > top   # the last code would pass the type
    scale = torch.where(over, (scale.view(torch.int16) - 1).view(x.dtype), scale)
    step = scale.double()[..., None]
    code = torch.where(step > 0, torch.round((g.double() - lo.double()[..., None]) / step), torch.zeros_like(step))   # in 64 bits: halves
    code = code.clamp(0, 15).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale, lo.to(x.dtype)


def _values(code, scale, lo):
    """What codes stand for: [N, heads, dim] in the cache's type."""
    q = torch.stack((code & 15, code >> 4), -1).flatten(-2).float()
    return (lo.float()[..., None] + scale.float()[..., None] * q).to(lo.dtype).flatten(-2)


def _store_plain(s):
    keep = s["slots"] >= 0
    at = s["slots"][keep]
    out = []
    for i, x in enumerate((s["k"], s["v"])):
        for dst, src in zip(s["packed"], _quantize(x[keep])):
            dst[i][at] = src
        back = torch.zeros_like(x)
        back[keep] = _values(*(p[i][at] for p in s["packed"]))
        out.append(back)
    return out


def _score_plain(s):
    case, x, tokens = s["case"], s["logits"].float() + 0.0, s["tokens"]      # (-0 and 0 tie)
    top = x.amax(1, keepdim=True)
    z = x - top
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    lse = torch.log(total)
    given = torch.gather(z, 1, tokens.view(case["rows"], -1)) - lse
    terms = torch.where(e > 0, e * z, torch.zeros_like(z))
    out = [given.view(tokens.shape), lse[:, 0] - terms.sum(1) / total[:, 0]]
    if case["top"]:
        bits = x.view(torch.int32).long()                           # in the numbers' order, ties by the lowest index
        order = torch.where(bits < 0, -1 - (bits & 0x7fffffff), bits)
        key = order * 2 ** 32 + (case["vocab"] - 1 - torch.arange(case["vocab"], device=DEV))
        best = torch.topk(key, case["top"], dim=1).values
        ids = case["vocab"] - 1 - (best & 0xffffffff)
        out += [ids, torch.gather(z, 1, ids) - lse]
    return out


def _attn_plain(s):
    case = s["case"]
    hk, d, page, win, sinks = case["kv_heads"], case["dim"], case["page"], case["window"], case["sinks"]
    rep = case["q_heads"] // hk
    scale = 1.0 / math.sqrt(d)
    out = torch.empty_like(s["q"])
    at = 0
    for b, (c, n) in enumerate(zip(s["ctx_host"], s["new_host"])):
        pos = torch.arange(c + n, device=DEV)
        slot = s["table"][b].long()[pos // page] * page + pos % page
        for i0 in range(0, n, 2048):                                # tokens of a chunk against the keys up to it
            ni = min(2048, n - i0)
            end = c + n if case["tree"] else c + i0 + ni
            token = torch.arange(i0, i0 + ni, device=DEV)[:, None]
            if s["mask"] is None:
                visible = pos[None, :end] <= c + token
                back = c + token - pos[None, :end]                  # visible keys after this one
            else:
                bits = (s["mask"][at + i0:at + i0 + ni] >> torch.arange(n, device=DEV)[None, :]) & 1
                depth = bits.sum(1, keepdim=True)
                later = torch.cat((c - 1 - pos[None, :c] + depth, depth - torch.cumsum(bits, 1)), 1)
                visible = torch.cat((torch.ones((ni, c), dtype=torch.bool, device=DEV), bits != 0), 1)
                back = later
            if win:
                visible = visible & ((back < win) | (pos[None, :end] < sinks))
            # a chunk's window leaves most of a long context out
            some = torch.nonzero(visible.any(0))[:, 0] if win else pos[:end]
            seen = visible[:, some][:, None, :]
            for h in range(hk):
                if case["bits"] == 16:
                    k, v = (s[name].flatten(0, 1)[slot[some], h].float() for name in ("kc", "vc"))
                else:
                    k, v = (_values(*(t[slot[some], h] for t in packed)).float() for packed in s["packed"])
                q = s["q"][at + i0:at + i0 + ni, h * rep:(h + 1) * rep].float().reshape(ni * rep, d)
                score = (q @ k.t()).view(ni, rep, -1) * scale
                score = torch.where(seen, score, torch.full_like(score, -math.inf))
                p = torch.exp(score - score.amax(2, keepdim=True))
                p = (p / p.sum(2, keepdim=True)).view(ni * rep, -1)
                out[at + i0:at + i0 + ni, h * rep:(h + 1) * rep] = (p @ v).view(ni, rep, d).to(out.dtype)
        at += n
    return out


# ------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def _stored(x):
    """What a cache in 4 bits holds of x [..., dim], as 64-bit numbers."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for c in range(0, x.shape[-1], GROUP):
        g = x[..., c:c + GROUP].double()
        lo, span = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values - g.min(-1, keepdim=True).values
        s = (span / 15).to(x.dtype).double()
        if torch.any((lo + 15 * s).to(x.dtype).isinf()):
            return None                                             # (no input here reaches the end of the type)
        q = torch.round((g - lo) / torch.where(s == 0, torch.ones_like(s), s)).clamp(max=15) * (s != 0)
        out[..., c:c + GROUP] = (lo + s * q).to(x.dtype).double()
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "store":
        outs = []
        for x in (s["k"], s["v"]):
            y = _stored(x)
            y[s["slots"] < 0] = 0
            outs.append(y)
        return outs
    if case["op"] == "score":
        given, entropy, tops = [], [], []
        tokens = s["tokens"].view(case["rows"], -1)
        for r0 in range(0, case["rows"], 64):
            logp = torch.log_softmax(s["logits"][r0:r0 + 64].double(), 1)
            given.append(logp.gather(1, tokens[r0:r0 + 64]))
            entropy.append(-torch.xlogy(logp.exp(), logp.exp()).sum(1))
            if case["top"]:
                tops.append(logp.sort(1, descending=True).values[:, :case["top"]])
        out = [torch.cat(given).view(s["tokens"].shape), torch.cat(entropy)]
        return out + [None, torch.cat(tops)] if case["top"] else out
    return _attn_exact(s)


def _attn_exact(s):
    case = s["case"]
    hk, hq, d, page, win, sinks = (case[n] for n in ("kv_heads", "q_heads", "dim", "page", "window", "sinks"))
    rep = hq // hk
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    flat = [s[name].view(-1, hk, d) for name in ("kc", "vc")]
    row = 0
    for b, (c, n) in enumerate(zip(s["ctx_host"], s["new_host"])):
        at = torch.arange(c + n, device=DEV)
        slot = s["table"][b].long()[at // page] * page + at % page
        for i0 in range(0, n, 512):
            ni = min(512, n - i0)
            end = c + n if case["tree"] else c + i0 + ni
            if case["tree"]:
                ancestors = torch.zeros((ni, n), dtype=torch.bool, device=DEV)
                for j in range(n):
                    ancestors[:, j] = (s["mask"][row + i0:row + i0 + ni, 0] & (1 << j if j < 63 else -(1 << 63))) != 0
            else:
                ancestors = torch.ones((ni, n), dtype=torch.bool, device=DEV).tril(i0)[:, :end - c]
            see = torch.cat((torch.ones((ni, c), dtype=torch.bool, device=DEV), ancestors), 1)
            if win:                                                 # the last `win` that it sees, and the first `sinks` positions
                rank = see.int().flip(1).cumsum(1).flip(1)
                see = see & ((rank <= win) | (at[:end] < sinks))
            used = see.any(0).nonzero()[:, 0]
            bias = torch.where(see[:, used], 0.0, -math.inf).double()
            for h in range(hk):
                k, v = (x[slot[used], h] for x in flat)
                k, v = (k.double(), v.double()) if case["bits"] == 16 else (_stored(k), _stored(v))
                q = s["q"][row + i0:row + i0 + ni, h * rep:(h + 1) * rep].double()
                weight = torch.softmax(torch.einsum("nrd,kd->nrk", q, k) / math.sqrt(d) + bias[:, None], 2)
                out[row + i0:row + i0 + ni, h * rep:(h + 1) * rep] = torch.einsum("nrk,kd->nrd", weight, v)
        row += n
    return out
