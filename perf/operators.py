"""Operators of decoding over a long paged cache, case by case: rotary positions with the store into the cache, block attention of
a batch that shares a prefix, the weights its keys have received, and the eviction that goes by them.

``run`` makes one call: in plain torch operations, or the framework's.  Caches are [pages, 256, kv heads, channels], the
page lists are shuffled, and requests of one batch have different lengths.
"""
import importlib
import math
import random

import torch

own = False

PAGE, HEAD, BF, F32, F64 = 256, 128, torch.bfloat16, torch.float32, torch.float64
DEV = "cuda"
TYPES = {"bf16": BF, "fp32": F32}
BASE = 1000000.0        # of the rotary frequencies


def listed():
    return [
        # a block of masked tokens of one request: queries rotated, keys and values into the cache; one such call per layer and step
        {"name": "rotary_block_32", "kind": "rotary", "n": 32, "hq": 16, "hkv": 8, "dim": 128, "rot": 128, "layout": "half",
         "type": "bf16", "store": True, "first": 8000},
        # a prompt of 16384 tokens, a quarter of every head rotated, pairs of neighbours, positions up to 131072
        {"name": "rotary_prompt_16384", "kind": "rotary", "n": 16384, "hq": 32, "hkv": 8, "dim": 128, "rot": 32, "layout": "pairs",
         "type": "bf16", "store": False, "first": 114688},
        # a ragged prompt in fp32, heads of 64, all channels
        {"name": "rotary_fp32_1057", "kind": "rotary", "n": 1057, "hq": 16, "hkv": 4, "dim": 64, "rot": 64, "layout": "half",
         "type": "fp32", "store": True, "first": 0},
        # four questions on one page image (1024 visual rows and 32 ids): the smallest batch worth sharing for
        {"name": "shared_4x32_1056", "kind": "shared", "bs": 4, "block": 32, "prefix": 1056, "ctx": 300, "hq": 16, "hkv": 8},
        # 32 denoising blocks behind one document
        {"name": "shared_32x32_8192", "kind": "shared", "bs": 32, "block": 32, "prefix": 8192, "ctx": 1024, "hq": 16, "hkv": 8},
        # single tokens of 64 samples of one long document
        {"name": "shared_64x1_16384", "kind": "shared", "bs": 64, "block": 1, "prefix": 16384, "ctx": 2048, "hq": 32, "hkv": 8},
        # the largest: 64 denoising blocks behind a long document
        {"name": "shared_64x32_16384", "kind": "shared", "bs": 64, "block": 32, "prefix": 16384, "ctx": 2048, "hq": 16, "hkv": 8},
        # what the keys of one request received from its block
        {"name": "weights_1x32_2000", "kind": "weights", "bs": 1, "block": 32, "ctx": 2000, "hq": 16, "hkv": 8},
        # ... of 32 requests with long contexts
        {"name": "weights_32x32_8192", "kind": "weights", "bs": 32, "block": 32, "ctx": 8192, "hq": 16, "hkv": 8},
        # ... from single tokens with eight query heads to a key head
        {"name": "weights_16x1_32768", "kind": "weights", "bs": 16, "block": 1, "ctx": 32768, "hq": 32, "hkv": 4},
        # one request gives half of its cache back
        {"name": "evict_1_4100", "kind": "evict", "bs": 1, "len": 4100, "budget": 2048, "recent": 128, "hkv": 8},
        # sixteen long requests keep a quarter
        {"name": "evict_16_32768", "kind": "evict", "bs": 16, "len": 32768, "budget": 8192, "recent": 512, "hkv": 8},
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["rotary", "shared", "shared", "weights", "evict"])
    c = {"kind": kind}
    if kind == "rotary":
        c["dim"] = rng.choice([64, 96, 128, 128])
        c.update(n=log(1, 16384), rot=rng.choice([16, 32, c["dim"] // 2, c["dim"]]), layout=rng.choice(["half", "pairs"]),
                 type=rng.choice(["bf16", "bf16", "fp32"]), store=rng.choice([False, True]), first=rng.randint(0, 114688))
        c["hq"], c["hkv"] = rng.choice([(16, 8), (32, 8), (8, 4), (16, 2)] if c["type"] == "bf16" else [(16, 4), (8, 4)])
        return c
    if kind == "evict":
        c.update(bs=log(1, 16), len=log(300, 32768), hkv=rng.choice([2, 4, 8]))
        c["budget"] = rng.randint(max(1, c["len"] // 8), c["len"] // 4)
        c["recent"] = rng.randint(0, c["budget"] // 2)
        return c
    c["hq"], c["hkv"] = rng.choice([(16, 8), (16, 8), (32, 8), (8, 4), (16, 16), (32, 4)])
    c["block"] = rng.choice([1, 8, 16, 32, 32, 64])
    if kind == "shared":
        c.update(bs=log(1, 64), prefix=log(100, 16384), ctx=log(1, 2048))
        c["bs"] = max(1, min(c["bs"], 2048 * 16 // (c["block"] * c["hq"])))
    else:
        c.update(bs=log(1, 32), ctx=log(1, 8192))
        c["bs"] = max(1, min(c["bs"], 1024 * 16 // (c["block"] * c["hq"])))
    return c


# ----------------------------------------------------------------------------- sizes that follow from a case
def lengths(case):
    """Keys of every request's own pages: the longest first, the others between half of it and it."""
    r = random.Random(str(sorted((k, v) for k, v in case.items() if k != "name")))
    n = case["len"] if case["kind"] == "evict" else case["ctx"]
    return [n] + [r.randint(n // 2, n) for _ in range(case["bs"] - 1)]


def work(case):
    kind = case["kind"]
    if kind == "rotary":
        e = 2 if case["type"] == "bf16" else 4
        heads = case["hq"] + case["hkv"] * (2 if case["store"] else 1)
        return {"bytes": 2 * case["n"] * heads * case["dim"] * e + case["n"] * (12 if case["store"] else 8),
                "flops": 3 * case["n"] * (case["hq"] + case["hkv"]) * case["rot"]}
    lens, hkv = lengths(case), case["hkv"]
    if kind == "evict":
        kept = sum(min(n, case["budget"]) for n in lens)
        return {"bytes": hkv * (4 * sum(lens) + kept * (2 * 2 * 2 * HEAD + 4 + 4)), "flops": hkv * sum(lens)}
    rows, hq = case["bs"] * case["block"], case["hq"]
    if kind == "shared":
        keys = case["prefix"] + sum(lens)
        return {"bytes": keys * hkv * HEAD * 4 + rows * hq * (HEAD * 4 + 4),
                "flops": 4 * HEAD * case["block"] * hq * (case["bs"] * case["prefix"] + sum(lens))}
    return {"bytes": sum(lens) * hkv * (HEAD * 2 + 8) + rows * hq * (HEAD * 2 + 4), "flops": 2 * HEAD * case["block"] * hq * sum(lens)}


# ----------------------------------------------------------------------------- inputs
def frequencies(rot):
    """64-bit frequencies, the slow ones drawn out by 4 for contexts beyond the trained 32768 (between 32 turns and one over
    them the two are blended), and the factor on queries and keys that goes with it."""
    i = torch.arange(rot // 2, dtype=F64, device=DEV)
    f = BASE ** (-2.0 * i / rot)
    turns = 32768 * f / (2 * math.pi)
    keep = (turns.log() / math.log(32.0)).clamp(0.0, 1.0)
    return f * keep + f / 4.0 * (1.0 - keep), 0.1 * math.log(4.0) + 1.0


def pages_for(lens, g, behind=0):
    """Shuffled page list of requests of these lengths: (int32 table, pages in all)."""
    need = torch.tensor([max(1, -(-n // PAGE)) for n in lens], device=DEV)[:, None]
    pages, column = int(need.sum()), torch.arange(int(need.max()), device=DEV)
    perm = torch.randperm(pages, generator=g, device=DEV).to(torch.int32) + behind
    at = (need.cumsum(0) - need + column).clamp(max=pages - 1)
    return torch.where(column < need, perm[at], -1), pages


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def randn(*shape, dtype=BF, scale=1.0):
        return (torch.randn(*shape, generator=g, device=DEV, dtype=F32) * scale).to(dtype)

    def int32(v):
        return torch.tensor(v, dtype=torch.int32, device=DEV)

    kind = case["kind"]
    if kind == "rotary":
        n, hq, hkv, d, t = case["n"], case["hq"], case["hkv"], case["dim"], TYPES[case["type"]]
        # views of one projection's output, as a decoder has them
        qkv = randn(n, (hq + 2 * hkv) * d, dtype=t)
        q, k, v = (x.unflatten(1, (-1, d)) for x in qkv.split([hq * d, hkv * d, hkv * d], dim=1))
        s = {"q": q, "k": k, "v": v, "rot": case["rot"], "pairs": case["layout"] == "pairs"}
        s["inv_freq"], s["factor"] = frequencies(case["rot"])
        s["positions"] = case["first"] + torch.arange(n, device=DEV) + seed % 97
        if case["store"]:
            pages = -(-n // PAGE) + 1
            s["k_cache"], s["v_cache"] = (torch.zeros(pages, PAGE, hkv, d, dtype=t, device=DEV) for _ in range(2))
            s["slots"] = torch.randperm(pages * PAGE, generator=g, device=DEV)[:n].to(torch.int32)
        return {"kind": kind, **s}
    lens, bs, hkv = lengths(case), case["bs"], case["hkv"]
    if kind == "evict":
        table, pages = pages_for(lens, g)
        to, more = pages_for([min(n, case["budget"]) for n in lens], g, behind=pages)
        k_cache, v_cache = (torch.empty(pages + more, PAGE, hkv, HEAD, dtype=BF, device=DEV) for _ in range(2))
        for c in (k_cache, v_cache):
            c.normal_(generator=g)
            c[pages:] = 0
        # heavy-tailed sums; some keys have received nothing yet
        w = (torch.randn(bs, hkv, max(lens), generator=g, device=DEV) * 2.0).exp()
        w[torch.rand(w.shape, generator=g, device=DEV) < 0.05] = 0.0
        return {"kind": kind, "k_cache": k_cache, "v_cache": v_cache, "weights": w, "table": table, "to": to, "seqlens": int32(lens),
                "budget": case["budget"], "recent": case["recent"], "first_out": pages}
    block, hq = case["block"], case["hq"]
    prefix = case.get("prefix", 0)
    table, pages = pages_for(lens, g)
    prefix_table, more = pages_for([prefix], g, behind=pages)
    # keys share a mean, as trained ones do; values have a small one
    k_cache = torch.empty(pages + more, PAGE, hkv, HEAD, dtype=BF, device=DEV).normal_(generator=g)
    k_cache += randn(hkv, HEAD, scale=0.5)
    v_cache = torch.empty(pages + more, PAGE, hkv, HEAD, dtype=BF, device=DEV).normal_(generator=g)
    v_cache += randn(hkv, HEAD, scale=0.2)
    s = {"kind": kind, "q": randn(bs, block, hq, HEAD, scale=1.3), "k_cache": k_cache, "v_cache": v_cache, "table": table,
         "seqlens": int32(lens), "longest": max(lens), "scale": HEAD ** -0.5}
    if kind == "shared":
        s.update(prefix_table=prefix_table[0], prefix_len=int32([prefix]), prefix=prefix)
    else:
        s["lse"] = log_sums(s, F32)
        s["previous"] = (torch.randn(bs, hkv, max(lens), generator=g, device=DEV) - 1.0).exp()
        s["decay"] = 0.9
    return s


# ----------------------------------------------------------------------------- plain forms
def own_keys(cache, table, longest, dtype):
    """[bs, kv heads, longest, channels] of every request's own pages (whatever lies there behind its end)."""
    bs = table.shape[0]
    return cache[table.clamp(min=0).long()].flatten(1, 2)[:, :longest].transpose(1, 2).to(dtype).reshape(bs, cache.shape[2], longest, -1)


def stacked(q, hkv, dtype):
    """[bs, kv heads, block * group, channels]: the rows that share a key head."""
    bs, block, hq, d = q.shape
    return q.to(dtype).view(bs, block, hkv, hq // hkv, d).transpose(1, 2).reshape(bs, hkv, -1, d)


def unstacked(x, block):
    """[bs, block, query heads, ...] of stacked rows."""
    bs, hkv, rows = x.shape[:3]
    return x.view(bs, hkv, block, rows // block, *x.shape[3:]).transpose(1, 2).flatten(2, 3)


def own_scores(s, dtype):
    q, k = stacked(s["q"], s["k_cache"].shape[2], dtype), own_keys(s["k_cache"], s["table"], s["longest"], dtype)
    there = torch.arange(s["longest"], device=DEV) < s["seqlens"][:, None]
    return (q @ k.transpose(2, 3) * s["scale"]).masked_fill(~there[:, None, None], -math.inf), there


def log_sums(s, dtype):
    scores, _ = own_scores(s, dtype)
    top = scores.amax(-1, keepdim=True).clamp(min=-1e30)
    return unstacked(((scores - top).exp().sum(-1).log() + top[..., 0]), s["q"].shape[1]).contiguous()


def plain_rotary(s):
    r, pairs = s["rot"], s["pairs"]
    angle = s["positions"].to(F64)[:, None] * s["inv_freq"]
    cos, sin = ((f * s["factor"]).to(F32)[:, None] for f in (angle.cos(), angle.sin()))

    def turn(x):
        y = x.float()
        a, b = (y[..., 0:r:2], y[..., 1:r:2]) if pairs else (y[..., : r // 2], y[..., r // 2: r])
        c, d = a * cos - b * sin, b * cos + a * sin
        y = torch.cat([torch.stack([c, d], -1).flatten(-2) if pairs else torch.cat([c, d], -1), y[..., r:]], -1)
        return y.to(x.dtype)

    q, k = turn(s["q"]), turn(s["k"])
    if "slots" not in s:
        return q, k
    s["k_cache"].flatten(0, 1)[s["slots"].long()] = k
    s["v_cache"].flatten(0, 1)[s["slots"].long()] = s["v"]
    return q, s["k_cache"], s["v_cache"]


def plain_shared(s):
    hkv, block = s["k_cache"].shape[2], s["q"].shape[1]
    q = stacked(s["q"], hkv, F32)
    at_prefix = s["prefix_table"].long()
    k, v = (c[at_prefix].flatten(0, 1)[: s["prefix"]].transpose(0, 1).float() for c in (s["k_cache"], s["v_cache"]))
    mine, there = own_scores(s, F32)
    scores = torch.cat([q @ k.transpose(1, 2) * s["scale"], mine], -1)
    top = scores.amax(-1, keepdim=True)
    p = (scores - top).exp()
    total = p.sum(-1, keepdim=True)
    own_v = own_keys(s["v_cache"], s["table"], s["longest"], F32) * there[:, None, :, None]
    o = (p[..., : s["prefix"]] @ v + p[..., s["prefix"]:] @ own_v) / total
    return unstacked(o, block).to(BF), unstacked((total.log() + top)[..., 0], block)


def plain_weights(s):
    scores, there = own_scores(s, F32)
    lse = stacked(s["lse"][..., None], s["k_cache"].shape[2], F32)
    got = (scores - lse).exp().sum(2) + s["decay"] * s["previous"]
    return got.masked_fill(~there[:, None], 0.0)


def chosen(weights, seqlens, budget, recent):
    """(old places, ascending, and whether each is one) of the keys that stay: [bs, kv heads, budget]."""
    n = weights.shape[-1]
    at = torch.arange(n, device=DEV)
    end = seqlens[:, None, None]
    rank = torch.where(at >= end - recent, math.inf, weights.double()).masked_fill(at >= end, -math.inf)
    order = rank.argsort(dim=-1, descending=True, stable=True)[..., :budget]      # (the budget is at most the longest)
    order = torch.where(torch.arange(order.shape[-1], device=DEV) < end, order, n).sort(dim=-1).values
    return order.clamp(max=n - 1), order < n


def plain_evict(s):
    w, table, to, budget = s["weights"], s["table"], s["to"], s["budget"]
    place, real = chosen(w, s["seqlens"], budget, s["recent"])
    bs, hkv, _ = place.shape
    b, h, i = torch.where(real)
    old, new = place[b, h, i], i
    src = table[b, old // PAGE].long() * PAGE + old % PAGE
    dst = to[b, new // PAGE].long() * PAGE + new % PAGE
    for c in (s["k_cache"], s["v_cache"]):
        rows = c.flatten(0, 1)
        rows[dst, h] = rows[src, h]
    kept = torch.where(real, place, -1).to(torch.int32)
    return kept, s["seqlens"].clamp(max=budget), w.gather(2, place).masked_fill(~real, 0.0), s["k_cache"][s["first_out"]:], s["v_cache"][s["first_out"]:]


def run(s):
    if not own:
        return {"rotary": plain_rotary, "shared": plain_shared, "weights": plain_weights, "evict": plain_evict}[s["kind"]](s)
    ops = importlib.import_module("mineru-diffusion_b200").ops
    if s["kind"] == "rotary":
        if "slots" not in s:
            return ops.rotary_embed(s["q"], s["k"], s["positions"], s["inv_freq"], interleaved=s["pairs"], scale=s["factor"])
        q, _ = ops.rotary_embed(s["q"], s["k"], s["positions"], s["inv_freq"], interleaved=s["pairs"], scale=s["factor"], v=s["v"],
                                k_cache=s["k_cache"], v_cache=s["v_cache"], slot_mapping=s["slots"])
        return q, s["k_cache"], s["v_cache"]
    if s["kind"] == "shared":
        return ops.block_attn_shared_prefix(s["q"], s["k_cache"], s["v_cache"], s["prefix_len"], s["prefix_table"], s["seqlens"],
                                            s["table"], softmax_scale=s["scale"], want_lse=True)
    if s["kind"] == "weights":
        return ops.key_weights(s["q"], s["k_cache"], s["lse"], s["seqlens"], s["table"], softmax_scale=s["scale"],
                               previous=s["previous"], decay=s["decay"])
    kept, seqlens, weights = ops.evict_kvcache(s["k_cache"], s["v_cache"], s["weights"], s["seqlens"], s["table"], s["budget"],
                                               s["recent"], out_table=s["to"])
    return kept, seqlens, weights, s["k_cache"][s["first_out"]:], s["v_cache"][s["first_out"]:]


# ----------------------------------------------------------------------------- 64 bits, from the definitions
def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind == "rotary":
        r = s["rot"]
        z = torch.polar(torch.full((), s["factor"], dtype=F64, device=DEV).expand(case["n"], r // 2),
                        s["positions"].to(F64)[:, None] * s["inv_freq"])[:, None]

        def turn(x):
            y = x.to(F64).clone()
            first, second = (slice(0, r, 2), slice(1, r, 2)) if s["pairs"] else (slice(0, r // 2), slice(r // 2, r))
            turned = torch.complex(y[..., first], y[..., second]) * z
            y[..., first], y[..., second] = turned.real, turned.imag
            return y

        q, k = turn(s["q"]), turn(s["k"])
        if "slots" not in s:
            return q, k
        caches = [torch.zeros(c.shape, dtype=F64, device=DEV) for c in (s["k_cache"], s["v_cache"])]
        for c, x in zip(caches, (k, s["v"].to(F64))):
            c.view(-1, *c.shape[2:]).index_copy_(0, s["slots"].long(), x)
        return q, caches[0], caches[1]
    if kind == "evict":
        lens, table, to = lengths(case), s["table"].long(), s["to"].long()
        bs, hkv, budget = case["bs"], case["hkv"], case["budget"]
        kept = torch.full((bs, hkv, budget), -1, dtype=torch.int32, device=DEV)
        w_out = torch.zeros(bs, hkv, budget, dtype=F64, device=DEV)
        caches = [c.to(F32) for c in (s["k_cache"], s["v_cache"])]
        for b, n in enumerate(lens):
            m, free = min(n, budget), n - min(n, case["recent"])
            src = (table[b, :, None] * PAGE + torch.arange(PAGE, device=DEV)).flatten()[:n]
            dst = (to[b, :, None] * PAGE + torch.arange(PAGE, device=DEV)).flatten()[:m]
            for h in range(hkv):
                w = s["weights"][b, h, :n].to(F64)
                _, by_weight = torch.sort(-w[:free], stable=True)
                stay = torch.cat([by_weight[: m - (n - free)], torch.arange(free, n, device=DEV)]).sort().values
                kept[b, h, :m], w_out[b, h, :m] = stay.to(torch.int32), w[stay]
                for c in caches:
                    rows = c.view(-1, hkv, HEAD)
                    rows[dst, h] = rows[src[stay], h]
        return kept, torch.tensor([min(n, budget) for n in lens], dtype=torch.int32, device=DEV), w_out, \
            caches[0][s["first_out"]:].to(F64), caches[1][s["first_out"]:].to(F64)
    hq, hkv, block = case["hq"], case["hkv"], case["block"]
    group = hq // hkv

    def rows_of(cache, pages, n, h):
        return cache[pages.long(), :, h].reshape(-1, HEAD)[:n].to(F64)

    if kind == "weights":
        got = torch.zeros(s["previous"].shape, dtype=F64, device=DEV)
        for b, n in enumerate(lengths(case)):
            pages = s["table"][b, : -(-n // PAGE)]
            for h in range(hkv):
                q = s["q"][b, :, h * group:(h + 1) * group].reshape(-1, HEAD).to(F64)
                lse = s["lse"][b, :, h * group:(h + 1) * group].reshape(-1, 1).to(F64)
                p = torch.exp(q @ rows_of(s["k_cache"], pages, n, h).T / math.sqrt(HEAD) - lse)
                got[b, h, :n] = p.sum(0) + s["decay"] * s["previous"][b, h, :n].to(F64)
        return got
    out = torch.empty(s["q"].shape, dtype=F64, device=DEV)
    lse = torch.empty(s["q"].shape[:3], dtype=F64, device=DEV)
    for h in range(hkv):
        kp, vp = (rows_of(c, s["prefix_table"], case["prefix"], h) for c in (s["k_cache"], s["v_cache"]))
        for b, n in enumerate(lengths(case)):
            pages = s["table"][b, : -(-n // PAGE)]
            k, v = (torch.cat([x, rows_of(c, pages, n, h)]) for x, c in ((kp, s["k_cache"]), (vp, s["v_cache"])))
            q = s["q"][b, :, h * group:(h + 1) * group].reshape(-1, HEAD).to(F64)
            z = q @ k.T / math.sqrt(HEAD)
            lse[b, :, h * group:(h + 1) * group] = torch.logsumexp(z, 1).view(block, group)
            out[b, :, h * group:(h + 1) * group] = (torch.softmax(z, 1) @ v).view(block, group, HEAD)
    return out, lse
