"""Attention that reads less than the whole cache, and the layer that keeps a state in its place, as measurable cases.

Shapes are those of the layer that bench.py runs: q has 8192 rows and k and v 1024 each, that is 64 query heads and
8 key/value heads of 128, or 32 and 4 of 256; layers with a state have as many values in as many heads.

op        what one pass does
sinks     attention over the paged cache with a sliding window and a few first tokens that stay visible
shared    attention of a batch whose sequences begin with the same long prefix, on the same pages
linear    linear attention with a decay for each head: prompts, drafts and single tokens, from and to slots of states
"""
import importlib.util
import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NAME = "qwen_3_8_27b_optimizations_amd"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "q8": 1 + 2 / 32}


def package():
    """The library's Python side (its directory's name holds a dot)."""
    if NAME not in sys.modules:
        d = os.path.join(ROOT, "qwen_3.8_27b_optimizations_amd")
        spec = importlib.util.spec_from_file_location(NAME, os.path.join(d, "__init__.py"),
                                                      submodule_search_locations=[d])
        sys.modules[NAME] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[NAME])
    return sys.modules[NAME]


# ------------------------------------------------------------------ cases
def heads(D):
    """Query and key/value heads of the layer for a head of D."""
    return {"hq": 8192 // D, "hk": 1024 // D, "d": D}


def listed():
    return [
        # one token of a long stream through a layer with a short window: launch latency counts
        {"name": "sinks_b1_w1k", "op": "sinks", "b": 1, "q": 1, "kv": 9000, "spread": 1.0, **heads(128), "cache": "f16",
         "page": 16, "out": "f16", "window": 1024, "sinks": 4, "lse": False},
        # a batch of streams of all lengths, some shorter than the window
        {"name": "sinks_b64_w4k", "op": "sinks", "b": 64, "q": 1, "kv": 32768, "spread": 64.0, **heads(128),
         "cache": "bf16", "page": 16, "out": "bf16", "window": 4096, "sinks": 4, "lse": False},
        # verifying drafts over an 8-bit cache with wide heads, statistics kept for merging
        {"name": "sinks_q8_b8_q5", "op": "sinks", "b": 8, "q": 5, "kv": 9001, "spread": 4.0, **heads(256), "cache": "q8",
         "page": 64, "out": "bf16", "window": 2048, "sinks": 64, "lse": True},
        # a prompt chunk far into a stream
        {"name": "sinks_chunk_2048", "op": "sinks", "b": 1, "q": 2048, "kv": 16384, "spread": 1.0, **heads(128),
         "cache": "f16", "page": 64, "out": "f16", "window": 4096, "sinks": 16, "lse": False},
        # a few samples of one prompt, the next token of each
        {"name": "shared_b4_2k", "op": "shared", "b": 4, "groups": 1, "q": 1, "shared": 2048, "kv": 129, "spread": 4.0,
         **heads(128), "cache": "f16", "page": 16, "out": "f16", "lse": False},
        # a batch of requests behind one long system prompt
        {"name": "shared_b64_16k", "op": "shared", "b": 64, "groups": 1, "q": 1, "shared": 16384, "kv": 1025,
         "spread": 64.0, **heads(128), "cache": "bf16", "page": 16, "out": "bf16", "lse": False},
        # drafts behind prefixes that do not end with a page, 8-bit cache, wide heads
        {"name": "shared_q8_b32_q4", "op": "shared", "b": 32, "groups": 2, "q": 4, "shared": 8187, "kv": 2000,
         "spread": 8.0, **heads(256), "cache": "q8", "page": 64, "out": "bf16", "lse": True},
        # questions of different lengths about one of two documents
        {"name": "shared_b8_q509", "op": "shared", "b": 8, "groups": 2, "q": 509, "shared": 12288, "kv": 0,
         "spread": 4.0, **heads(128), "cache": "f16", "page": 64, "out": "f16", "lse": False},
        # the next token of one sequence
        {"name": "linear_b1", "op": "linear", "b": 1, "t": 1, "spread": 1.0, "h": 64, "hk": 16, "dk": 128, "dv": 128,
         "in": "bf16", "out": "bf16", "each": True},
        # the next token of a batch, straight from fp32 projections
        {"name": "linear_b64", "op": "linear", "b": 64, "t": 1, "spread": 1.0, "h": 64, "hk": 64, "dk": 128, "dv": 128,
         "in": "f32", "out": "f32", "each": True},
        # one long prompt
        {"name": "linear_t4096", "op": "linear", "b": 1, "t": 4096, "spread": 1.0, "h": 64, "hk": 16, "dk": 128,
         "dv": 128, "in": "bf16", "out": "bf16", "each": True},
        # prompts of different lengths, decays that are constants of the heads, wide heads
        {"name": "linear_prompts_b5", "op": "linear", "b": 5, "t": 4001, "spread": 8.0, "h": 32, "hk": 32, "dk": 128,
         "dv": 256, "in": "f16", "out": "f32", "each": False},
    ]


def draw(rng):
    """A case of the same kinds over the whole range of lengths, heads, pages and types."""
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["sinks", "shared", "linear"])
    if op == "linear":
        hk = rng.choice([1, 2, 4, 8, 16, 16, 32])
        c = {"op": op, "hk": hk, "h": hk * rng.choice([1, 1, 2, 3, 4]), "dk": rng.choice([64, 128, 128, 256]),
             "dv": rng.choice([64, 128, 128, 256]), "in": rng.choice(["f16", "bf16", "bf16", "f32"]),
             "out": rng.choice(["f16", "bf16", "f32"]), "each": rng.random() < 0.6, "b": spread(1, 64),
             "spread": rng.choice([1.0, 2.0, 8.0, 64.0])}
        kind = rng.choice(["decode", "draft", "prompt", "prompt"])
        c["t"] = {"decode": 1, "draft": rng.randrange(2, 17)}.get(kind) or spread(17, 4096)
        while c["b"] * c["h"] * c["dk"] * c["dv"] > 64 * 64 * 128 * 128 \
                or c["b"] * c["t"] * c["h"] * c["dk"] * c["dv"] > 4096 * 64 * 128 * 128:
            c["b"], c["t"] = max(1, c["b"] // 2), c["t"] if c["b"] > 1 else c["t"] // 2
        return c
    d = rng.choice([64, 128, 128, 128, 256])
    hk = rng.choice([1, 2, 3, 4, 8, 8])
    group = rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 8, 8, 12, 16])
    cache = rng.choice(["f16", "bf16", "q8"])
    c = {"op": op, "hq": hk * group, "hk": hk, "d": d, "cache": cache, "page": rng.choice([16, 16, 32, 64, 128, 256]),
         "out": cache if cache != "q8" else rng.choice(["f16", "bf16"]), "spread": rng.choice([1.0, 2.0, 8.0, 64.0]),
         "b": spread(1, 64), "lse": rng.random() < 0.3}
    kind = rng.choice(["decode", "decode", "verify", "chunk", "prompt"])
    c["q"] = {"decode": 1, "verify": rng.randrange(2, 17)}.get(kind) or spread(17, 2048)
    c["kv"] = 0 if kind == "prompt" else spread(c["q"], 32768 if op == "sinks" else 4096)
    if op == "sinks":
        c.update({"window": spread(1, 8192), "sinks": rng.choice([1, 4, 4, 16, spread(1, 512)])})
    else:
        c.update({"shared": spread(16, 32768), "groups": rng.choice([1, 1, 1, 2, 3])})
        c["b"] = max(2, c["b"])
        c["groups"] = min(c["groups"], c["b"])
    # no more work than the largest listed cases, and scores of the plain form that fit the card
    while c["b"] * c["hq"] * c["q"] * keys_at_most(c) > 1 << 31 \
            or c["b"] * c["hq"] * c["q"] * keys_at_most(c) * d > 64 * 2048 * 12000 * 128 \
            or c["b"] * (c["hq"] * c["q"] + hk * keys_at_most(c)) * d > 131072 * 1984:
        if c["b"] > 2:
            c["b"] //= 2
            if op == "shared":
                c["groups"] = min(c["groups"], c["b"])
        elif op == "shared" and c["shared"] > 4096:
            c["shared"] //= 2
        elif c["kv"] > 2 * c["q"]:
            c["kv"] //= 2
        else:
            c["q"] = max(1, c["q"] // 2)
            c["kv"] //= 2
    return c


def longest(c):
    return c["kv"] or c["q"]


def keys_at_most(c):
    return longest(c) + (c["shared"] if c["op"] == "shared" else 0)


def lengths(c):
    """(kv, q, shared): cached and new tokens of each sequence, and the shared tokens of each group.  The longest sequence
    has c's; the others are down to `spread` times shorter."""
    most = c["t"] if c["op"] == "linear" else longest(c)
    rng = random.Random("%s %s %s" % (c["b"], most, c["spread"]))
    kv = [most] + [max(1, int(most * math.exp(-rng.random() * math.log(c["spread"])))) for _ in range(c["b"] - 1)]
    if c["op"] == "linear":
        return kv, list(kv), []
    if not c["kv"]:
        q = list(kv)
    else:
        q = [c["q"]] + [c["q"] if c["q"] == 1 else rng.randrange(1, c["q"] + 1) for _ in range(c["b"] - 1)]
        kv = [max(a, b) for a, b in zip(kv, q)]
    if c["op"] == "sinks":
        return kv, q, []
    shared = [c["shared"]] + [max(1, int(c["shared"] * rng.uniform(0.5, 1))) for _ in range(c["groups"] - 1)]
    return [n + shared[g] for n, g in zip(kv, group_of(c))], q, shared


def first_of(c):
    """First sequence of each group, and the end."""
    return [i * c["b"] // c["groups"] for i in range(c["groups"] + 1)]


def group_of(c):
    f = first_of(c)
    return [g for g in range(c["groups"]) for _ in range(f[g], f[g + 1])]


# ------------------------------------------------------------------ inputs
def device():
    return torch.device("cuda:0")


def normal(gen, *shape):
    return torch.randn(*shape, device=device(), generator=gen)


def whole(v):
    return torch.tensor(v, dtype=torch.int32, device=device())


def starts_of(v):
    s = [0]
    for n in v:
        s.append(s[-1] + n)
    return whole(s)


def quantised(x):
    """Codes and fp16 scales of groups of 32 values along the last axis."""
    v = x.unflatten(-1, (-1, 32))
    d = (v.abs().amax(-1) / 127).clamp(max=65504 / 127).half()
    codes = torch.where(d[..., None] > 0, v / d[..., None].float(), torch.zeros_like(v)).round().clamp(-127, 127)
    return codes.flatten(-2).to(torch.int8), d


def inputs(c, seed):
    """Everything random in a case, from the seed alone."""
    gen = torch.Generator(device=device()).manual_seed(1000003 * seed + 31)
    if c["op"] == "linear":
        return linear_inputs(c, gen)
    hq, hk, d, page = c["hq"], c["hk"], c["d"], c["page"]
    kv, q, shared = lengths(c)
    ids = group_of(c) if shared else []
    # whole pages of a prefix are shared, the rest of it and what follows are each sequence's own
    common = [n // page for n in shared]
    per = [-(-n // page) - (common[ids[i]] if shared else 0) for i, n in enumerate(kv)]
    total = sum(per) + sum(common) + 3
    order = torch.randperm(total, device=device(), generator=gen).to(torch.int32)
    pool = normal(gen, 2, total, hk, page, d)
    table = torch.full((len(kv), max(-(-n // page) for n in kv)), -1, dtype=torch.int32, device=device())
    at = 0
    for g, n in enumerate(common):
        f = first_of(c)
        table[f[g]:f[g + 1], :n] = order[at:at + n]
        at += n
    for i, n in enumerate(per):
        n0 = common[ids[i]] if shared else 0
        table[i, n0:n0 + n] = order[at:at + n]
        at += n
    rows = 1.7 * normal(gen, sum(q), hq, d)
    if c["op"] == "sinks":
        # the first tokens draw weight from every row and have little to say
        toward = torch.sign(normal(gen, d))
        rows += 0.5 * toward
        j = torch.arange(min(c["sinks"], min(kv)), device=device())
        here, off = table[:, j // page].long(), (j % page).expand(len(kv), -1)
        pool[0][here, :, off] += 1.5 * toward
        pool[1][here, :, off] *= 0.1
    else:
        # tokens of a prefix in a page that it shares with what follows are the same in every sequence
        for g, n in enumerate(shared):
            for i in range(first_of(c)[g] + 1, first_of(c)[g + 1]):
                if n % page:
                    a, b = int(table[first_of(c)[g], n // page]), int(table[i, n // page])
                    pool[:, b, :, :n % page] = pool[:, a, :, :n % page]
    s = {"table": table, "kv_len": whole(kv), "most_kv": max(kv), "starts": starts_of(q), "total": sum(q),
         "most_q": max(q), "q": rows.to(TYPES[c["out"]]), **stored(c, pool)}
    if shared:
        f = first_of(c)
        s.update(shared_len=whole(shared), most_shared=max(shared), groups=whole(f) if len(shared) > 1 else None,
                 most_own=max(n - shared[ids[i]] for i, n in enumerate(kv)),
                 most_group=max(sum(q[f[g]:f[g + 1]]) for g in range(len(shared))))
    return s


def stored(c, pool):
    """Key and value pages [pages][heads][tokens of a page][head] in the cache's type."""
    if c["cache"] != "q8":
        k, v = pool.to(TYPES[c["cache"]])
        return {"k_pages": k.contiguous(), "v_pages": v.contiguous(), "k_scales": None, "v_scales": None}
    (k, v), (ks, vs) = quantised(pool)
    return {"k_pages": k.contiguous(), "v_pages": v.contiguous(), "k_scales": ks.contiguous(),
            "v_scales": vs.contiguous()}


def linear_inputs(c, gen):
    kind, n = TYPES[c["in"]], lengths(c)[0]
    total, b = sum(n), len(n)
    unit = lambda x: x / x.norm(dim=-1, keepdim=True)  # noqa: E731
    # how long a head remembers, from a few tokens to thousands, and with `each` how much of it a token lets go
    slow = torch.exp(torch.linspace(math.log(0.3), math.log(3e-4), c["h"], device=device()))
    decay = -slow[torch.randperm(c["h"], device=device(), generator=gen)]
    if c["each"]:
        decay = decay * torch.nn.functional.softplus(normal(gen, total, c["h"]) + 0.5)
    states = 0.3 * normal(gen, 2 * b, c["h"], c["dk"], c["dv"])
    slots = torch.randperm(2 * b, device=device(), generator=gen)
    return {"q": unit(normal(gen, total, c["hk"], c["dk"])).to(kind), "k": unit(normal(gen, total, c["hk"], c["dk"])).to(kind),
            "v": normal(gen, total, c["h"], c["dv"]).to(kind), "decay": decay.contiguous(), "states": states,
            "from_slots": slots[:b].contiguous(), "to_slots": slots[b:].contiguous(), "starts": starts_of(n),
            "most_q": max(n)}


def prepare(case, seed):
    return {"case": dict(case), **inputs(case, seed)}


# ------------------------------------------------------------------ the framework's calls
def cache_of(s):
    """The handle of the pages, which a program makes once."""
    if "handle" not in s:
        s["handle"] = package().KVCache(s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"])
    return s["handle"]


def own_run(s):
    pkg, c = package(), s["case"]
    if c["op"] == "linear":
        # a sequence's state comes from one slot and goes to another, as where a prompt's state is kept for later
        out = pkg.linear_attention(s["q"], s["k"], s["v"], s["decay"], s["starts"], s["most_q"], states=s["states"],
                                   from_slots=s["from_slots"], to_slots=s["to_slots"], scale=1.0,
                                   out_type=TYPES[c["out"]])
        return [out, s["states"]]
    if c["op"] == "sinks":
        got = pkg.paged_attention(s["q"], cache_of(s), s["table"], s["starts"], s["kv_len"], s["most_q"], s["most_kv"],
                                  window=c["window"], sinks=c["sinks"], lse=c["lse"])
    else:
        got = pkg.shared_attention(s["q"], cache_of(s), s["table"], s["starts"], s["kv_len"], s["shared_len"],
                                   s["most_q"], s["most_own"], s["most_shared"], groups=s["groups"],
                                   most_group=s["most_group"], lse=c["lse"])
    return list(got) if c["lse"] else got


# ------------------------------------------------------------------ the plain form
def rows_of(pages, scales, ids, off):
    """Tokens [...][heads][head] at pages `ids` and offsets `off` in them, in fp32."""
    x = pages[ids, :, off].float()
    if scales is None:
        return x
    return (x.unflatten(-1, (-1, 32)) * scales[ids, :, off].float()[..., None]).flatten(-2)


def keys_and_values(s, c, table, at, there):
    """Cached tokens `at` of the sequences of `table`: keys [b, hk, d, keys] and values [b, hk, keys, d]."""
    page = c["page"]
    ids = torch.where(there, torch.gather(table, 1, (at // page).clamp(max=table.shape[1] - 1)), 0).long()
    k = rows_of(s["k_pages"], s["k_scales"], ids, at % page).permute(0, 2, 3, 1).contiguous()
    v = rows_of(s["v_pages"], s["v_scales"], ids, at % page).transpose(1, 2).contiguous()
    return k, v


def plain_run(s):
    c = s["case"]
    if c["op"] == "linear":
        return plain_linear(s, c)
    hq, hk, d, dev = c["hq"], c["hk"], c["d"], device()
    b, group, most_q = s["kv_len"].numel(), hq // hk, s["most_q"]
    new = s["starts"][1:] - s["starts"][:-1]
    step = torch.arange(most_q, device=dev)
    row = torch.where(step < new[:, None], s["starts"][:-1, None] + step, 0).long()
    mine = (step < new[:, None]).nonzero(as_tuple=True)
    q = s["q"][row].float().view(b, most_q, hk, group, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)
    p = (s["kv_len"] - new)[:, None] + step  # a row's place
    if c["op"] == "sinks":
        # what some row of a sequence sees of it: the first tokens, and those after the first row's window
        lo = (s["kv_len"] - new - c["window"] + 1).clamp(min=0)
        span = min(s["most_kv"], c["window"] + most_q)
        at = torch.cat([torch.arange(min(c["sinks"], s["most_kv"]), device=dev).expand(b, -1),
                        lo[:, None] + torch.arange(span, device=dev)], 1)
        there = at < s["kv_len"][:, None]
        there[:, -span:] &= at[:, -span:] >= c["sinks"]
        seen = there[:, None] & (at[:, None] <= p[..., None])
        seen &= (at[:, None] > p[..., None] - c["window"]) | (at[:, None] < c["sinks"])
        k, v = keys_and_values(s, c, s["table"], at, there)
        score = torch.matmul(q, k).view(b, hk, group, most_q, -1) * d ** -0.5
        score.masked_fill_(~seen[:, None, None], -math.inf)
        return finish(c, score, lambda w: torch.matmul(w.view(b, hk, -1, at.shape[1]), v), mine)
    # the prefix of each group once, for the rows of all its sequences
    before = torch.zeros(b, dtype=torch.long, device=dev)
    first = first_of(c)
    for g in range(c["groups"]):
        before[first[g]:first[g + 1]] = s["shared_len"][g]
    at = before[:, None] + torch.arange(s["most_own"], device=dev)
    there = at < s["kv_len"][:, None]
    k, v = keys_and_values(s, c, s["table"], at, there)
    score = q.new_full((b, hk, group, most_q, s["most_shared"] + s["most_own"]), -math.inf)
    tail = torch.matmul(q, k).view(b, hk, group, most_q, -1) * d ** -0.5
    seen = there[:, None] & (at[:, None] <= p[..., None])
    score[..., s["most_shared"]:] = tail.masked_fill_(~seen[:, None, None], -math.inf)
    prefix = []
    for g in range(c["groups"]):
        i, n = slice(first[g], first[g + 1]), lengths(c)[2][g]
        at = torch.arange(n, device=dev)[None]
        pk, pv = keys_and_values(s, c, s["table"][first[g]:first[g] + 1], at, at < n)
        z = torch.matmul(q[i].transpose(0, 1).reshape(hk, -1, d), pk[0]) * d ** -0.5
        score[i, ..., :n] = z.view(hk, -1, group, most_q, n).transpose(0, 1)
        prefix.append((i, n, pv[0]))

    def product(w):
        o = torch.matmul(w[..., s["most_shared"]:].reshape(b, hk, -1, s["most_own"]), v)
        for i, n, pv in prefix:
            z = torch.matmul(w[i, ..., :n].transpose(0, 1).reshape(hk, -1, n), pv)
            o[i] += z.view(hk, i.stop - i.start, -1, d).transpose(0, 1)
        return o

    return finish(c, score, product, mine)


def finish(c, score, product, mine):
    """Softmax over the last axis of [b, hk, group, rows, keys] and its product with the values."""
    b, hk, group, rows, _ = score.shape
    top = score.amax(-1, keepdim=True)
    weight = score.sub_(torch.where(top == -math.inf, 0, top)).exp_()
    total = weight.sum(-1, keepdim=True)
    o = product(weight).view(b, hk, group, rows, c["d"])
    o = torch.where(total > 0, o / total, 0).permute(0, 3, 1, 2, 4).reshape(b, rows, c["hq"], c["d"])
    if not c["lse"]:
        return o[mine].to(TYPES[c["out"]])
    lse = (top + total.log()).squeeze(-1).permute(0, 3, 1, 2).reshape(b, rows, c["hq"])
    return [o[mine].to(TYPES[c["out"]]), lse[mine]]


def plain_linear(s, c):
    """All sequences padded to the longest, in chunks of 128 tokens (a single token is a chunk of one)."""
    b, h, T, dev = c["b"], c["h"], s["most_q"], device()
    new = s["starts"][1:] - s["starts"][:-1]
    step = torch.arange(T, device=dev)
    in_it = step < new[:, None]
    row = torch.where(in_it, s["starts"][:-1, None] + step, 0).long()

    def padded(x):
        x = torch.where(in_it[..., None, None], x[row].float(), 0).transpose(1, 2)
        return x.repeat_interleave(h // x.shape[1], dim=1) if x.shape[1] < h else x

    q, k, v = padded(s["q"]), padded(s["k"]), padded(s["v"])
    decay = s["decay"][row] if c["each"] else s["decay"].expand(b, T, h)
    decay = torch.where(in_it[..., None], decay, 0).transpose(1, 2).double()
    S = s["states"][s["from_slots"]]
    out = torch.empty_like(v)
    for t in range(0, T, 128):
        qc, kc, vc = q[:, :, t:t + 128], k[:, :, t:t + 128], v[:, :, t:t + 128]
        G = decay[:, :, t:t + 128].cumsum(-1)
        n = G.shape[-1]
        later = torch.ones(n, n, dtype=torch.bool, device=dev).triu(1)
        w = (G[..., :, None] - G[..., None, :]).masked_fill_(later, -math.inf).float().exp_()
        w *= torch.matmul(qc, kc.transpose(-1, -2).contiguous())
        out[:, :, t:t + 128] = torch.matmul(w, vc) + torch.matmul(qc * G.exp()[..., None].float(), S)
        keep = (G[..., -1:] - G).exp()[..., None].float()
        S = S * G[..., -1:, None].exp().float() + torch.matmul((kc * keep).transpose(-1, -2).contiguous(), vc)
    s["states"][s["to_slots"]] = S
    return [out.transpose(1, 2)[in_it].to(TYPES[c["out"]]), s["states"]]


def run(state):
    return own_run(state) if own else plain_run(state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(c):
    kv, q, shared = lengths(c)
    if c["op"] == "linear":
        total, size = sum(q), c["h"] * c["dk"] * c["dv"]
        n = total * (2 * c["hk"] * c["dk"] + c["h"] * c["dv"]) * BYTES[c["in"]] + total * c["h"] * c["dv"] * BYTES[c["out"]]
        n += 4 * c["h"] * (total if c["each"] else 1)
        return {"bytes": n + 2 * 4 * len(q) * size, "flops": 4 * total * size}
    hq, hk, d = c["hq"], c["hk"], c["d"]
    pairs = keys = 0
    for n, new in zip(kv, q):
        if c["op"] == "sinks":
            for p in range(n - new, n):
                lo = max(0, p + 1 - c["window"])
                pairs += p + 1 - lo + min(lo, c["sinks"])
            lo = max(0, n - new + 1 - c["window"])
            keys += n - lo + min(lo, c["sinks"])
        else:
            pairs += new * n - new * (new - 1) // 2
    if shared:
        keys = sum(shared) + sum(n - shared[g] for n, g in zip(kv, group_of(c)))
    rows = sum(q)
    return {"bytes": 2 * keys * hk * d * BYTES[c["cache"]] + 2 * rows * hq * d * BYTES[c["out"]]
            + 4 * rows * hq * c["lse"], "flops": 4 * pairs * hq * d}


# ------------------------------------------------------------------ the same in 64 bits
def exact(case, seed):
    c, s = case, inputs(case, seed)
    kv, q, _ = lengths(c)
    if c["op"] == "linear":
        return exact_linear(c, s, q)
    outs, sums, first = [], [], 0
    for i, n in enumerate(kv):
        per = -(-n // c["page"])
        x = {}
        for name in "kv":
            pages = s[name + "_pages"][s["table"][i, :per].long()].double()
            if c["cache"] == "q8":
                scales = s[name + "_scales"][s["table"][i, :per].long()].double()
                pages = pages * scales.repeat_interleave(32, dim=-1)
            x[name] = pages.transpose(0, 1).reshape(c["hk"], -1, c["d"])[:, :n].contiguous()
        kt = x["k"].transpose(1, 2).contiguous()
        j = torch.arange(n, device=device())
        for r in range(0, q[i], 64):
            m = min(64, q[i] - r)
            p = n - q[i] + r + torch.arange(m, device=device())[:, None]
            hidden = j > p
            if c["op"] == "sinks":
                hidden |= (j <= p - c["window"]) & (j >= c["sinks"])
            y = s["q"][first + r:first + r + m].double().view(m, c["hk"], -1, c["d"]).permute(1, 2, 0, 3)
            z = (y.reshape(c["hk"], -1, c["d"]) @ kt).view(c["hk"], -1, m, n) / math.sqrt(c["d"])
            z = z.masked_fill(hidden, -math.inf)
            o = torch.softmax(z, -1).view(c["hk"], -1, n) @ x["v"]
            outs.append(o.view(c["hk"], -1, m, c["d"]).permute(2, 0, 1, 3).reshape(m, c["hq"], c["d"]))
            sums.append(torch.logsumexp(z, -1).permute(2, 0, 1).reshape(m, c["hq"]))
        first += q[i]
    return [torch.cat(outs), torch.cat(sums)] if c["lse"] else torch.cat(outs)


def exact_linear(c, s, n):
    """Token by token, all sequences together."""
    S = s["states"][s["from_slots"]].double()
    out = torch.zeros(sum(n), c["h"], c["dv"], dtype=torch.float64, device=device())
    group = c["h"] // c["hk"]
    lens = torch.tensor(n, device=device())
    first = s["starts"][:-1].long()
    decay = s["decay"].double().exp()
    for t in range(max(n)):
        live = (lens > t).nonzero(as_tuple=True)[0] if min(n) <= t else slice(None)
        rows = first[live] + t
        a = decay[rows] if c["each"] else decay[None]
        k = s["k"][rows].double().repeat_interleave(group, dim=1)
        q = s["q"][rows].double().repeat_interleave(group, dim=1)
        new = S[live] * a[..., None, None] + k[..., None] * s["v"][rows].double()[..., None, :]
        S[live] = new
        out[rows] = (q[..., None] * new).sum(-2)
    states = s["states"].double()
    states[s["to_slots"]] = S
    return [out, states]
