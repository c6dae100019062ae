"""The operators of token generation, as timed and compared cases: the paged key-value cache, the
attention of one new token over it, eviction from it, and the draw of the next token.

Kinds and their fields:
  append  B, S, L, Hq, Hkv, D, page, dtype, ragged, weights: packed QKV rows of S new tokens a sequence go
          into a cache that holds up to L tokens a sequence already
  decode  B, L, Hq, Hkv, D, page, dtype, ragged, weights (the softmax weights are added to the cache's)
  evict   B, L, budget, sink, recent, Hkv, D, page, dtype: sequences of L/2 to L tokens are cut to the budget,
          into pages of their own
  sample  rows, V, dtype, k, p, mp: k, p, mp say whether top-k, top-p and min-p are used

Layout of the cache: pages of `page` tokens in 32 x 32 blocks, K [pages, Hkv, page/32, D/32, 32 tokens, 32 dims]
and V [pages, Hkv, page/32, D/32, 32 dims, 32 tokens]; table [B, max_pages] names a sequence's pages.
"""
from __future__ import annotations

import math

import torch

own = False

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one decoding step of a batch: a row a sequence, bound by the launch
        {"name": "append-step", "kind": "append", "B": 64, "S": 1, "L": 512, "Hq": 32, "Hkv": 8, "D": 128, "page": 64,
         "dtype": "bf16", "ragged": 1, "weights": 0},
        # prompts of several users, appended behind what their sequences hold already
        {"name": "append-prompt", "kind": "append", "B": 6, "S": 1531, "L": 700, "Hq": 16, "Hkv": 4, "D": 64,
         "page": 32, "dtype": "f16", "ragged": 1, "weights": 1},
        # the first tokens of a single chat: latency
        {"name": "decode-small", "kind": "decode", "B": 1, "L": 200, "Hq": 8, "Hkv": 8, "D": 64, "page": 32,
         "dtype": "f16", "ragged": 0, "weights": 0},
        # one user with a very long document
        {"name": "decode-one-long", "kind": "decode", "B": 1, "L": 131035, "Hq": 32, "Hkv": 8, "D": 128, "page": 256,
         "dtype": "bf16", "ragged": 0, "weights": 0},
        # a serving batch of grouped heads, each sequence at a length of its own
        {"name": "decode-batch", "kind": "decode", "B": 64, "L": 4096, "Hq": 32, "Hkv": 8, "D": 128, "page": 64,
         "dtype": "f16", "ragged": 1, "weights": 0},
        # all query heads on one key head
        {"name": "decode-mqa", "kind": "decode", "B": 16, "L": 8192, "Hq": 32, "Hkv": 1, "D": 128, "page": 128,
         "dtype": "bf16", "ragged": 1, "weights": 0},
        # a step whose weights decide a later eviction
        {"name": "decode-weights", "kind": "decode", "B": 12, "L": 2500, "Hq": 16, "Hkv": 4, "D": 64, "page": 64,
         "dtype": "f16", "ragged": 1, "weights": 1},
        # a small cache that went over its budget
        {"name": "evict-small", "kind": "evict", "B": 4, "L": 1180, "budget": 1000, "sink": 4, "recent": 256, "Hkv": 4,
         "D": 64, "page": 32, "dtype": "f16"},
        # long contexts of a batch cut to half
        {"name": "evict-half", "kind": "evict", "B": 16, "L": 8192, "budget": 4096, "sink": 4, "recent": 512, "Hkv": 8,
         "D": 128, "page": 64, "dtype": "bf16"},
        # one row of the 8192-word decoder's logits
        {"name": "sample-one", "kind": "sample", "rows": 1, "V": 8192, "dtype": "f16", "k": 1, "p": 1, "mp": 0},
        # a serving batch, every sequence with its own settings
        {"name": "sample-batch", "kind": "sample", "rows": 64, "V": 32003, "dtype": "bf16", "k": 1, "p": 1, "mp": 1},
        # a large batch over a large vocabulary in fp32, nucleus sampling
        {"name": "sample-large", "kind": "sample", "rows": 256, "V": 131072, "dtype": "f32", "k": 0, "p": 1, "mp": 1},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choices(("append", "decode", "evict", "sample"), (2, 5, 2, 3))[0]
    if kind == "sample":
        v = _log_int(rng, 300, 131072)
        return {"kind": kind, "rows": _log_int(rng, 1, min(256, (1 << 24) // v)), "V": v,
                "dtype": rng.choice(("f16", "bf16", "f32")), "k": rng.randint(0, 1), "p": rng.randint(0, 1),
                "mp": rng.randint(0, 1)}
    most = 1 << 27                        # elements of K in the cache
    while True:
        hkv, d, page = rng.choice((1, 2, 4, 8, 16)), rng.choice((64, 128)), rng.choice((32, 64, 128, 256))
        c = {"kind": kind, "B": _log_int(rng, 1, 128), "L": _log_int(rng, 1, 131072), "Hkv": hkv, "D": d, "page": page,
             "dtype": rng.choice(("f16", "bf16"))}
        if kind == "evict":
            c["L"] = max(64, c["L"])
            c["budget"] = rng.randint(max(32, c["L"] // 4), c["L"])
            c["sink"], c["recent"] = rng.choice((0, 1, 4, 16)), rng.randint(0, c["budget"] // 2)
            n = c["L"] + c["budget"]
        else:
            c["Hq"] = hkv * rng.choice((1, 2, 3, 4, 8, 16))
            c["ragged"], c["weights"] = int(c["B"] > 1), rng.randint(0, 1)
            c["S"] = rng.choice((1, _log_int(rng, 1, 2048)))
            n = c["L"] + (c["S"] if kind == "append" else 0)
            if kind == "decode":
                del c["S"]
        if c.get("Hq", 1) <= 64 and c["B"] * n * hkv * d <= most // (2 if kind == "append" else 1):
            return c


# ---- inputs ---------------------------------------------------------------------------------


def _gen(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 64 + salt)
    return g


def _randn(shape, seed, salt, mul=1.0, dtype=torch.float32):
    return torch.randn(shape, generator=_gen(seed, salt), device="cuda", dtype=dtype) * mul


def _ints(lo, hi, n, seed, salt):
    return torch.randint(lo, hi + 1, (n,), generator=_gen(seed, salt), device="cuda").to(torch.int32)


def _pages(n, page):
    return (n + page - 1) // page


def _cache(case, seed, tables):
    """A pool with just the pages of the tables' sequences, in random order; `tables`: pages a sequence, one number
    a table."""
    B, total = case["B"], case["B"] * sum(tables)
    blocks = (total, case["Hkv"], case["page"] // 32, case["D"] // 32, 32, 32)
    s = {"k": _randn(blocks, seed, 1, 1.0, DT[case["dtype"]]), "v": _randn(blocks, seed, 2, 1.0, DT[case["dtype"]])}
    perm = torch.randperm(total, generator=_gen(seed, 3), device="cuda").to(torch.int32)
    s["tables"], at = [], 0
    for n in tables:
        s["tables"].append(perm[at:at + B * n].reshape(B, n).contiguous())
        at += B * n
    return s


def _inputs(case, seed):
    kind, dt = case["kind"], DT[case["dtype"]]
    if kind == "sample":
        n, V = case["rows"], case["V"]
        s = {"logits": (_randn((n, V), seed, 1, 3.0)).to(dt), "u": torch.rand(n, generator=_gen(seed, 2), device="cuda"),
             "temperature": 0.5 + torch.rand(n, generator=_gen(seed, 3), device="cuda"), "top_k": None, "top_p": None,
             "min_p": None}
        if n > 2:
            s["temperature"][1] = 0.0     # a greedy user
        if case["k"]:
            s["top_k"] = _ints(1, max(1, min(V // 2, 200)), n, seed, 4)
        if case["p"]:
            s["top_p"] = 0.5 + 0.5 * torch.rand(n, generator=_gen(seed, 5), device="cuda")
        if case["mp"]:
            s["min_p"] = 0.1 * torch.rand(n, generator=_gen(seed, 6), device="cuda")
        return s
    B, L, Hkv, D, page = (case[k] for k in ("B", "L", "Hkv", "D", "page"))
    if kind == "evict":
        s = _cache(case, seed, (_pages(L, page), _pages(case["budget"], page)))
        s["len"] = _ints(L // 2, L, B, seed, 4)
        s["len"][0] = L
        s["len_out"] = torch.zeros_like(s["len"])
        # few keys gather most of the weight; the newest have none yet
        w = torch.rand((B, Hkv, _pages(L, page) * page), generator=_gen(seed, 5), device="cuda") ** 8
        s["weight"] = torch.where(w < 1e-6, torch.zeros_like(w), w)
        s["weight_out"] = torch.zeros((B, Hkv, _pages(case["budget"], page) * page), device="cuda")
        return s
    S = case.get("S", 0)
    s = _cache(case, seed, (_pages(L + S, page),))
    s["len"] = _ints(max(1, L // 4), L, B, seed, 4) if case["ragged"] else torch.full((B,), L, dtype=torch.int32, device="cuda")
    if case["ragged"]:
        s["len"][0] = L
        if B >= 8:
            s["len"][B // 2] = 0          # a slot of the batch that no sequence has taken yet
    s["weight"] = torch.rand((B, Hkv, _pages(L + S, page) * page), generator=_gen(seed, 5), device="cuda") if case["weights"] else None
    s["qkv"] = _randn((B, max(1, S), (case["Hq"] + 2 * Hkv) * D), seed, 6, 1.0, dt)
    if kind == "append":
        s["start"] = s["len"].clone()
        s["n_new"] = _ints((S + 1) // 2, S, B, seed, 7) if case["ragged"] else None
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        if case["kind"] == "sample":
            from tokamak_amd import runtime
            runtime.lib()
        else:
            from tokamak_amd import attn
            s["cache"] = attn.KvCache(s["k"], s["v"], s["tables"][0], s["len"], s["weight"])
            if case["kind"] == "evict":
                s["dst"] = attn.KvCache(s["k"], s["v"], s["tables"][1], s["len_out"], s["weight_out"])
    return s


# ---- the passes -----------------------------------------------------------------------------


def _dense(x, table, v=False):
    """A sequence's keys (values) in order, fp32: [B, Hkv, tokens, D]."""
    x = x[table.long()].float()                      # [B, pages, Hkv, page/32, D/32, 32, 32]
    x = x.permute(0, 2, 1, 3, 6, 4, 5) if v else x.permute(0, 2, 1, 3, 5, 4, 6)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[5] * 32)


def _plain_append(s, case):
    B, S, Hq, Hkv, D, page = (case[k] for k in ("B", "S", "Hq", "Hkv", "D", "page"))
    n = torch.full_like(s["start"], S) if s["n_new"] is None else s["n_new"]
    i = torch.arange(S, device="cuda")
    pos = s["start"].long()[:, None] + i
    b, i = torch.nonzero(i < n[:, None], as_tuple=True)
    pos = pos[b, i]
    at, tile, r = s["tables"][0][b, pos // page].long(), pos % page // 32, pos % 32
    rows = s["qkv"][b, i].reshape(-1, Hq + 2 * Hkv, D // 32, 32)
    s["k"][at, :, tile, :, r, :] = rows[:, Hq:Hq + Hkv]
    s["v"][at, :, tile, :, :, r] = rows[:, Hq + Hkv:]
    if s["weight"] is not None:
        s["weight"][b, :, pos] = 0.0
    s["len"].copy_(s["start"] + n)


def _plain_decode(s, case):
    B, Hq, Hkv, D = (case[k] for k in ("B", "Hq", "Hkv", "D"))
    q = s["qkv"][:, 0, :Hq * D].reshape(B, Hkv, Hq // Hkv, D).float()
    k, v = _dense(s["k"], s["tables"][0]), _dense(s["v"], s["tables"][0], True)
    seen = (torch.arange(k.shape[2], device="cuda") < s["len"][:, None])[:, None]         # [B, 1, tokens]
    x = torch.matmul(q, k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(D))
    x = x.masked_fill(~seen[:, :, None], -math.inf)
    m = x.amax(3, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = torch.exp(x - m)
    total = p.sum(3, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    o = torch.matmul(p, v.masked_fill(~seen[..., None], 0.0))
    out = {"o": o.reshape(B, Hq * D).to(s["qkv"].dtype), "lse": (m + torch.log(total)).reshape(B, Hq)}
    if s["weight"] is not None:
        s["weight"] += p.sum(2)
        out["weight"] = s["weight"]
    return out


def _plain_evict(s, case):
    B, budget, Hkv, page = (case[k] for k in ("B", "budget", "Hkv", "page"))
    n, w = s["len"].long()[:, None, None], s["weight"]
    t = torch.arange(w.shape[2], device="cuda").expand(w.shape)
    kind = (t < n).int() + ((t < n) & ((t < case["sink"]) | (t >= n - case["recent"]))).int()
    order = torch.sort(w, dim=2, descending=True, stable=True).indices
    order = order.gather(2, torch.sort(kind.gather(2, order), dim=2, descending=True, stable=True).indices)
    room = torch.arange(budget, device="cuda")
    have = room < n                                                                       # [B, 1, budget]
    at = torch.where(have, order[..., :budget], w.shape[2])
    at = torch.sort(at, dim=2).values                                                     # ascending, none at the end
    kept = torch.where(have, at, -1)
    src = kept.clamp(min=0)
    for name, val in (("k", False), ("v", True)):
        x = s[name]
        old, new = _dense(x, s["tables"][1], val), _dense(x, s["tables"][0], val)
        new = new.gather(2, src[..., None].expand(-1, -1, -1, new.shape[3]))
        old[:, :, :budget] = torch.where(have[..., None], new, old[:, :, :budget])
        y = old.reshape(B, Hkv, -1, page // 32, 32, case["D"] // 32, 32)
        x[s["tables"][1].long()] = (y.permute(0, 2, 1, 3, 5, 6, 4) if val else y.permute(0, 2, 1, 3, 5, 4, 6)).to(x.dtype)
    s["weight_out"][:, :, :budget] = torch.where(have, w.gather(2, src), s["weight_out"][:, :, :budget])
    s["len_out"].copy_(s["len"].clamp(max=budget))
    return kept.to(torch.int32)


def _plain_sample(s):
    x = s["logits"].double()
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    V, m = x.shape[1], x.amax(1, keepdim=True)
    temp = s["temperature"].double()[:, None]
    w = torch.exp((x - m) / torch.where(temp > 0, temp, torch.ones_like(temp)))
    w = torch.where(x == m, torch.ones_like(w), torch.where(x == -math.inf, torch.zeros_like(w), w))
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    if s["top_k"] is not None:
        k = s["top_k"][:, None]
        ws = ws * ((torch.arange(V, device="cuda") < k) | (k <= 0))
    if s["top_p"] is not None:
        p, run = s["top_p"].double()[:, None], ws.cumsum(1)
        ws = ws * ((run - ws < p * run[:, -1:]) | (p >= 1))
    if s["min_p"] is not None:
        ws = ws * (ws >= s["min_p"].double()[:, None])
    run = torch.zeros_like(w).scatter(1, order, ws).cumsum(1)
    token = (run <= s["u"].double()[:, None] * run[:, -1:]).sum(1)
    last = (run < run[:, -1:]).sum(1)                                                     # the last kept token
    best = torch.where(x == m, torch.arange(V, device="cuda"), V).amin(1)
    token = torch.where(temp[:, 0] > 0, torch.minimum(token, last), best)
    return torch.where(m[:, 0] == -math.inf, -1, token).to(torch.int32)


def run(s):
    case = s["case"]
    if case["kind"] == "sample":
        if not own:
            return {"token": _plain_sample(s)}
        from tokamak_amd import runtime
        return {"token": runtime.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                                        top_p=s["top_p"], min_p=s["min_p"])}
    if own:
        from tokamak_amd import attn
    if case["kind"] == "append":
        if own:
            attn.kv_append(s["qkv"], s["cache"], case["Hq"], start=s["start"], n_new=s["n_new"])
        else:
            _plain_append(s, case)
        out = {"k": s["k"], "v": s["v"], "len": s["len"]}
        return out if s["weight"] is None else {**out, "weight": s["weight"]}
    if case["kind"] == "decode":
        if not own:
            return _plain_decode(s, case)
        o, lse = attn.gqa_decode(s["qkv"][:, 0], s["cache"], case["Hq"], add_weights=bool(case["weights"]))
        return {"o": o, "lse": lse} if s["weight"] is None else {"o": o, "lse": lse, "weight": s["weight"]}
    if own:
        kept = attn.kv_evict(s["cache"], case["budget"], sink=case["sink"], recent=case["recent"], dst=s["dst"])
    else:
        kept = _plain_evict(s, case)
    return {"kept": kept, "k": s["k"], "v": s["v"], "len": s["len_out"], "weight": s["weight_out"]}


# ---- what a pass cannot do without ------------------------------------------------------------


def work(case):
    if case["kind"] == "sample":
        e = 4 if case["dtype"] == "f32" else 2
        return {"bytes": float(case["rows"] * (case["V"] * e + 8)), "flops": 0.0}
    B, L, Hkv, D = (case[k] for k in ("B", "L", "Hkv", "D"))
    if case["kind"] == "append":
        rows = B * case["S"] * (0.75 if case["ragged"] and case["S"] > 1 else 1.0)
        return {"bytes": rows * Hkv * (8 * D + (4 if case["weights"] else 0)), "flops": 0.0}
    if case["kind"] == "decode":
        tokens = B * L * (0.625 if case["ragged"] else 1.0)              # what _inputs gives on average
        per = 4 * D + (8 if case["weights"] else 0)
        return {"bytes": tokens * Hkv * per + B * case["Hq"] * (4 * D + 4), "flops": 4.0 * tokens * case["Hq"] * D}
    tokens = B * 0.75 * L
    kept = min(tokens, B * case["budget"])
    return {"bytes": Hkv * (tokens * 4 + kept * (8 * D + 8)), "flops": 0.0}


# ---- the same in 64 bits ----------------------------------------------------------------------


def _exact_append(case, seed):
    s = _inputs(case, seed)
    Hq, Hkv, D, page = (case[k] for k in ("Hq", "Hkv", "D", "page"))
    k, v, w = s["k"].double(), s["v"].double(), s["weight"]
    w = None if w is None else w.double()
    n = [case["S"]] * case["B"] if s["n_new"] is None else s["n_new"].tolist()
    for b, first in enumerate(s["start"].tolist()):
        x = s["qkv"][b, :n[b]].double().reshape(n[b], Hq + 2 * Hkv, D // 32, 32)
        at = torch.arange(first, first + n[b], device="cuda")
        pages = s["tables"][0][b].long()[at // page]
        for h in range(Hkv):
            k[pages, h, at % page // 32, :, at % 32] = x[:, Hq + h]
            v[pages, h, at % page // 32, :, :, at % 32] = x[:, Hq + Hkv + h]
        if w is not None:
            w[b, :, first:first + n[b]] = 0
    out = {"k": k, "v": v, "len": s["start"] + torch.tensor(n, dtype=torch.int32, device="cuda")}
    return out if w is None else {**out, "weight": w}


def _tokens(x, pages, head, n, v):
    """The first n keys (values) of one head of a sequence, 64 bits: [n, D]."""
    x = x[pages, head].double()                      # [pages, page/32, D/32, 32, 32]
    x = x.transpose(3, 4) if v else x
    return x.transpose(2, 3).reshape(-1, x.shape[2] * 32)[:n]


def _exact_decode(case, seed):
    s = _inputs(case, seed)
    B, Hq, Hkv, D = (case[k] for k in ("B", "Hq", "Hkv", "D"))
    if B * Hkv > 4096:
        return None
    G, table = Hq // Hkv, s["tables"][0].long()
    o = torch.zeros((B, Hq, D), dtype=torch.float64, device="cuda")
    lse = torch.full((B, Hq), -math.inf, dtype=torch.float64, device="cuda")
    w = None if s["weight"] is None else s["weight"].double()
    for b, n in enumerate(s["len"].tolist()):
        q = s["qkv"][b, 0].double()[:Hq * D].reshape(Hkv, G, D)
        for h in range(Hkv if n else 0):
            x = q[h] @ _tokens(s["k"], table[b], h, n, False).T / math.sqrt(D)
            L = torch.logsumexp(x, 1)
            p = torch.exp(x - L[:, None])
            o[b, h * G:(h + 1) * G], lse[b, h * G:(h + 1) * G] = p @ _tokens(s["v"], table[b], h, n, True), L
            if w is not None:
                w[b, h, :n] += p.sum(0)
    out = {"o": o.reshape(B, Hq * D), "lse": lse}
    return out if w is None else {**out, "weight": w}


def _exact_evict(case, seed):
    s = _inputs(case, seed)
    B, Hkv, D, page, budget = (case[k] for k in ("B", "Hkv", "D", "page", "budget"))
    k, v, wo = s["k"].double(), s["v"].double(), s["weight_out"].double()
    kept = torch.full((B, Hkv, budget), -1, dtype=torch.int32, device="cuda")
    src, dst = (t.long() for t in s["tables"])
    for b, n in enumerate(s["len"].tolist()):
        for h in range(Hkv):
            w = s["weight"][b, h, :n].double()
            idx = torch.arange(n, device="cuda")
            if n > budget:
                mid = idx[case["sink"]:n - case["recent"]]
                top = mid[torch.sort(-w[mid], stable=True).indices[:budget - case["sink"] - case["recent"]]]
                idx = torch.cat((idx[:case["sink"]], torch.sort(top).values, idx[n - case["recent"]:]))
            c = idx.numel()
            kept[b, h, :c] = idx.to(torch.int32)
            wo[b, h, :c] = w[idx]
            at = torch.arange(c, device="cuda")
            pg, tile, r = dst[b, at // page], at % page // 32, at % 32
            k[pg, h, tile, :, r] = _tokens(s["k"], src[b], h, n, False)[idx].reshape(c, D // 32, 32)
            v[pg, h, tile, :, :, r] = _tokens(s["v"], src[b], h, n, True)[idx].reshape(c, D // 32, 32)
    return {"kept": kept, "k": k, "v": v, "len": s["len"].clamp(max=budget), "weight": wo}


def _exact_sample(case, seed):
    s = _inputs(case, seed)
    got = []
    for r in range(case["rows"]):
        x = s["logits"][r].double()
        t = float(s["temperature"][r])
        if t <= 0:
            got.append(int(torch.nonzero(x == x.max())[0]))
            continue
        p = torch.softmax(x / t, 0)
        keep = torch.sort(-x, stable=True).indices
        if case["k"]:
            keep = keep[:int(s["top_k"][r])]
        if case["p"]:
            run = torch.cumsum(p[keep], 0) / p[keep].sum()
            keep = keep[:1 + int((run < float(s["top_p"][r])).sum())]
        if case["mp"]:
            keep = keep[p[keep] >= float(s["min_p"][r]) * p.max()]
        keep = torch.sort(keep).values
        run = torch.cumsum(p[keep], 0)
        got.append(int(keep[min(len(keep) - 1, int((run <= float(s["u"][r]) * run[-1]).sum()))]))
    return {"token": torch.tensor(got, dtype=torch.int32, device="cuda")}


def exact(case, seed):
    """What run() returns for these inputs, in 64 bits."""
    return {"append": _exact_append, "decode": _exact_decode, "evict": _exact_evict, "sample": _exact_sample}[case["kind"]](case, seed)
