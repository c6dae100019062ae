"""The operators of a serving step over the paged key-value cache, as timed and compared cases: pages and
slots for the rows of a step, rotary positions, the append of packed rows, and the attention of several
new tokens a sequence over the cache.

Kinds and their fields:
  plan    B, L, S, Hkv, D, page, mix, tight: sequences of up to L tokens ask for up to S rows each (mix: all but a
          few ask for one); some have ended and give their pages back; tight: fewer pages than asked for
  rope    rows, Hq, Hkv, D, rot, layout, scaling, far, dtype, bwd: rows at positions up to `far`, or (bwd) their
          gradients
  append  B, L, S, Hq, Hkv, D, page, mix, dtype, rot, layout, scaling, weights: packed rows go behind up to L
          cached tokens a sequence, Q and K rotated (rot 0: not rotated)
  chunk   B, L, S, Hq, Hkv, D, page, mix, dtype, causal, window: up to S new tokens a sequence attend over the
          up to L that were there and themselves

Layout of the cache: pages of `page` tokens in 32 x 32 blocks, K [pages, Hkv, page/32, D/32, 32 tokens, 32 dims]
and V [pages, Hkv, page/32, D/32, 32 dims, 32 tokens]; table [B, max_pages] names a sequence's pages.  Rows of
a step are packed, sequence after sequence; row_start holds where each begins.  What lies behind the last
sequence's rows stays as it was.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # a decoding step of a batch: a row each, few new pages: latency
        {"name": "plan-step", "kind": "plan", "B": 64, "L": 4096, "S": 1, "Hkv": 1, "D": 64, "page": 64, "mix": 0, "tight": 0},
        # a busy server: many sequences decode, some bring prompts, and the pool runs out
        {"name": "plan-prompts", "kind": "plan", "B": 600, "L": 8000, "S": 2000, "Hkv": 1, "D": 64, "page": 32, "mix": 1, "tight": 1},
        # a decoding step far out in a long context
        {"name": "rope-step", "kind": "rope", "rows": 64, "Hq": 32, "Hkv": 8, "D": 128, "rot": 128, "layout": "halves",
         "scaling": "yarn", "far": 1000000, "dtype": "bf16", "bwd": 0},
        # the training batch of the headline attention shape
        {"name": "rope-train", "kind": "rope", "rows": 8192, "Hq": 16, "Hkv": 16, "D": 128, "rot": 128, "layout": "pairs",
         "scaling": "none", "far": 2048, "dtype": "f16", "bwd": 0},
        # its gradient with grouped heads, where a part of the head is rotated
        {"name": "rope-grad", "kind": "rope", "rows": 16384, "Hq": 32, "Hkv": 4, "D": 64, "rot": 40, "layout": "halves",
         "scaling": "bands", "far": 32768, "dtype": "bf16", "bwd": 1},
        # a decoding step's rows into the cache
        {"name": "append-step", "kind": "append", "B": 64, "L": 4000, "S": 1, "Hq": 32, "Hkv": 8, "D": 128, "page": 64,
         "mix": 0, "dtype": "bf16", "rot": 128, "layout": "halves", "scaling": "bands", "weights": 0},
        # prompts of several users, their weights for a later eviction cleared
        {"name": "append-prompts", "kind": "append", "B": 7, "L": 3000, "S": 2900, "Hq": 20, "Hkv": 4, "D": 128, "page": 128,
         "mix": 0, "dtype": "f16", "rot": 64, "layout": "pairs", "scaling": "ntk", "weights": 1},
        # a draft of a few tokens checked for each of a few short chats: latency
        {"name": "chunk-draft", "kind": "chunk", "B": 4, "L": 500, "S": 5, "Hq": 8, "Hkv": 4, "D": 64, "page": 32, "mix": 0,
         "dtype": "f16", "causal": 1, "window": 0},
        # a question of a few tokens about one very long document
        {"name": "chunk-one-long", "kind": "chunk", "B": 1, "L": 131000, "S": 13, "Hq": 32, "Hkv": 8, "D": 128, "page": 256,
         "mix": 0, "dtype": "bf16", "causal": 1, "window": 0},
        # a serving step: most sequences decode, a few bring pieces of their prompts
        {"name": "chunk-mixed", "kind": "chunk", "B": 48, "L": 6000, "S": 512, "Hq": 32, "Hkv": 8, "D": 128, "page": 64,
         "mix": 1, "dtype": "bf16", "causal": 1, "window": 0},
        # long prompts, the second half of each
        {"name": "chunk-prompts", "kind": "chunk", "B": 2, "L": 5000, "S": 4096, "Hq": 32, "Hkv": 8, "D": 128, "page": 128,
         "mix": 0, "dtype": "f16", "causal": 1, "window": 0},
        # prompts of a model with windowed layers and as many key heads as query heads
        {"name": "chunk-window", "kind": "chunk", "B": 5, "L": 9000, "S": 1300, "Hq": 12, "Hkv": 12, "D": 64, "page": 64,
         "mix": 0, "dtype": "bf16", "causal": 1, "window": 1024},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choices(("plan", "rope", "append", "chunk"), (2, 3, 3, 5))[0]
    while True:
        d = rng.choice((64, 128))
        c = {"kind": kind, "D": d, "Hkv": rng.choice((1, 2, 4, 8, 16))}
        rotary = {"rot": rng.choice((d, d // 2, 2 * rng.randint(1, d // 2))), "layout": rng.choice(("halves", "pairs")),
                  "scaling": rng.choice(("none", "linear", "ntk", "bands", "yarn"))}
        if kind == "rope":
            c.update(rotary, rows=_log_int(rng, 1, 32768), Hq=c["Hkv"] * rng.choice((1, 2, 4, 8)), far=_log_int(rng, 16, 1 << 22),
                     dtype=rng.choice(("f16", "bf16")), bwd=rng.randint(0, 1))
            if c["rows"] * (c["Hq"] + 2 * c["Hkv"]) * d <= 5e7:
                return c
            continue
        c.update(B=_log_int(rng, 1, 600), L=_log_int(rng, 1, 131072), S=rng.choice((1, _log_int(rng, 1, 4096))),
                 page=rng.choice((32, 64, 128, 256)))
        c["mix"] = int(c["B"] > 3 and c["S"] > 1 and rng.random() < 0.5)
        asked = c["B"] * c["S"] * (0.15 if c["mix"] else 1)
        if kind == "plan":
            c.update(Hkv=1, D=64, tight=rng.randint(0, 1))
            if asked <= 1 << 17 and c["B"] * (c["L"] + c["S"]) <= 1 << 23:
                return c
            continue
        c.update(Hq=c["Hkv"] * rng.choice((1, 2, 3, 4, 8, 16)), dtype=rng.choice(("f16", "bf16")))
        if c["Hq"] > 64 or c["B"] * (c["L"] + c["S"]) * c["Hkv"] * d > 1 << 26:
            continue
        if kind == "append":
            c.update(rotary, weights=rng.randint(0, 1))
            if rng.random() < 0.2:
                c["rot"] = 0
            if asked * (c["Hq"] + 2 * c["Hkv"]) * d <= 5e7:
                return c
            continue
        c["causal"] = int(rng.random() < 0.85)
        c["window"] = rng.choice((0, 0, _log_int(rng, 1, 8192))) if c["causal"] else 0
        if asked * (c["L"] + c["S"] / 2) * c["Hq"] * d <= 1.5e11:
            return c


# ---- inputs ---------------------------------------------------------------------------------


def _gen(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 64 + salt)
    return g


def _randn(shape, seed, salt, mul, dtype):
    x = torch.randn(shape, generator=_gen(seed, salt), device="cuda", dtype=dtype)
    return x if mul == 1.0 else x * mul


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _pages(n, page):
    return (n + page - 1) // page


def _requests(case, seed):
    """Host lists of a step: tokens that each sequence has, rows that it brings, and pages that it holds.  The
    case decides on the requests, the seed on their order."""
    rng = random.Random("requests")
    B, L, S = case["B"], case["L"], case["S"]
    have = [L] + [rng.randint(L // 4, L) for _ in range(B - 1)]
    rows = [S] + [rng.randint((S + 1) // 2, S) for _ in range(B - 1)]
    if case["mix"]:
        rows = [n if i % 8 == 0 else 1 for i, n in enumerate(rows)]
    if B >= 8:
        rows[B // 2] = 0                 # a sequence that sits this step out
        have[B // 3] = 0                 # one that begins
    held = [_pages(n, case["page"]) for n in have]
    if case["kind"] == "plan":
        for b in range(3, B, 7):         # ended: no tokens are left, the pages go back
            have[b], rows[b] = 0, 0
    order = list(range(B))
    random.Random(f"order {seed}").shuffle(order)
    return [[x[b] for b in order] for x in (have, rows, held)]


def _inputs(case, seed):
    kind = case["kind"]
    if kind == "rope":
        rng, far = random.Random(f"rows {seed}"), case["far"]
        C = (case["Hq"] + 2 * case["Hkv"]) * case["D"]
        at = torch.randint(0, far, (case["rows"],), generator=_gen(seed, 1), device="cuda").to(torch.int32)
        at[rng.randrange(case["rows"])] = far - 1
        if case["rows"] > 64:            # rows of whole sequences, as in training
            at = ((torch.arange(case["rows"], device="cuda") + rng.randrange(far)) % far).to(torch.int32)
        return {"x": _randn((case["rows"], C), seed, 2, 1.0, DT[case["dtype"]]), "pos": at}
    B, L, S, Hkv, D, page = (case[k] for k in ("B", "L", "S", "Hkv", "D", "page"))
    have, rows, held = _requests(case, seed)
    total, most = sum(rows), _pages(L + S, page)
    s = {"have": have, "n": rows, "start": _i32(have)}
    if kind == "plan":
        need = sum(max(0, _pages(h + n, page) - c) for h, n, c in zip(have, rows, held))
        spare = need // 2 if case["tight"] else need + 5
        num = sum(held) + spare
        ids = list(range(num))
        random.Random(f"pages {seed}").shuffle(ids)
        table, used = [], 0
        for c in held:
            table.append(ids[used:used + c] + [-1] * (most - c))
            used += c
        s["want"], s["num_pages"], s["rows"] = _i32(rows), num, total + 3
        s["table"], s["held"] = _i32(table), _i32(held)
        s["free"], s["n_free"] = _i32(ids[used:] + [-1] * used), _i32([spare])
        s["len"] = torch.zeros(B, dtype=torch.int32, device="cuda")
        # K and V are not touched: what plans is the table
        s["k"], s["v"] = (torch.zeros((num, Hkv, page // 32, D // 32, 32, 32), dtype=torch.float16, device="cuda") for _ in range(2))
        return s
    dt, num = DT[case["dtype"]], sum(_pages(h + n, page) for h, n in zip(have, rows)) + 1
    perm = torch.randperm(num, generator=_gen(seed, 3), device="cuda").to(torch.int32)
    s["table"] = torch.full((B, most), -1, dtype=torch.int32, device="cuda")
    used = 0
    for b, (h, n) in enumerate(zip(have, rows)):
        c = _pages(h + n, page)
        s["table"][b, :c] = perm[used:used + c]
        used += c
    s["len"] = _i32([h + n for h, n in zip(have, rows)])
    s["n_new"] = _i32(rows)
    ends = torch.cumsum(s["n_new"], 0).to(torch.int32)
    s["row_start"] = torch.cat((torch.zeros_like(ends[:1]), ends))
    blocks, R = (num, Hkv, page // 32, D // 32, 32, 32), total + 3           # three rows behind the last sequence's
    s["k"], s["v"] = _randn(blocks, seed, 4, 1.0, dt), _randn(blocks, seed, 5, 1.0, dt)
    s["qkv"] = _randn((R, (case["Hq"] + 2 * Hkv) * D), seed, 6, 1.5 if kind == "chunk" else 1.0, dt)
    if kind == "append":
        r = torch.arange(R, device="cuda")
        seq = torch.searchsorted(ends.long(), r, right=True).clamp(max=B - 1)
        pos = s["start"].long()[seq] + r - s["row_start"].long()[seq]
        slot = s["table"].long()[seq, (pos // page).clamp(max=most - 1)] * page + pos % page
        behind = r >= total
        s["seq"], s["pos"] = (torch.where(behind, -1, x).to(torch.int32) for x in (seq, pos))
        s["slot"] = torch.where(behind, -1, slot)
        s["weight"] = torch.rand((B, Hkv, most * page), generator=_gen(seed, 7), device="cuda") if case["weights"] else None
        s["q"] = torch.zeros((R, case["Hq"] * D), dtype=dt, device="cuda")
    else:
        s["o"] = torch.zeros((R, case["Hq"] * D), dtype=dt, device="cuda")
        s["lse"] = torch.zeros((R, case["Hq"]), device="cuda")
    return s


# A context of 8192 trained positions, four times longer.
THETA, SCALE, TRAINED, LOW, HIGH, SLOW, FAST = 10000.0, 4.0, 8192.0, 1.0, 4.0, 1.0, 32.0


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case.get("rot"):
        s["freq"], s["factor"] = _freqs(case)
    if own:
        from tokamak_amd import attn
        if case.get("rot"):
            s["rope"] = attn.Rope(case["rot"], layout=case["layout"], theta=THETA,
                                  **{"none": {}, "linear": {"scaling": "linear", "scale": SCALE},
                                     "ntk": {"scaling": "ntk", "scale": SCALE},
                                     "bands": {"scaling": "bands", "scale": SCALE, "original": TRAINED, "low": LOW, "high": HIGH},
                                     "yarn": {"scaling": "yarn", "scale": SCALE, "original": TRAINED, "low": SLOW, "high": FAST}}
                                  [case["scaling"]])
        if case["kind"] != "rope":
            s["cache"] = attn.KvCache(s["k"], s["v"], s["table"], s["len"], s.get("weight"))
        if case["kind"] == "plan":
            s["pages"] = attn.KvPages(s["free"], s["n_free"], s["held"])
            s["plan"] = attn.KvPlan.empty(case["B"], s["rows"])
        if case["kind"] == "append":
            s["plan"] = attn.KvPlan(s["n_new"], s["row_start"], s["seq"], s["pos"], s["slot"])
    return s


# ---- the passes -----------------------------------------------------------------------------


def _plain_plan(s, case):
    page, start, want, rows, num = case["page"], s["start"].long(), s["want"].long(), s["rows"], s["num_pages"]
    table, held, most = s["table"], s["held"].long(), s["table"].shape[1]
    valid = (start >= 0) & (start <= most * page)
    want = torch.where(valid & (start + want <= most * page), want.clamp(min=0), 0)
    target = (start + want + page - 1) // page
    back = torch.where(valid, (held - target).clamp(min=0), 0)
    need = torch.where(want > 0, (target - held).clamp(min=0), 0)
    n_free = s["n_free"].long()
    top = n_free + back.sum()
    n = torch.where((need == 0) | (need.cumsum(0) <= top), want, 0)
    n = torch.where(n.cumsum(0) <= rows, n, 0)
    take = torch.where(n > 0, need, 0)
    # released pages go on the stack, taken ones come off its top
    p = torch.arange(most, device="cuda")
    gone = (p >= target[:, None]) & (p < (target + back)[:, None])
    place = torch.where(gone, n_free + (back.cumsum(0) - back)[:, None] + p - target[:, None], num)
    free = torch.cat((s["free"], s["free"][:1]))
    free.scatter_(0, place.reshape(-1), table.reshape(-1))
    new = (p >= held[:, None]) & (p < (held + take)[:, None])
    place = torch.where(new, top - 1 - ((take.cumsum(0) - take)[:, None] + p - held[:, None]), 0)
    table.copy_(torch.where(new, free[place], torch.where(gone, -1, table)))
    s["free"].copy_(free[:num])
    s["n_free"].copy_(top - take.sum())
    s["held"].copy_(held - back + take)
    s["len"].copy_(s["start"] + n)
    ends = n.cumsum(0)
    r = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(ends, r, right=True)
    behind = seq >= case["B"]
    seq = seq.clamp(max=case["B"] - 1)
    pos = start[seq] + r - (ends - n)[seq]
    at = table[seq, (pos // page).clamp(max=most - 1)].long()
    slot = torch.where(behind | (at < 0) | (at >= num), -1, at * page + pos % page)
    return {"table": table, "free": s["free"], "n_free": s["n_free"], "held": s["held"], "len": s["len"],
            "n_new": n.to(torch.int32), "row_start": torch.cat((torch.zeros_like(ends[:1]), ends)).to(torch.int32),
            "seq": torch.where(behind, -1, seq).to(torch.int32), "pos": torch.where(behind, -1, pos).to(torch.int32), "slot": slot}


def _freqs(case):
    """Angle of each pair a position, and what the rotated dims are multiplied by."""
    rot, kind, theta, factor = case["rot"], case["scaling"], THETA, 1.0
    if kind == "ntk" and rot > 2:
        theta *= SCALE ** (rot / (rot - 2))
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    f = theta ** (-2.0 * i / rot)
    if kind == "linear":
        f = f / SCALE
    if kind == "bands":
        turns = TRAINED * f / (2 * math.pi)
        f = torch.lerp(f / SCALE, f, ((turns - LOW) / (HIGH - LOW)).clamp(0, 1))
    if kind == "yarn":
        lo, hi = (rot * math.log(TRAINED / (2 * math.pi * t)) / (2 * math.log(theta)) for t in (FAST, SLOW))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), rot - 1)
        f = torch.lerp(f, f / SCALE, ((i - lo) / (hi - lo if hi > lo else 0.001)).clamp(0, 1))
        factor = 0.1 * math.log(SCALE) + 1.0
    return f, factor


def _plain_rotate(x, pos, s, case, sign):
    """x [rows, heads, D] in fp32, its first `rot` dims rotated."""
    rot, a = case["rot"], pos.double()[:, None, None] * s["freq"]
    c, sn = (torch.cos(a) * s["factor"]).float(), (torch.sin(a) * (s["factor"] * sign)).float()
    i = torch.arange(rot // 2, device="cuda")
    i0, i1 = (i, i + rot // 2) if case["layout"] == "halves" else (2 * i, 2 * i + 1)
    x0, x1 = x[..., i0], x[..., i1]
    y = x.clone()
    y[..., i0], y[..., i1] = x0 * c - x1 * sn, x0 * sn + x1 * c
    return y


def _plain_rope(s, case):
    R, Hq, Hkv, D = (case[k] for k in ("rows", "Hq", "Hkv", "D"))
    x = s["x"].reshape(R, Hq + 2 * Hkv, D)
    y = _plain_rotate(x[:, :Hq + Hkv].float(), s["pos"], s, case, -1.0 if case["bwd"] else 1.0).to(x.dtype)
    return torch.cat((y, x[:, Hq + Hkv:]), 1).reshape(R, -1)


def _plain_append(s, case):
    Hq, Hkv, D, page = (case[k] for k in ("Hq", "Hkv", "D", "page"))
    n = sum(s["n"])
    x = s["qkv"][:n].reshape(n, Hq + 2 * Hkv, D)
    qk = x[:, :Hq + Hkv]
    if case["rot"]:
        qk = _plain_rotate(qk.float(), s["pos"][:n], s, case, 1.0).to(x.dtype)
    s["q"][:n] = qk[:, :Hq].reshape(n, -1)
    slot = s["slot"][:n]
    at, tile, r = slot // page, slot % page // 32, slot % 32
    s["k"][at, :, tile, :, r, :] = qk[:, Hq:].reshape(n, Hkv, D // 32, 32)
    s["v"][at, :, tile, :, :, r] = x[:, Hq + Hkv:].reshape(n, Hkv, D // 32, 32)
    if s["weight"] is not None:
        s["weight"][s["seq"][:n].long(), :, s["pos"][:n].long()] = 0.0


def _plain_chunk(s, case):
    Hq, Hkv, D, page = (case[k] for k in ("Hq", "Hkv", "D", "page"))
    G, first = Hq // Hkv, 0
    for b, (had, n) in enumerate(zip(s["have"], s["n"])):
        if n == 0:
            continue
        L = had + n
        pg = s["table"][b, :_pages(L, page)].long()
        k = s["k"][pg].float().permute(1, 0, 2, 4, 3, 5).reshape(Hkv, -1, D)[:, :L]
        v = s["v"][pg].float().permute(1, 0, 2, 5, 3, 4).reshape(Hkv, -1, D)[:, :L]
        q = s["qkv"][first:first + n, :Hq * D].float().reshape(n, Hkv, G, D).transpose(0, 1).reshape(Hkv, n * G, D)
        x = torch.matmul(q, k.transpose(1, 2).contiguous()).reshape(Hkv, n, G, L) * (1.0 / math.sqrt(D))
        if case["causal"]:
            p, j = torch.arange(had, L, device="cuda")[:, None], torch.arange(L, device="cuda")
            hidden = j > p
            if case["window"]:
                hidden |= j <= p - case["window"]
            x = x.masked_fill(hidden[:, None], -math.inf)
        m = x.amax(3, keepdim=True)
        x = torch.exp(x - m)
        total = x.sum(3, keepdim=True)
        o = torch.matmul(x.reshape(Hkv, n * G, L), v).reshape(Hkv, n, G, D) / total
        s["o"][first:first + n] = o.transpose(0, 1).reshape(n, Hq * D).to(s["o"].dtype)
        s["lse"][first:first + n] = (m + torch.log(total)).transpose(0, 1).reshape(n, Hq)
        first += n


def run(s):
    case, kind = s["case"], s["case"]["kind"]
    if own:
        from tokamak_amd import attn
    if kind == "plan":
        if not own:
            return _plain_plan(s, case)
        p = attn.kv_plan(s["cache"], s["pages"], s["want"], start=s["start"], plan=s["plan"])
        return {"table": s["table"], "free": s["free"], "n_free": s["n_free"], "held": s["held"], "len": s["len"],
                "n_new": p.n_new, "row_start": p.row_start, "seq": p.seq, "pos": p.pos, "slot": p.slot}
    if kind == "rope":
        if not own:
            return {"y": _plain_rope(s, case)}
        call = attn.rope_bwd if case["bwd"] else attn.rope_fwd
        return {"y": call(s["x"], s["rope"], case["Hq"], case["Hkv"], case["D"], pos=s["pos"])}
    if kind == "append":
        if own:
            attn.kv_append_rows(s["qkv"], s["cache"], case["Hq"], s["plan"], rope=s.get("rope"), q=s["q"])
        else:
            _plain_append(s, case)
        out = {"q": s["q"], "k": s["k"], "v": s["v"]}
        return out if s["weight"] is None else {**out, "weight": s["weight"]}
    if own:
        attn.gqa_chunk(s["qkv"], s["cache"], case["Hq"], row_start=s["row_start"], n_new=s["n_new"],
                       causal=bool(case["causal"]), window=case["window"], out=s["o"], lse=s["lse"])
    else:
        _plain_chunk(s, case)
    return {"o": s["o"], "lse": s["lse"]}


# ---- what a pass cannot do without ------------------------------------------------------------


def work(case):
    Hq, Hkv, D = case.get("Hq", 0), case["Hkv"], case["D"]
    if case["kind"] == "rope":
        return {"bytes": case["rows"] * (4.0 * (Hq + 2 * Hkv) * D + 4), "flops": 3.0 * case["rows"] * (Hq + Hkv) * case["rot"]}
    B, S, L = case["B"], case["S"], case["L"]
    each = [S] + [0.75 * S + 0.25] * (B - 1)               # what _requests gives on average
    if case["mix"]:
        each = [n if i % 8 == 0 else 1 for i, n in enumerate(each)]
    if B >= 8:
        each[B // 2] = 0
    rows = float(sum(each))
    if case["kind"] == "plan":
        share = 0.7 if case["tight"] else 1.0              # of the rows, what the pool has pages for, about
        return {"bytes": 28.0 * B + 16 * rows + 8 * share * rows / case["page"], "flops": 0.0}
    if case["kind"] == "append":
        per = 4 * (Hq + 2 * Hkv) * D + 16 + (4 * Hkv if case["weights"] else 0)
        return {"bytes": rows * per, "flops": 3.0 * rows * (Hq + Hkv) * case["rot"]}
    tokens = pairs = 0.0
    for i, n in enumerate(each):
        had = L if i == 0 else 0.625 * L
        if B >= 8 and i == B // 3:
            had = 0
        w = case["window"] or had + n
        tokens += min(had + n, w + n) if n else 0
        pairs += n * (min(had + n / 2, w) if case["causal"] else had + n)
    return {"bytes": tokens * Hkv * D * 4 + rows * Hq * (4 * D + 4), "flops": 4.0 * pairs * Hq * D}


# ---- the same in 64 bits ----------------------------------------------------------------------


def _exact_plan(case, seed):
    s = _inputs(case, seed)
    page, most, num, rows = case["page"], s["table"].shape[1], s["num_pages"], s["rows"]
    table, free, held = (s[k].tolist() for k in ("table", "free", "held"))
    start, want, top = s["start"].tolist(), s["want"].tolist(), int(s["n_free"])
    goal = [-(-(h + n) // page) for h, n in zip(start, want)]
    for b in range(case["B"]):
        for p in range(goal[b], held[b]):
            free[top], table[b][p], top = table[b][p], -1, top + 1
        held[b] = min(held[b], goal[b])
    pool, asked, used, n_new = top, 0, 0, []
    for b in range(case["B"]):
        need = goal[b] - held[b] if want[b] else 0
        asked += need
        n = want[b] if need == 0 or asked <= pool else 0
        used += n
        n_new.append(n if used <= rows else 0)
        for _ in range(need if n_new[b] else 0):
            top -= 1
            table[b][held[b]], held[b] = free[top], held[b] + 1
    seq = [b for b, n in enumerate(n_new) for _ in range(n)]
    pos = [start[b] + i for b, n in enumerate(n_new) for i in range(n)]
    slot = [table[b][p // page] * page + p % page for b, p in zip(seq, pos)]
    first = [0]
    for n in n_new:
        first.append(first[-1] + n)
    pad = [-1] * (rows - len(seq))
    return {"table": _i32(table), "free": _i32(free), "n_free": _i32([top]), "held": _i32(held),
            "len": _i32([h + n for h, n in zip(start, n_new)]), "n_new": _i32(n_new), "row_start": _i32(first),
            "seq": _i32(seq + pad), "pos": _i32(pos + pad), "slot": torch.tensor(slot + pad, dtype=torch.int64, device="cuda")}


def _exact_turned(x, pos, case, back=False):
    """Rows of heads [rows, heads, D] as complex numbers times exp(i pos w), 64 bits."""
    rot, kind = case["rot"], case["scaling"]
    half, angle, grow = rot // 2, [], 1.0
    for i in range(half):
        w = THETA ** (-2 * i / rot)
        if kind == "linear":
            w /= SCALE
        elif kind == "ntk" and rot > 2:
            w = (THETA * SCALE ** (rot / (rot - 2))) ** (-2 * i / rot)
        elif kind == "bands":
            wave = 2 * math.pi / w
            if wave > TRAINED / LOW:
                w /= SCALE
            elif wave >= TRAINED / HIGH:
                t = (TRAINED / wave - LOW) / (HIGH - LOW)
                w = (1 - t) * w / SCALE + t * w
        elif kind == "yarn":
            def edge(turns):
                return rot * math.log(TRAINED / (turns * 2 * math.pi)) / (2 * math.log(THETA))
            a, b = max(math.floor(edge(FAST)), 0), min(math.ceil(edge(SLOW)), rot - 1)
            t = min(1.0, max(0.0, (i - a) / ((b - a) if b > a else 0.001)))
            w = w / SCALE * t + w * (1 - t)
            grow = 0.1 * math.log(SCALE) + 1.0
        angle.append(w)
    phase = pos.double()[:, None] * torch.tensor(angle, dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.full_like(phase, grow), -phase if back else phase)[:, None]
    y = x.double()
    part = y[..., :rot]
    if case["layout"] == "pairs":
        z = torch.view_as_complex(part.reshape(*part.shape[:-1], half, 2).contiguous()) * turn
        part = torch.view_as_real(z).reshape(part.shape)
    else:
        z = torch.complex(part[..., :half].contiguous(), part[..., half:].contiguous()) * turn
        part = torch.cat((z.real, z.imag), -1)
    return torch.cat((part, y[..., rot:]), -1)


def _exact_rope(case, seed):
    s = _inputs(case, seed)
    H = case["Hq"] + case["Hkv"]
    x = s["x"].reshape(case["rows"], -1, case["D"])
    return {"y": torch.cat((_exact_turned(x[:, :H], s["pos"], case, bool(case["bwd"])), x[:, H:].double()), 1).reshape(case["rows"], -1)}


def _exact_append(case, seed):
    s = _inputs(case, seed)
    Hq, Hkv, D, page = (case[k] for k in ("Hq", "Hkv", "D", "page"))
    k, v, q, w = s["k"].double(), s["v"].double(), s["q"].double(), s["weight"]
    w, first = None if w is None else w.double(), 0
    for b, (had, n) in enumerate(zip(s["have"], s["n"])):
        x = s["qkv"][first:first + n].reshape(n, Hq + 2 * Hkv, D)
        at = torch.arange(had, had + n, device="cuda")
        x = torch.cat((_exact_turned(x[:, :Hq + Hkv], at, case) if case["rot"] else x[:, :Hq + Hkv].double(), x[:, Hq + Hkv:].double()), 1)
        q[first:first + n] = x[:, :Hq].reshape(n, Hq * D)
        pg = s["table"][b].long()[at // page]
        for h in range(Hkv):
            k[pg, h, at % page // 32, :, at % 32] = x[:, Hq + h].reshape(n, D // 32, 32)
            v[pg, h, at % page // 32, :, :, at % 32] = x[:, Hq + Hkv + h].reshape(n, D // 32, 32)
        if w is not None:
            w[b, :, had:had + n] = 0
        first += n
    out = {"q": q, "k": k, "v": v}
    return out if w is None else {**out, "weight": w}


def _exact_chunk(case, seed):
    if case["B"] * case["Hkv"] > 4096:
        return None
    s = _inputs(case, seed)
    Hq, Hkv, D, page = (case[k] for k in ("Hq", "Hkv", "D", "page"))
    G, first = Hq // Hkv, 0
    o, lse = s["o"].double(), s["lse"].double()
    for b, (had, n) in enumerate(zip(s["have"], s["n"])):
        L, pg = had + n, s["table"][b].long()
        pg = pg[:_pages(L, page)]
        for h in range(Hkv if n else 0):
            k = s["k"][pg, h].double().transpose(2, 3).reshape(-1, D)[:L]
            v = s["v"][pg, h].double().permute(0, 1, 4, 2, 3).reshape(-1, D)[:L]
            for g in range(G):
                c = h * G + g
                for i in range(0, n, 2048):
                    m = min(2048, n - i)
                    x = s["qkv"][first + i:first + i + m, c * D:(c + 1) * D].double() @ k.T / math.sqrt(D)
                    if case["causal"]:
                        age = torch.arange(had + i, had + i + m, device="cuda")[:, None] - torch.arange(L, device="cuda")
                        x[(age < 0) | (age >= (case["window"] or L + 1))] = -math.inf
                    t = torch.logsumexp(x, 1)
                    o[first + i:first + i + m, c * D:(c + 1) * D] = torch.exp(x - t[:, None]) @ v
                    lse[first + i:first + i + m, c] = t
        first += n
    return {"o": o, "lse": lse}


def exact(case, seed):
    """What run() returns for these inputs, in 64 bits."""
    return {"plan": _exact_plan, "rope": _exact_rope, "append": _exact_append, "chunk": _exact_chunk}[case["kind"]](case, seed)
