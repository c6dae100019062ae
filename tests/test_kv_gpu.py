"""The paged key-value cache on the GPU: append, attention of one new token, eviction, against the operators in 64
bits (kv_cases.py has the bounds).  Moves are compared bit for bit."""
import math

import pytest
import torch

from kv_cases import DT, Case, blocks, check_decode, dense, evict_ref

pytestmark = pytest.mark.gpu

LENS = {
    "one": [1], "edges": [0, 1, 31, 32, 33, 63, 64, 65], "empty": [0, 0, 0], "ragged": [700, 0, 1, 2049, 513, 96],
    "long": [5003], "two": [4097, 40], "many": [(37 * i) % 301 for i in range(150)], "wide": [1300 + i for i in range(9)],
}


def q_of(case, Hq, seed=7, packed=False, mul=1.0):
    W = (Hq + (2 * case.Hkv if packed else 0)) * case.D
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(case.B, W, generator=g) * mul).to(DT[case.dtype]).to(case.dev)


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("Hq,Hkv,D,page,dtype", [
    (4, 4, 64, 32, "f16"), (8, 2, 128, 64, "bf16"), (32, 2, 128, 128, "f16"), (3, 1, 64, 256, "bf16"),
    (40, 1, 64, 64, "f16"), (34, 2, 128, 32, "bf16"), (100, 1, 64, 64, "f16"), (130, 2, 128, 128, "bf16")])
def test_decode(gpu, lens, Hq, Hkv, D, page, dtype):
    from tokamak_amd import attn
    print(f"[case] {lens} Hq{Hq} Hkv{Hkv} D{D} page{page} {dtype}", flush=True)
    case = Case(gpu, LENS[lens], Hkv, D, page, dtype, weights=True)
    q = q_of(case, Hq, packed=True)
    o, lse = attn.gqa_decode(q, case.cache, Hq)
    check_decode(case, q[:, :Hq * D], o, lse, Hq)
    assert torch.equal(case.cache.weight.cpu(), case.weight)
    again = attn.gqa_decode(q[:, :Hq * D], case.cache, Hq)
    assert torch.equal(o, again[0]) and torch.equal(lse, again[1])
    o, lse = attn.gqa_decode(q, case.cache, Hq, add_weights=True)      # may split the rows in another way
    check_decode(case, q[:, :Hq * D], o, lse, Hq)


@pytest.mark.parametrize("Hq,Hkv,D,page,dtype", [(4, 4, 64, 32, "f16"), (8, 2, 128, 64, "bf16"), (20, 1, 128, 128, "f16"), (70, 1, 64, 32, "bf16")])
@pytest.mark.parametrize("lens", ["edges", "ragged", "long", "many"])
def test_weights(gpu, lens, Hq, Hkv, D, page, dtype):
    from tokamak_amd import attn
    case = Case(gpu, LENS[lens], Hkv, D, page, dtype, weights=True)
    q = q_of(case, Hq)
    o, lse = attn.gqa_decode(q, case.cache, Hq, add_weights=True)
    w = check_decode(case, q, o, lse, Hq)
    got = case.cache.weight.cpu().double()
    for b, n in enumerate(case.lens):
        ref = case.weight[b, :, :n].double() + w[b]
        # each exponential within 1e-4 (kv_cases' bound of a score, twice, is below that here), one rounding of the sum
        assert ((got[b, :, :n] - ref).abs() <= 1e-4 * w[b] + 2.0 ** -23 * ref).all()
        assert torch.equal(got[b, :, n:], case.weight[b, :, n:].double())


@pytest.mark.parametrize("B,S,lens,Hq,Hkv,D,page,dtype", [
    (3, 1, [0, 31, 200], 4, 2, 64, 32, "f16"), (2, 77, [5, 64], 2, 2, 128, 64, "bf16"), (4, 33, [0, 1, 32, 95], 6, 3, 64, 32, "f16"),
    (1, 300, [130], 8, 1, 128, 256, "bf16"), (5, 2, [31, 63, 64, 0, 7], 4, 4, 128, 32, "f16")])
@pytest.mark.parametrize("ragged", [0, 1])
@pytest.mark.parametrize("given", [0, 1])
def test_append(gpu, B, S, lens, Hq, Hkv, D, page, dtype, ragged, given):
    from tokamak_amd import attn
    pages = max((n + S + page - 1) // page for n in lens)
    case = Case(gpu, [pages * page] * B, Hkv, D, page, dtype, extra_pages=0, weights=True)
    c = case.cache
    n_new = torch.tensor([(S * (b + 1)) // B for b in range(B)], dtype=torch.int32, device=gpu) if ragged else None
    if ragged and B > 1:
        n_new[0] = 0
    start = torch.tensor(lens, dtype=torch.int32, device=gpu)
    if not given:
        c.kv_len.copy_(start)
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(B, S, (Hq + 2 * Hkv) * D, generator=g).to(DT[dtype])
    attn.kv_append(qkv.to(gpu), c, Hq, start=start if given else None, n_new=n_new)
    n = [S] * B if n_new is None else n_new.tolist()
    assert c.kv_len.tolist() == [a + b for a, b in zip(lens, n)]
    x = qkv.double().reshape(B, S, Hq + 2 * Hkv, D)
    for b in range(B):
        k, v, w = case.k[b].clone(), case.v[b].clone(), case.weight[b].clone()
        at = slice(lens[b], lens[b] + n[b])
        k[:, at], v[:, at], w[:, at] = x[b, :n[b], Hq:Hq + Hkv].transpose(0, 1), x[b, :n[b], Hq + Hkv:].transpose(0, 1), 0
        t = c.table[b].long()
        assert torch.equal(dense(c.k[t].cpu().double(), False), k) and torch.equal(dense(c.v[t].cpu().double(), True), v)
        assert torch.equal(c.weight[b].cpu(), w)


@pytest.mark.parametrize("lens,Hkv,D,page,dtype,budget,sink,recent", [
    ([300, 100, 0, 257], 2, 64, 32, "f16", 100, 4, 20), ([513, 512, 1], 1, 128, 64, "bf16", 512, 0, 0),
    ([90, 33], 3, 64, 32, "f16", 32, 16, 16), ([1500], 2, 128, 128, "f16", 1, 0, 1), ([1500, 1200], 1, 64, 256, "bf16", 700, 700, 0),
    ([9500, 40000], 1, 64, 256, "f16", 5000, 3, 100), ([1400], 1, 64, 32, "bf16", 1399, 0, 300)])
@pytest.mark.parametrize("in_place", [0, 1])
@pytest.mark.parametrize("kind", ["random", "ties", "odd"])
def test_evict(gpu, lens, Hkv, D, page, dtype, budget, sink, recent, in_place, kind):
    from tokamak_amd import attn
    print(f"[case] {lens} budget {budget} sink {sink} recent {recent} in_place {in_place} {kind}", flush=True)
    B, pages = len(lens), (budget + page - 1) // page
    case = Case(gpu, lens, Hkv, D, page, dtype, spare=B * pages + 1, weights=True)
    c, w = case.cache, case.weight
    if kind == "ties":
        w = (w * 4).floor() / 4
    if kind == "odd":
        odd = torch.tensor([float("nan"), float("inf"), -float("inf"), -0.0, 0.0, -1.5, 1e-40, 3e38])
        w = odd[(w * 8).long()]
    c.weight.copy_(w)
    before = [x.clone() for x in (c.k, c.v, c.weight, c.kv_len)]
    if in_place:
        d = c
        kept = attn.kv_evict(c, budget, sink, recent)
    else:
        table = case.free[:B * pages].reshape(B, pages).to(torch.int32).to(gpu)
        d = attn.KvCache(c.k, c.v, table, torch.full((B,), 77, dtype=torch.int32, device=gpu), torch.full((B, Hkv, pages * page), -7.0, device=gpu))
        kept = attn.kv_evict(c, budget, sink, recent, dst=d)
        assert torch.equal(c.kv_len, before[3]) and torch.equal(c.weight.nan_to_num(123.0), before[2].nan_to_num(123.0))
    kept = kept.cpu()
    assert d.kv_len.tolist() == [min(n, budget) for n in lens]
    moved = [x.clone() for x in before[:2]]
    for b, n in enumerate(lens):
        for h in range(Hkv):
            ref = evict_ref(w[b, h].tolist(), n, budget, sink, recent)
            assert kept[b, h].tolist() == ref + [-1] * (budget - len(ref))
            at, new = torch.tensor(ref, dtype=torch.long), torch.arange(len(ref))
            assert torch.equal(d.weight[b, h, :len(ref)].cpu().view(torch.int32), w[b, h, at].view(torch.int32))
            tail = before[2][b, h, len(ref):] if in_place else torch.full_like(d.weight[b, h, len(ref):], -7.0)
            assert torch.equal(d.weight[b, h, len(ref):].view(torch.int32), tail.view(torch.int32))
            pg = d.table[b].cpu().long()[new // page]
            for m, x, isv in ((moved[0], case.k, False), (moved[1], case.v, True)):
                y = x[b][h, at].to(DT[dtype]).reshape(len(ref), D // 32, 32).to(gpu)
                if isv:
                    m[pg, h, new % page // 32, :, :, new % 32] = y
                else:
                    m[pg, h, new % page // 32, :, new % 32] = y
    # every other value of the pool is as it was, NaN and infinities included
    assert torch.equal(c.k.view(torch.int16), moved[0].view(torch.int16)) and torch.equal(c.v.view(torch.int16), moved[1].view(torch.int16))
