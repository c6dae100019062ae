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
    "crowd": [(13 * i) % 100 for i in range(69)] + [0, 3000, 0, 65] + [1] * 60,
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
@pytest.mark.parametrize("lens", ["edges", "ragged", "long", "many", "crowd"])
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
    ([9500, 40000], 1, 64, 256, "f16", 5000, 3, 100), ([1400], 1, 64, 32, "bf16", 1399, 0, 300),
    ([2000], 2, 64, 32, "f16", 1800, 0, 0)])
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


@pytest.mark.parametrize("n,extra", [(2047, 0), (2048, 0), (2048, 1), (8191, 0), (8192, 0), (8193, 0), (16383, 0), (16384, 0), (16385, 3),
                                     (32768, 0), (49153, 0)])
@pytest.mark.parametrize("budget,sink,recent", [(33, 0, 0), (1500, 0, 1500), (1999, 1024, 64), (2000, 4, 1000)])
@pytest.mark.parametrize("weights", [0, 1])
def test_evict_chooses_at_the_sizes_of_its_chunks(gpu, n, extra, budget, sink, recent, weights):
    """Sequences as long as what a workgroup holds at a time, and one more or less; weights that are equal in crowds,
    the border's among them; with weights in the new cache and without."""
    from tokamak_amd import attn
    page = 64
    pages = (budget + page - 1) // page
    case = Case(gpu, [n, n - 5], 1, 64, page, "f16", spare=2 * pages, extra_pages=extra, weights=True)
    w = (case.weight * 40).floor() / 8 - 1
    case.cache.weight.copy_(w)
    d = attn.KvCache(case.cache.k, case.cache.v, case.free[:2 * pages].reshape(2, pages).to(torch.int32).to(gpu),
                     torch.zeros(2, dtype=torch.int32, device=gpu), torch.zeros((2, 1, pages * page), device=gpu) if weights else None)
    kept = attn.kv_evict(case.cache, budget, sink, recent, dst=d).cpu()
    assert d.kv_len.tolist() == [budget] * 2
    for b in range(2):
        ref = evict_ref(w[b, 0].tolist(), n - 5 * b, budget, sink, recent)
        assert kept[b, 0].tolist() == ref
        if weights:
            assert torch.equal(d.weight[b, 0, :budget].cpu(), w[b, 0, torch.tensor(ref)])


@pytest.mark.parametrize("Hq,Hkv,D,dtype", [(4, 2, 64, "f16"), (8, 1, 128, "bf16")])
@pytest.mark.parametrize("trend", [3.0, 12.0, -12.0])
@pytest.mark.parametrize("n", [190, 4500])
def test_scores_that_grow_or_fall_along_the_keys(gpu, Hq, Hkv, D, dtype, trend, n):
    """The running maximum moves again and again, or stays at the first tile while the rest fades."""
    from tokamak_amd import attn
    case = Case(gpu, [n, n // 2], Hkv, D, 64, dtype, trend=trend)
    q = q_of(case, Hq).abs()
    o, lse = attn.gqa_decode(q, case.cache, Hq)
    check_decode(case, q, o, lse, Hq)


@pytest.mark.parametrize("scale", [1e-6, 0.02, 3.0])
def test_scale(gpu, scale):
    from tokamak_amd import attn
    case = Case(gpu, [70, 1000], 2, 64, 32, "f16", weights=True)
    q = q_of(case, 4)
    o, lse = attn.gqa_decode(q, case.cache, 4, scale=scale, add_weights=True)
    check_decode(case, q, o, lse, 4, scale=float(torch.tensor(scale, dtype=torch.float32)))


def test_strides_and_given_buffers(gpu):
    from guarded import Guarded
    from tokamak_amd import attn
    case = Case(gpu, [100, 1, 700], 2, 128, 64, "bf16")
    wide = torch.full((3, 1400), float("nan"), dtype=torch.bfloat16, device=gpu)
    q = q_of(case, 8)
    wide[:, 16:16 + 8 * 128] = q
    o, lse = Guarded(3 * 8 * 128, torch.bfloat16, gpu), Guarded(3 * 8, torch.float32, gpu)
    ws = Guarded(attn.decode_workspace_bytes(case.cache, 8) + 16, torch.uint8, gpu)
    got = attn.gqa_decode(wide[:, 16:16 + 8 * 128], case.cache, 8, out=o.t.view(3, -1), lse=lse.t.view(3, 8), workspace=ws.t)
    check_decode(case, q, *got, 8)
    assert o.intact() and lse.intact() and ws.intact()
    ref = attn.gqa_decode(q, case.cache, 8)
    assert torch.equal(ref[0], got[0]) and torch.equal(ref[1], got[1])
    one = Case(gpu, [40], 1, 64, 32, "f16")
    q1 = q_of(one, 2)
    check_decode(one, q1, *attn.gqa_decode(q1.expand(1, -1), one.cache, 2), 2)
    with pytest.raises(ValueError):
        attn.gqa_decode(q[:2], case.cache, 8)
    with pytest.raises(ValueError):
        attn.gqa_decode(q.half(), case.cache, 8)
    with pytest.raises(ValueError):
        attn.gqa_decode(q[:, ::2], case.cache, 4)
    with pytest.raises(attn.AttnError):
        attn.gqa_decode(wide[:, 1:1 + 8 * 128], case.cache, 8)        # not on 16 bytes
    with pytest.raises(attn.AttnError):
        attn.gqa_decode(q[:1].expand(3, -1), case.cache, 8)           # a row for all: stride 0
    with pytest.raises(attn.AttnError):
        attn.gqa_decode(q, case.cache, 8, add_weights=True)           # the cache has none
    with pytest.raises(ValueError):
        attn.kv_append(q, case.cache, 8)                              # not packed QKV
    with pytest.raises(AttributeError):
        case.cache.table = case.cache.table.clone()                   # the handle knows the first one's address
    with pytest.raises(ValueError):
        attn.kv_append(torch.zeros(3, 12 * 128, dtype=torch.bfloat16, device=gpu), case.cache, 8, start=case.cache.kv_len.long())


@pytest.mark.parametrize("caps", [0, 30])
@pytest.mark.parametrize("D,dtype", [(64, "f16"), (128, "bf16")])
def test_pages_and_lengths_that_cannot_be(gpu, caps, D, dtype):
    """A page outside the pool is not touched, a length outside the table not walked: the sequence gets NaN and its
    weights stay; the others are as they were.  caps: more pages a table, so that the rows are split."""
    from tokamak_amd import attn
    lens = [100, 70, 200, 64, 33, 130, 90]
    case = Case(gpu, lens, 2, D, 64, dtype, weights=True, extra_pages=caps)
    c, cap = case.cache, case.max_pages * 64
    good = [t.clone() for t in (c.table, c.kv_len)]
    c.table[0, 1], c.table[2, 0], c.table[5, 2] = -1, c.num_pages, 2147483647
    c.kv_len[3], c.kv_len[6] = cap + 1, -1
    bad, ok = [0, 2, 3, 5, 6], [1, 4]
    q = q_of(case, 4)
    o, lse = attn.gqa_decode(q, c, 4, add_weights=True)
    assert torch.isnan(o[bad]).all() and torch.isnan(lse[bad]).all()
    assert torch.equal(c.weight[bad].cpu(), case.weight[bad])
    sub = Case.__new__(Case)
    sub.__dict__.update(case.__dict__)
    sub.B, sub.k, sub.v = 2, [case.k[b] for b in ok], [case.v[b] for b in ok]
    w = check_decode(sub, q[ok], o[ok], lse[ok], 4)
    for i, b in enumerate(ok):
        ref = case.weight[b, :, :lens[b]].double() + w[i]
        assert ((c.weight[b, :, :lens[b]].cpu().double() - ref).abs() <= 1e-4 * w[i] + 2.0 ** -23 * ref).all()
    # eviction leaves them alone and says so
    before = [t.clone() for t in (c.k, c.v, c.weight)]
    kept = attn.kv_evict(c, 40)
    assert (kept[bad] == -1).all() and c.kv_len.tolist() == [-1, 40, -1, -1, 33, -1, -1]
    assert torch.equal(c.weight[bad], before[2][bad])
    hit = torch.unique(good[0][[1, 4]][good[0][[1, 4]] >= 0]).long()
    rest = torch.ones(c.num_pages, dtype=torch.bool, device=gpu)
    rest[hit] = False
    assert torch.equal(c.k.view(torch.int16)[rest], before[0].view(torch.int16)[rest])
    assert torch.equal(c.v.view(torch.int16)[rest], before[1].view(torch.int16)[rest])
    # appended rows that fall there are dropped
    c.table[:, :] = good[0]
    c.table[0, 1], c.table[1, 0] = c.num_pages, -5
    start = torch.tensor([60, 10, -3, cap - 2, cap, 2147483647, 0], dtype=torch.int32, device=gpu)
    before = [t.clone() for t in (c.k, c.v, c.weight)]
    for S in (1, 5):
        qkv = torch.ones(7, S, 8 * D, dtype=DT[dtype], device=gpu)
        attn.kv_append(qkv, c, 4, start=start)
        assert c.kv_len.tolist() == [60 + S, 10 + S, -1, cap - 2 + S, cap + S, 2147483647, S]
    k, v = before[0].clone(), before[1].clone()
    for b, at in ((0, range(60, 64)), (6, range(5))) + (((3, range(cap - 2, cap)),) if c.table[3, -1] >= 0 else ()):
        for j in at:
            pg = int(c.table[b, j // 64])
            k[pg, :, j % 64 // 32, :, j % 32] = 1
            v[pg, :, j % 64 // 32, :, :, j % 32] = 1
    assert torch.equal(c.k.view(torch.int16), k.view(torch.int16)) and torch.equal(c.v.view(torch.int16), v.view(torch.int16))


def test_pages_beyond_32_bit_offsets(gpu):
    """A pool of 5 GB of K and as much of V, the sequence's pages at its end: the same results as from a small one."""
    from tokamak_amd import attn
    case = Case(gpu, [700], 8, 128, 256, "bf16", weights=True, spare=4)
    c, n = case.cache, 9600
    big = attn.KvCache(torch.empty((n,) + tuple(c.k.shape[1:]), dtype=c.dtype, device=gpu), torch.empty((n,) + tuple(c.k.shape[1:]), dtype=c.dtype, device=gpu),
                       torch.where(c.table >= 0, c.table + (n - c.num_pages), c.table), c.kv_len.clone(), c.weight.clone())
    assert big.k.numel() * 2 > 4 << 30
    big.k[-c.num_pages:], big.v[-c.num_pages:] = c.k, c.v
    q = q_of(case, 16, packed=True)
    for one in (c, big):
        # a page more, for the rows to come
        one.table[0, 3] = int(case.free[0]) + (0 if one is c else n - c.num_pages)
    got = []
    for one in (c, big):
        attn.kv_append(q, one, 16)
        o, lse = attn.gqa_decode(q, one, 16, add_weights=True)
        attn.kv_append(q[:, None].expand(1, 300, -1).contiguous(), one, 16)
        kept = attn.kv_evict(one, 500, sink=2, recent=30)
        got.append((o, lse, kept, one.weight, one.kv_len, *case.held(0, one)))
    for x, y in zip(*got):
        assert torch.equal(x, y)


def _clone(c):
    from tokamak_amd import attn
    return attn.KvCache(c.k.clone(), c.v.clone(), c.table.clone(), c.kv_len.clone(), None if c.weight is None else c.weight.clone())


@pytest.mark.parametrize("pages", [10, 60])
def test_a_step_captured_and_replayed(gpu, pages):
    """append, decode with weights, evict as one graph, replayed on inputs, lengths and tables that change, with
    eager work between; every replay against the eager calls, bit for bit.  Two graphs share nothing."""
    from tokamak_amd import attn
    B, Hq, Hkv, D, page = 5, 8, 2, 64, 64
    case = Case(gpu, [300, 1, 64, 639, 0], Hkv, D, page, "f16", weights=True, extra_pages=pages - 10, spare=8)
    c = case.cache
    c.table[torch.tensor([1, 2, 4]), torch.tensor([1, 1, 0])] = case.free[:3].to(torch.int32).to(gpu)
    qkv = torch.empty(B, (Hq + 2 * Hkv) * D, dtype=torch.float16, device=gpu)
    kept = torch.empty(B, Hkv, 320, dtype=torch.int32, device=gpu)

    def step(c, qkv, kept):
        attn.kv_append(qkv, c, Hq)
        o, lse = attn.gqa_decode(qkv, c, Hq, add_weights=True)
        attn.kv_evict(c, 320, 4, 100, kept=kept)
        return o, lse

    start = [t.clone() for t in (c.k, c.v, c.table, c.kv_len, c.weight)]
    step(c, qkv.normal_(), kept)
    graphs, outs, caches = [], [], [c, _clone(c)]
    for one in caches:
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(one, qkv, kept if one is c else kept.clone()))
        graphs.append(g)
    for one in caches:
        for t, s in zip((one.k, one.v, one.table, one.kv_len, one.weight), start):
            t.copy_(s)
    eager, ek = _clone(c), kept.clone()
    side = torch.cuda.Stream()
    for i in range(4):
        qkv.normal_()
        o, lse = step(eager, qkv, ek)
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        for one, out in zip(caches, outs):
            for x, y in zip((*out, one.k, one.v, one.kv_len, one.weight), (o, lse, eager.k, eager.v, eager.kv_len, eager.weight)):
                assert torch.equal(x.view(torch.int16), y.view(torch.int16))      # bits: there are NaN among them
        assert torch.equal(kept, ek)
        # lengths set anew, in part beyond what was ever stored: NaN come from there
        for one in caches + [eager]:
            one.kv_len[i] = 7 * i
            one.kv_len[3] = 500 + i


def test_calls_on_streams_of_their_own(gpu):
    """Several calls at once on one cache, each on a stream of its own, against the same ones in a row."""
    from tokamak_amd import attn
    case = Case(gpu, [3000, 777, 2048], 4, 64, 64, "bf16")
    qs = [q_of(case, 16, seed=i) for i in range(4)]
    ref = [attn.gqa_decode(q, case.cache, 16) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    got = [attn.gqa_decode(q, case.cache, 16, stream=s) for _ in range(5) for q, s in zip(qs, streams)]
    torch.cuda.synchronize()
    for i, (o, lse) in enumerate(got):
        assert torch.equal(o, ref[i % 4][0]) and torch.equal(lse, ref[i % 4][1])
    with torch.cuda.stream(streams[0]):
        o, lse = attn.gqa_decode(qs[0], case.cache, 16)
    torch.cuda.synchronize()
    assert torch.equal(o, ref[0][0]) and torch.equal(lse, ref[0][1])


def test_into_another_pool_without_weights(gpu):
    from tokamak_amd import attn
    case = Case(gpu, [300, 40], 2, 64, 64, "f16", weights=True)
    d = attn.KvCache.empty(2, 3, 6, 2, 64, 64, device=gpu)
    d.table.copy_(torch.randperm(6).reshape(2, 3).to(torch.int32))
    before = [t.clone() for t in (case.cache.k, case.cache.v)]
    kept = attn.kv_evict(case.cache, 150, 1, 10, dst=d)
    assert torch.equal(case.cache.k.view(torch.int16), before[0].view(torch.int16)) and d.kv_len.tolist() == [150, 40]
    for b in range(2):
        k, v = case.held(b, d)
        for h in range(2):
            at = [j for j in kept[b, h].tolist() if j >= 0]
            assert at == evict_ref(case.weight[b, h].tolist(), case.lens[b], 150, 1, 10)
            assert torch.equal(k[h], case.k[b][h, at]) and torch.equal(v[h], case.v[b][h, at])
    q = q_of(case, 4)
    o, lse = attn.gqa_decode(q, d, 4)
    sub = Case.__new__(Case)
    sub.__dict__.update(case.__dict__)
    sub.k, sub.v = map(list, zip(*[case.held(b, d) for b in range(2)]))
    check_decode(sub, q, o, lse, 4)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_generation(gpu, dtype):
    """The operators as a decoder's step uses them: the prompt's attention and its append, then tokens one by one,
    each an append, a decode with weights, logits and a draw, with an eviction when the cache is full.  Every
    step's O, LSE, weights and token against 64 bits on what the cache then holds."""
    from sample_cases import draw_ref
    from tokamak_amd import attn, runtime
    B, S, Hq, Hkv, D, page, budget, V = 3, 90, 4, 2, 64, 32, 96, 500
    g = torch.Generator().manual_seed(5)
    dt, pages = DT[dtype], 4
    c = attn.KvCache.empty(B, pages, B * pages, Hkv, D, page, dt, gpu, weights=True)
    c.table.copy_(torch.randperm(B * pages, generator=g).reshape(B, pages).to(torch.int32))
    n_new = torch.tensor([90, 31, 64], dtype=torch.int32, device=gpu)
    qkv = torch.randn(B, S, (Hq + 2 * Hkv) * D, generator=g).to(dt).to(gpu)
    o, lse = attn.gqa_fwd(qkv, B, S, Hq, Hkv, D, kv_len=n_new)
    attn.kv_append(qkv, c, Hq, n_new=n_new)
    head = torch.randn(Hq * D, V, generator=g).to(gpu)
    case = Case.__new__(Case)
    case.B, case.Hkv, case.D, case.page, case.dtype, case.dev = B, Hkv, D, page, dtype, gpu
    x = qkv.cpu().double().reshape(B, S, Hq + 2 * Hkv, D)
    hist = [[list(x[b, :n, Hq + h].unbind(0)) for h in range(2 * Hkv)] for b, n in enumerate(n_new.tolist())]   # K heads, V heads
    weight = [[[0.0] * n for _ in range(Hkv)] for n in n_new.tolist()]
    # the prompt's last row, asked of the cache, is the row the whole-sequence forward gave
    last = qkv[torch.arange(B), n_new.long() - 1]
    o1, lse1 = attn.gqa_decode(last, c, Hq)
    at = (n_new.long() - 1).to(gpu)
    d = (o1.float() - o[torch.arange(B, device=gpu), at].float()).abs()
    assert (d <= 2 * 2.0 ** (-11 if dtype == "f16" else -8) * o1.float().abs() + 2e-3).all()       # two roundings, and the forward's own bar
    assert (lse1 - lse[torch.arange(B, device=gpu), :, at]).abs().max() < 2e-3
    for step in range(12):
        row = torch.randn(B, (Hq + 2 * Hkv) * D, generator=g).to(dt).to(gpu)
        attn.kv_append(row, c, Hq)
        r = row.cpu().double().reshape(B, Hq + 2 * Hkv, D)
        for b in range(B):
            for h in range(2 * Hkv):
                hist[b][h].append(r[b, Hq + h])
            for h in range(Hkv):
                weight[b][h].append(0.0)
        case.k = [torch.stack([torch.stack(hist[b][h]) for h in range(Hkv)]) for b in range(B)]
        case.v = [torch.stack([torch.stack(hist[b][Hkv + h]) for h in range(Hkv)]) for b in range(B)]
        for b in range(B):
            k, v = case.held(b, c)
            assert torch.equal(k, case.k[b]) and torch.equal(v, case.v[b])
        o, lse = attn.gqa_decode(row, c, Hq, add_weights=True)
        w = check_decode(case, row[:, :Hq * D], o, lse, Hq)
        for b in range(B):
            n = len(weight[b][0])
            ref = torch.tensor(weight[b], dtype=torch.float64) + w[b]
            got = c.weight[b, :, :n].cpu().double()
            assert ((got - ref).abs() <= 1e-4 * w[b] + 2.0 ** -23 * ref).all()
            weight[b] = got.tolist()
        logits, u = o.float() @ head, torch.rand(B, generator=g).to(gpu)
        p = torch.full((B,), 0.9, device=gpu)
        token = runtime.sample(logits, u, top_p=p, top_k=torch.full((B,), 50, dtype=torch.int32, device=gpu))
        assert token.tolist() == [draw_ref(logits[b].cpu().double().numpy(), float(u[b]), top_k=50, top_p=float(p[b]))[0] for b in range(B)]
        if int(c.kv_len.max()) > budget:
            kept = attn.kv_evict(c, budget - 8, sink=2, recent=20).cpu()
            for b in range(B):
                n = len(weight[b][0])
                for h in range(Hkv):
                    ref = evict_ref(weight[b][h], n, budget - 8, 2, 20)
                    assert [j for j in kept[b, h].tolist() if j >= 0] == ref
                    hist[b][h], hist[b][Hkv + h] = [hist[b][h][j] for j in ref], [hist[b][Hkv + h][j] for j in ref]
                    weight[b][h] = [weight[b][h][j] for j in ref]
    assert c.kv_len.tolist() == [len(weight[b][0]) for b in range(B)] and max(c.kv_len.tolist()) <= budget
