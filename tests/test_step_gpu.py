"""A serving step's calls on the GPU: rotary positions, the plan, the append of packed rows and the attention of new
rows, against the operators in 64 bits (step_cases.py has the bounds).  Moves and whole numbers are compared exactly."""
import math

import pytest
import torch

from kv_cases import DT, HALF, TINY, Case, dense
from step_cases import check_chunk, check_rounded, chunk_ref, freqs_ref, plan_ref, rope_ref, visible

pytestmark = pytest.mark.gpu

ROPES = [(128, 128, "halves", None), (128, 64, "pairs", "yarn"), (64, 40, "halves", "bands"), (64, 62, "pairs", "ntk"),
         (64, 20, "pairs", "linear"), (128, 36, "halves", None), (64, 2, "halves", None), (128, 126, "halves", "linear"), (64, 2, "pairs", "ntk")]
SCALED = {None: {}, "linear": {"scale": 4.0}, "ntk": {"scale": 4.0}, "bands": {"scale": 8.0}, "yarn": {"scale": 4.0}}


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def randn(shape, dtype, seed=0, mul=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * mul).to(DT[dtype])


def rope_of(rot, layout, scaling, theta=10000.0):
    from tokamak_amd import attn
    return attn.Rope(rot, theta=theta, layout=layout, scaling=scaling, **SCALED[scaling]), freqs_ref(rot, theta, scaling, **SCALED[scaling])


# ---- rotary positions ---------------------------------------------------------------------------------


@pytest.mark.parametrize("D,rot,layout,scaling", ROPES)
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows,Hq,Hkv", [(1, 1, 1), (37, 8, 2), (9, 5, 0), (1500, 6, 3), (4100, 1, 1)])
def test_rope(gpu, D, rot, layout, scaling, dtype, rows, Hq, Hkv):
    from tokamak_amd import attn
    print(f"[case] rows {rows} Hq{Hq} Hkv{Hkv} D{D} rot {rot} {layout} {scaling} {dtype}", flush=True)
    r, (freqs, factor) = rope_of(rot, layout, scaling)
    C = (Hq + 2 * Hkv) * D
    g = torch.Generator().manual_seed(rows)
    pos = torch.randint(0, 1 << 20, (rows,), generator=g)
    pos[rows // 2], pos[-1] = 0, (1 << 31) - 1
    if rows > 5:
        pos[3], pos[4] = -1, -(1 << 31)
    x = randn((rows, C), dtype, 1)
    wide = torch.full((rows, C + 24), 7.0, dtype=DT[dtype], device=gpu)
    for inverse, call in ((False, attn.rope_fwd), (True, attn.rope_bwd)):
        e = x.double().reshape(rows, Hq + 2 * Hkv, D)
        y, err = e.clone(), torch.zeros_like(e)
        y[:, :Hq + Hkv], err[:, :Hq + Hkv] = rope_ref(e[:, :Hq + Hkv], pos.tolist(), freqs, factor, layout, inverse)
        gone = pos < 0
        wide.fill_(7.0)
        wide[:, 8:8 + C] = -3.0
        out = call(x.to(gpu), r, Hq, Hkv, D, i32(pos.tolist(), gpu), None, wide[:, 8:8 + C])      # rows apart, another stride
        assert attn.last_kernels() == ["rope"]
        got = out.cpu().double().reshape(e.shape)
        assert (got[gone] == -3.0).all() and (wide[:, :8] == 7.0).all() and (wide[:, 8 + C:] == 7.0).all()
        check_rounded(got[~gone], y[~gone], err[~gone], dtype, "inverse" if inverse else "forward")
        assert torch.equal(got[~gone][..., rot:], e[~gone][..., rot:]) and torch.equal(got[~gone][:, Hq + Hkv:], e[~gone][:, Hq + Hkv:])
        inp = x.to(gpu)
        assert call(inp, r, Hq, Hkv, D, i32(pos.tolist(), gpu), None, inp) is inp               # in place
        assert torch.equal(inp.cpu()[~gone], out.cpu()[~gone]) and torch.equal(inp.cpu()[gone], x[gone])


@pytest.mark.parametrize("layout", ["halves", "pairs"])
def test_rope_is_a_training_step(gpu, layout):
    """Rows of sequences of S, by their place; the gradient is that of the rotation: <dy, R x> = <R^T dy, x>, and
    differences of the rotation along dx give the same (64 bits on the CPU for both)."""
    from tokamak_amd import attn
    B, S, Hq, Hkv, D = 3, 50, 4, 2, 64
    r, (freqs, factor) = rope_of(48, layout, "yarn")
    x, dy = randn((B, S, (Hq + 2 * Hkv) * D), "f16", 1), randn((B, S, (Hq + 2 * Hkv) * D), "f16", 2)
    y = attn.rope_fwd(x.to(gpu), r, Hq, Hkv, D, S=S)
    dx = attn.rope_bwd(dy.to(gpu), r, Hq, Hkv, D, S=S)
    pos = [i % S for i in range(B * S)]

    def turned(v, inverse=False):
        v = v.double().reshape(B * S, Hq + 2 * Hkv, D)
        out, e = v.clone(), torch.zeros_like(v)
        out[:, :Hq + Hkv], e[:, :Hq + Hkv] = rope_ref(v[:, :Hq + Hkv], pos, freqs, factor, layout, inverse)
        return out, e
    for got, (want, e), what in ((y, turned(x), "y"), (dx, turned(dy, True), "dx")):
        check_rounded(got.cpu().double().reshape(want.shape), want, e, "f16", what)
    # the gradient against differences: a linear map's are exact up to the rounding of dx, half a step a value
    step = randn(x.shape, "f16", 3).double()
    along = ((turned(x.double() + step)[0] - turned(x.double() - step)[0]) / 2 * dy.double().reshape(B * S, -1, D)).sum()
    d = dx.cpu().double()
    bound = ((HALF["f16"] * d.abs() + 2.0 ** -19 * dy.double().abs().amax() * factor + TINY["f16"]) * step.abs()).sum()
    assert abs((d * step).sum() - along) <= bound


def test_rope_agrees_with_prep(gpu):
    """The rows that the qkv-prep kernels turn by their place, up to their fp32 angles: S of 300 at 1 radian a row is
    off by 2^-24 * 300, and its sine and cosine by no more."""
    from tokamak_amd import attn, prep
    Hq, Hkv, D, S = 4, 2, 64, 300
    p = prep.Prep(Hq, Hkv, D, S, rope=True, dtype="f16", scale=4.0)
    x = randn((2 * S, p.C), "f16", 5).to(gpu)
    want = p.fwd(x, torch.zeros(p.C, device=gpu))[0].double()
    got = attn.rope_fwd(x, attn.Rope.of_prep(p.desc), Hq, Hkv, D, S=S).double()
    size = x.double().abs().reshape(-1, D // 2, 2).sum(2).repeat_interleave(2, 1).reshape(got.shape)
    assert ((got - want).abs() <= 2 * HALF["f16"] * want.abs() + (2 * 300 * 2.0 ** -24 + 2.0 ** -20) * size + 2 * TINY["f16"]).all()


# ---- the plan -------------------------------------------------------------------------------------------


class Pool:
    """A cache without data to speak of, its pages and a few requests."""

    def __init__(self, dev, B, page, max_pages, num_pages, held, seed=0):
        from tokamak_amd import attn
        g = torch.Generator().manual_seed(seed)
        ids = torch.randperm(num_pages, generator=g).tolist()
        self.B, self.page, self.max_pages, self.num_pages, self.dev = B, page, max_pages, num_pages, dev
        self.table, used = [], 0
        for n in held:
            self.table.append(ids[used:used + n] + [-1] * (max_pages - n))
            used += n
        self.held, self.n_free = list(held), num_pages - used
        self.free = ids[used:] + [-5] * used
        pool = torch.zeros((num_pages, 1, page // 32, 2, 32, 32), dtype=torch.float16, device=dev)
        self.cache = attn.KvCache(pool, pool.clone(), i32(self.table, dev), torch.zeros(B, dtype=torch.int32, device=dev))
        self.pages = attn.KvPages(i32(self.free, dev), i32([self.n_free], dev), i32(self.held, dev))

    def step(self, want, start, rows, given=True, plan=None):
        from tokamak_amd import attn
        ref = plan_ref(self.table, self.free, self.n_free, self.held, want, start, self.page, self.num_pages, rows)
        if not given:
            self.cache.kv_len.copy_(i32(start, self.dev))
        p = attn.kv_plan(self.cache, self.pages, i32(want, self.dev), rows=rows, start=i32(start, self.dev) if given else None, plan=plan)
        assert attn.last_kernels() == ["plan"]
        self.compare(p, ref)
        self.table, self.free, self.n_free, self.held = ref["table"], ref["free"], ref["n_free"][0], ref["held"]
        return p, ref

    def compare(self, p, ref):
        got = {"table": self.cache.table, "free": self.pages.free, "n_free": self.pages.n_free, "held": self.pages.held,
               "kv_len": self.cache.kv_len, "n_new": p.n_new, "row_start": p.row_start, "seq": p.seq, "pos": p.pos, "slot": p.slot}
        for k, v in got.items():
            assert v.tolist() == ref[k], k


@pytest.mark.parametrize("B,page,rows,num", [(1, 32, 1, 3), (7, 64, 900, 40), (64, 32, 64, 400), (300, 32, 5000, 900), (1024, 256, 700, 3000),
                                             (1025, 32, 9000, 2500), (2600, 64, 6000, 9000), (5000, 32, 5001, 9000)])
@pytest.mark.parametrize("given", [0, 1])
def test_plan(gpu, B, page, rows, num, given):
    """Several steps in a row, with sequences that grow, end, shrink, ask for too much and lie outside their tables."""
    g = torch.Generator().manual_seed(B)
    most = 9
    held = torch.randint(0, max(1, min(most, num // B) + 1), (B,), generator=g).tolist()
    pool = Pool(gpu, B, page, most, num, held)
    start = [max(0, h * page - int(x)) for h, x in zip(held, torch.randint(0, page, (B,), generator=g))]
    for step in range(4):
        print(f"[case] B{B} page{page} rows{rows} step {step}", flush=True)
        kind = torch.randint(0, 12, (B,), generator=g).tolist()
        size = torch.randint(1, 3 * rows // B + 3, (B,), generator=g).tolist()
        want = [1 if k < 5 else n if k < 8 else 0 if k < 10 else -3 if k == 10 else (1 << 31) - 1 for k, n in zip(kind, size)]
        for b in range(1, B, 5):
            if kind[b] == 9:
                start[b] = 0
        if B > 6:
            start[5], start[6] = -1, most * page + 1
        _, ref = pool.step(want, start, rows, bool(given))
        _, again = pool.step(want, start, rows, True) if given else (None, None)
        if given:          # whoever got its rows gets the same again
            assert all(a == n for a, n in zip(again["n_new"], ref["n_new"]) if n)
        start = [max(0, n) if b not in (5, 6) else 0 for b, n in enumerate(ref["kv_len"])]


def test_plan_edges(gpu):
    from tokamak_amd import attn
    pool = Pool(gpu, 3, 32, 4, 12, [4, 0, 1])
    pool.step([0, 128, 31], [128, 0, 1], 200)                 # exactly full tables and pages
    pool.step([1, 1, 1], [128, 128, 32], 200)                 # over them
    pool.step([0, 0, 0], [0, 0, 0], 200)                      # all end
    assert pool.n_free == 12
    pool.step([128, 128, 128], [0, 0, 0], 384)                # the whole pool
    assert pool.n_free == 0
    pool.step([0, 5, 0], [0, 128, 128], 0)                    # no rows at all; the first one's pages come back
    # a stack that says more than there is, and table entries and pages outside the pool, reach nothing
    pool.pages.n_free.fill_(1 << 30)
    pool.pages.held.copy_(i32([1 << 30, -7, 4], gpu))
    pool.pages.free.fill_(99)
    p = attn.kv_plan(pool.cache, pool.pages, i32([5, 70, 1], gpu), rows=100, start=i32([0, 0, 127], gpu))
    assert p.n_new.tolist() == [5, 70, 1] and (p.slot[5:75] == -1).all() and pool.cache.table[1, :3].tolist() == [99, 99, 99]   # 70 tokens: 3 pages of none held
    with pytest.raises(ValueError):
        attn.kv_plan(pool.cache, pool.pages, i32([5, 70, 1], gpu))
    with pytest.raises(ValueError):
        attn.kv_plan(pool.cache, pool.pages, i32([5, 70], gpu), rows=4)


# ---- packed rows into the cache ----------------------------------------------------------------------------


def packed(starts, n_new, case, behind=3):
    """(seq, pos, slot, row_start) lists of packed rows at the given positions of a case's pages, some rows behind."""
    table, page = case.cache.table.tolist(), case.page
    seq = [b for b, n in enumerate(n_new) for _ in range(n)]
    pos = [starts[b] + i for b, n in enumerate(n_new) for i in range(n)]
    slot = [table[b][p // page] * page + p % page for b, p in zip(seq, pos)]
    row_start = [sum(n_new[:b]) for b in range(len(n_new) + 1)]
    pad = [-1] * behind
    return seq + pad, pos + pad, slot + pad, row_start


@pytest.mark.parametrize("D,rot,layout,scaling", ROPES[:6] + [(64, 0, "halves", None), (128, 0, "halves", None)])
@pytest.mark.parametrize("starts,n_new,Hq,Hkv,page,dtype", [
    ([0], [1], 1, 1, 32, "f16"), ([0, 31, 200, 5], [1, 1, 1, 0], 4, 2, 32, "bf16"), ([5, 64, 0, 33], [77, 1, 0, 140], 2, 2, 64, "f16"),
    ([3, 500], [700, 611], 6, 3, 128, "bf16"), ([0] + [7] * 40, [40] * 41, 8, 1, 256, "f16")])
def test_append_rows(gpu, D, rot, layout, scaling, starts, n_new, Hq, Hkv, page, dtype):
    from tokamak_amd import attn
    print(f"[case] {len(starts)} sequences Hq{Hq} Hkv{Hkv} D{D} page{page} rot {rot} {layout} {dtype}", flush=True)
    pages = max((s + n + page - 1) // page for s, n in zip(starts, n_new))
    case = Case(gpu, [pages * page] * len(starts), Hkv, D, page, dtype, extra_pages=0, weights=True)
    c = case.cache
    seq, pos, slot, row_start = packed(starts, n_new, case)
    rows, total = len(seq), len(seq) - 3
    if total > 2:
        slot[2] = case.cache.num_pages * page        # not a slot of the pool: the row's K and V go nowhere, Q is turned
    plan = attn.KvPlan(i32(n_new, gpu), i32(row_start, gpu), i32(seq, gpu), i32(pos, gpu), torch.tensor(slot, device=gpu))
    r, (freqs, factor) = rope_of(rot, layout, scaling) if rot else (None, (None, None))
    W = (Hq + 2 * Hkv) * D
    x = randn((rows, W), dtype, 3)
    before = [t.clone() for t in (c.k, c.v, c.weight, c.kv_len)]
    ref = x.double().reshape(rows, Hq + 2 * Hkv, D)
    err = torch.zeros_like(ref)
    if rot:
        ref[:, :Hq + Hkv], err[:, :Hq + Hkv] = rope_ref(ref[:, :Hq + Hkv], [max(0, p) for p in pos], freqs, factor, layout)
    for mode in ("new", "given", "in place"):
        for t, old in zip((c.k, c.v, c.weight), before):
            t.copy_(old)
        inp = torch.full((rows, W + 16), 9.0, dtype=DT[dtype], device=gpu)[:, :W]      # rows further apart
        inp.copy_(x)
        given = torch.full((rows, Hq * D + 8), 5.0, dtype=DT[dtype], device=gpu)
        q = attn.kv_append_rows(inp, c, Hq, plan, rope=r, q={"new": None, "given": given, "in place": inp}[mode])
        assert attn.last_kernels() == ["append"]
        if mode == "given":
            assert q is given and (given[:, Hq * D:] == 5.0).all() and (given[total:] == 5.0).all()
        elif mode == "in place" or rot == 0:
            assert q is inp and torch.equal(inp[:, Hq * D:].cpu(), x[:, Hq * D:]) and torch.equal(inp[total:].cpu(), x[total:])
        got = q[:total, :Hq * D].cpu().double().reshape(total, Hq, D)
        check_rounded(got, ref[:total, :Hq], err[:total, :Hq], dtype, f"q {mode}")
        assert torch.equal(got[..., rot:], ref[:total, :Hq, rot:])
    k, v, w = (t.clone().cpu() for t in before[:3])
    ek = torch.zeros(k.shape, dtype=torch.float64)
    k, v = k.double(), v.double()
    for i in range(total):
        if 0 <= slot[i] < c.num_pages * page:
            at, tile, tok = slot[i] // page, slot[i] % page // 32, slot[i] % 32
            k[at, :, tile, :, tok] = ref[i, Hq:Hq + Hkv].reshape(Hkv, D // 32, 32)
            ek[at, :, tile, :, tok] = err[i, Hq:Hq + Hkv].reshape(Hkv, D // 32, 32)
            v[at, :, tile, :, :, tok] = ref[i, Hq + Hkv:].reshape(Hkv, D // 32, 32)
            w[seq[i], :, pos[i]] = 0
    assert torch.equal(c.v.cpu().double().nan_to_num(77.0), v.nan_to_num(77.0))
    assert torch.equal(c.weight.cpu(), w) and torch.equal(c.kv_len, before[3])
    gk = c.k.cpu().double()
    there = torch.isfinite(k)
    assert torch.equal(gk[~there].nan_to_num(77.0), k[~there].nan_to_num(77.0))
    check_rounded(gk[there], k[there], ek[there] + (0 if rot else -TINY[dtype] / 2), dtype, "k")


# ---- attention of new rows -----------------------------------------------------------------------------------

SETS = {
    "one": ([1], [1]), "edges": ([1, 31, 32, 33, 64, 65, 0, 96], [1, 5, 32, 1, 64, 2, 0, 33]), "few": ([3, 10], [7, 12]),
    "nothing": ([0, 0], [3, 0]), "ragged": ([700, 0, 2049, 513, 96, 40], [1, 0, 300, 513, 17, 40]), "long": ([5003], [3]), "prompt": ([1500], [1500]),
    "many": ([(37 * i) % 301 + 4 for i in range(150)], [1 + i % 3 for i in range(150)]), "two": ([4097, 40], [150, 1]),
}
HEADS = [(4, 4, 64, 32, "f16"), (8, 2, 128, 64, "bf16"), (16, 1, 128, 128, "f16"), (3, 1, 64, 256, "bf16"), (10, 2, 64, 64, "f16"),
         (34, 2, 128, 32, "bf16"), (150, 1, 64, 64, "f16")]


def queries(total, Hq, Hkv, D, dtype, dev, seed=7, mul=1.0, wide=True):
    return randn((total, (Hq + (2 * Hkv if wide else 0)) * D), dtype, seed, mul).to(dev)


@pytest.mark.parametrize("name", SETS)
@pytest.mark.parametrize("Hq,Hkv,D,page,dtype", HEADS)
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 1), (True, 70), (True, 1000)])
def test_chunk(gpu, name, Hq, Hkv, D, page, dtype, causal, window):
    from tokamak_amd import attn
    lens, n_new = SETS[name]
    if sum(n_new) * Hq * max(lens) > 3e7:
        n_new = [min(n, 130) for n in n_new]
    print(f"[case] {name} Hq{Hq} Hkv{Hkv} D{D} page{page} {dtype} causal {causal} window {window}", flush=True)
    case = Case(gpu, lens, Hkv, D, page, dtype)
    total = sum(n_new)
    q = queries(total + 3, Hq, Hkv, D, dtype, gpu)
    row_start = [sum(n_new[:b]) for b in range(len(n_new) + 1)]
    out = torch.full((total + 3, Hq * D), 4.0, dtype=DT[dtype], device=gpu)
    lse = torch.full((total + 3, Hq), 4.0, device=gpu)
    attn.gqa_chunk(q, case.cache, Hq, i32(row_start, gpu), i32(n_new, gpu), causal=causal, window=window, out=out, lse=lse)
    assert attn.last_kernels()[-1] == "chunk"
    assert (out[total:] == 4.0).all() and (lse[total:] == 4.0).all()
    check_chunk(case, lens, n_new, q, out, lse, Hq, causal=causal, window=window)
    again = attn.gqa_chunk(q[:total, :Hq * D].contiguous(), case.cache, Hq, i32(row_start, gpu)[:len(lens)], i32(n_new, gpu), causal=causal, window=window)
    check_chunk(case, lens, n_new, q, *again, Hq, causal=causal, window=window)


@pytest.mark.parametrize("Hq,Hkv,D,page,dtype", HEADS[:3])
def test_chunk_of_padded_rows(gpu, Hq, Hkv, D, page, dtype):
    """A batch of S rows a sequence, all of them or the first n_new."""
    from tokamak_amd import attn
    lens, S = [100, 33, 900], 33
    case = Case(gpu, lens, Hkv, D, page, dtype)
    q = queries(3 * S, Hq, Hkv, D, dtype, gpu)
    o, lse = attn.gqa_chunk(q, case.cache, Hq)
    check_chunk(case, lens, [S] * 3, q, o, lse, Hq)
    out = torch.full((3 * S, Hq * D), 4.0, dtype=DT[dtype], device=gpu)
    o, lse = attn.gqa_chunk(q, case.cache, Hq, n_new=i32([5, 0, 32], gpu), out=out)
    check_chunk(case, lens, [5, 0, 32], q, o, lse, Hq, row_start=[0, S, 2 * S])
    for rows in ([5, 2 * S], [2 * S + 32, 3 * S]):
        assert (out[rows[0]:rows[1]] == 4.0).all()


@pytest.mark.parametrize("Hq,Hkv,D,page,dtype", HEADS[:2])
@pytest.mark.parametrize("mul,trend,scale", [(8.0, 0.0, None), (1.0, 30.0, None), (1.0, -30.0, None), (0.01, 0.0, 1.0), (1.0, 0.0, 1e-6), (4.0, 300.0, 1.0)])
def test_chunk_of_steep_scores(gpu, Hq, Hkv, D, page, dtype, mul, trend, scale):
    """Scores that grow or fall along the keys by far more than fp16 holds, and flat ones."""
    from tokamak_amd import attn
    lens, n_new = [1400, 70], [70, 70]
    case = Case(gpu, lens, Hkv, D, page, dtype, mul=mul, trend=trend)
    q = queries(140, Hq, Hkv, D, dtype, gpu, mul=mul)
    o, lse = attn.gqa_chunk(q, case.cache, Hq, scale=scale)
    check_chunk(case, lens, n_new, q, o, lse, Hq, scale=scale)


@pytest.mark.parametrize("Hq,Hkv,D,page,dtype,extra", [(2, 2, 64, 32, "f16", 1), (8, 2, 128, 64, "bf16", 1), (8, 1, 64, 64, "bf16", 40),
                                                       (2, 2, 128, 32, "bf16", 60), (12, 2, 128, 64, "f16", 40), (1, 1, 128, 128, "f16", 1)])
@pytest.mark.parametrize("n", [40, 20])
def test_chunk_of_odd_values(gpu, Hq, Hkv, D, page, dtype, extra, n):
    """NaN and infinities among keys and values: rows that see one have one of them there, the others nothing of it, in
    calls of one launch and of three (extra pages make the tables long)."""
    from tokamak_amd import attn
    print(f"[case] odd values Hq{Hq} Hkv{Hkv} D{D} {dtype} n{n}", flush=True)
    L, G = 300, Hq // Hkv
    case = Case(gpu, [L, 33], Hkv, D, page, dtype, extra_pages=extra)
    odd = [(281, 3, math.inf), (285, 5, math.nan), (290, 7, -math.inf), (293, 7, math.inf), (10, 9, -math.inf), (299, 11, math.inf)]
    v = case.v[0].clone()
    for j, d, x in odd:
        v[Hkv - 1, j, d] = x
        at, tok = case.cache.table[0, j // page], j % page
        case.cache.v[at, Hkv - 1, tok // 32, d // 32, d % 32, tok % 32] = x
        case.v[0][Hkv - 1, j, d] = 0.0
    at, tok = case.cache.table[0, 296 // page], 296 % page
    case.cache.k[at, 0, tok // 32, 0, tok % 32, 4] = math.nan
    case.k[0][0, 296] = 0.0
    q = queries(n + 5, Hq, Hkv, D, dtype, gpu)
    for window in (0, 100):
        o, lse = attn.gqa_chunk(q, case.cache, Hq, i32([0, n], gpu), i32([n, 5], gpu), window=window)
        got, pos = o.cpu().double().reshape(-1, Hq, D), [L - n + i for i in range(n)]
        see = lambda i, j: j <= pos[i] and (window == 0 or j > pos[i] - window)
        for i in range(n):
            for h in range(Hq):
                if h // G == 0 and see(i, 296):
                    assert torch.isnan(got[i, h]).all() and math.isnan(lse[i, h].item())
                    got[i, h] = 0.0
                elif h // G == Hkv - 1:
                    for d in (3, 5, 7, 9, 11):
                        hit = [x for j, dd, x in odd if dd == d and see(i, j)]
                        if hit:
                            assert not math.isfinite(got[i, h, d]), (i, h, d)
                            got[i, h, d] = 0.0
        for b, (length, m, first) in enumerate(((L, n, 0), (33, 5, n))):
            qq = q.cpu().double()[first:first + m, :Hq * D].reshape(m, Hq, D)
            ro, rl, eo, el = chunk_ref(qq, case.k[b], case.v[b], visible(length, m, True, window), Hkv, 1 / math.sqrt(D), dtype)
            g = got[first:first + m]
            same = torch.ones_like(g, dtype=torch.bool)
            if b == 0:         # what was compared above is 0 in g
                for i in range(m):
                    if see(i, 296):
                        same[i, :G] = False
                    for j, d, x in odd:
                        if see(i, j):
                            same[i, (Hkv - 1) * G:, d] = False
            assert torch.isfinite(g).all()
            tol = eo + HALF[dtype] * (ro.abs() + eo) + TINY[dtype]
            assert ((g - ro).abs() <= tol)[same].all()


@pytest.mark.parametrize("Hq,Hkv,D,page,dtype", [(2, 2, 64, 32, "f16"), (16, 2, 128, 64, "bf16")])
@pytest.mark.parametrize("extra", [1, 60])
def test_chunk_of_bad_pages_and_lengths(gpu, Hq, Hkv, D, page, dtype, extra):
    """A page outside the pool makes NaN of the rows that see it, a length outside the table of all the sequence's;
    the others are as they were."""
    from tokamak_amd import attn
    lens, n_new = [200, 200, 90, 70, 200], [30, 30, 40, 5, 30]
    case = Case(gpu, lens, Hkv, D, page, dtype, extra_pages=extra)
    c = case.cache
    c.table[0, (200 - 15) // page] = c.num_pages          # the page of row 15
    c.table[1, 0] = -1
    c.kv_len[2] = c.max_pages * page + 1
    c.kv_len[3] = -1
    q = queries(sum(n_new), Hq, Hkv, D, dtype, gpu)
    row_start = [sum(n_new[:b]) for b in range(6)]
    o, lse = attn.gqa_chunk(q, c, Hq, i32(row_start, gpu), i32(n_new, gpu))
    first = (200 - 15) // page * page                     # rows from this position on see the bad page
    clean = max(0, first - 170)
    assert torch.isnan(o[clean:30]).all() and torch.isnan(lse[clean:30]).all()
    for b in (1, 2, 3):
        assert torch.isnan(o[row_start[b]:row_start[b + 1]]).all() and torch.isnan(lse[row_start[b]:row_start[b + 1]]).all()
    check_chunk(case, lens, n_new, q, o, lse, Hq, skip=(0, 1, 2, 3))
    if clean:
        k, v = case.k[0], case.v[0]
        case.k[0], case.v[0] = k[:, :170 + clean], v[:, :170 + clean]
        check_chunk(case, [170 + clean], [clean], q, o, lse, Hq)
    o2, _ = attn.gqa_chunk(q, c, Hq, i32(row_start, gpu), i32(n_new, gpu), window=10)      # the first page is not seen any more
    assert torch.isfinite(o2[row_start[1]:row_start[2]]).all()


def test_chunk_of_rows_outside(gpu):
    """Rows that a batch does not have are passed over."""
    from tokamak_amd import attn
    case = Case(gpu, [100, 100, 100, 100], 2, 64, 64, "f16")
    q = queries(20, 4, 2, 64, "f16", gpu)
    out = torch.full((20, 256), 4.0, dtype=torch.float16, device=gpu)
    o, lse = attn.gqa_chunk(q, case.cache, 4, i32([-5, 3, 18, 20], gpu), i32([4, 5, 7, 3], gpu), out=out)
    check_chunk(case, [100] * 4, [0, 5, 0, 0], q, o, lse, 4, row_start=[0, 3, 0, 0])
    assert (out[:3] == 4.0).all() and (out[8:18] == 4.0).all() and torch.isfinite(out[18:]).all()


# ---- together ---------------------------------------------------------------------------------------------------


def rewound(case, b, n):
    """The case's sequence b cut to its first n tokens."""
    case.k[b], case.v[b] = case.k[b][:, :n], case.v[b][:, :n]


@pytest.mark.parametrize("Hq,Hkv,D,page,dtype,most,rope", [(8, 2, 64, 32, "f16", 12, (64, "halves", None)), (4, 4, 128, 64, "bf16", 40, (96, "pairs", "yarn")),
                                                           (6, 1, 64, 64, "bf16", 30, None)])
def test_steps_of_a_server(gpu, Hq, Hkv, D, page, dtype, most, rope):
    """Prompts, drafts of which a part is kept, single tokens, sequences that end and others in their place, a request
    too long for its table: two layers that share pages and lengths, each step planned once, appended and attended in both."""
    from tokamak_amd import attn
    print(f"[case] server Hq{Hq} Hkv{Hkv} D{D} page{page} {dtype}", flush=True)
    B, rows, W = 4, 400, (Hq + 2 * Hkv) * D
    layers = [Case(gpu, [0] * B, Hkv, D, page, dtype, spare=24, extra_pages=most - 1, seed=i) for i in range(2)]
    c = layers[0].cache
    layers[1].cache = attn.KvCache(layers[1].cache.k, layers[1].cache.v, c.table, c.kv_len)
    pages = attn.KvPages.all_free(c)
    assert pages.free.tolist() == list(range(c.num_pages - 1, -1, -1)) and int(pages.n_free) == c.num_pages
    r, (freqs, factor) = rope_of(*rope) if rope else (None, (None, None))
    plan = attn.KvPlan.empty(B, rows, gpu)
    lens, tokens = [0] * B, c.num_pages * page
    steps = [([130, 40, 0, 7], None), ([5, 5, 0, 5], None), ([1, 1, 90, 1], [132, 45, 0, 9]), ([1, 1, 1, 1], None), ([0, 0, 3, 3], [0, 46, 91, 11]),
             ([170, tokens, 1, 1], None), ([1, 1, 1, 1], None)]
    for i, (want, start) in enumerate(steps):
        start = list(lens) if start is None else start
        ref = plan_ref(c.table.tolist(), pages.free.tolist(), int(pages.n_free), pages.held.tolist(), want, start, page, c.num_pages, rows)
        attn.kv_plan(c, pages, i32(want, gpu), start=i32(start, gpu), plan=plan)
        n_new, row_start, lens = ref["n_new"], ref["row_start"], ref["kv_len"]
        assert plan.n_new.tolist() == n_new and plan.row_start.tolist() == row_start and plan.pos.tolist() == ref["pos"]
        assert c.kv_len.tolist() == lens and pages.held.tolist() == ref["held"]
        assert i != 5 or n_new == [170, 0, 1, 1]         # more than its table holds
        total = row_start[-1]
        for x, case in enumerate(layers):
            qkv = randn((rows, W), dtype, 10 * i + x).to(gpu)
            q = attn.kv_append_rows(qkv, case.cache, Hq, plan, rope=r)
            o, lse = attn.gqa_chunk(q, case.cache, Hq, plan.row_start, plan.n_new)
            new = qkv[:total].cpu().double().reshape(total, Hq + 2 * Hkv, D)
            err = torch.zeros_like(new)
            if rope:
                new[:, :Hq + Hkv], err[:, :Hq + Hkv] = rope_ref(new[:, :Hq + Hkv], ref["pos"][:total], freqs, factor, rope[1])
            check_rounded(q[:total, :Hq * D].cpu().double().reshape(total, Hq, D), new[:, :Hq], err[:, :Hq], dtype, "q")
            for b in range(B):
                rewound(case, b, start[b])
                at = slice(row_start[b], row_start[b + 1])
                k, v = case.held(b, case.cache)
                assert torch.equal(k[:, :start[b]], case.k[b]) and torch.equal(v[:, :start[b]], case.v[b])       # what was there
                check_rounded(k[:, start[b]:], new[at, Hq:Hq + Hkv].transpose(0, 1), err[at, Hq:Hq + Hkv].transpose(0, 1), dtype, "k")
                assert torch.equal(v[:, start[b]:], new[at, Hq + Hkv:].transpose(0, 1))
                case.k[b], case.v[b] = k, v
            check_chunk(case, lens, n_new, q, o, lse, Hq)
            if all(n == 1 for n in n_new):           # a token each: the decoding call has the same to do
                check_chunk(case, lens, n_new, q, *attn.gqa_decode(q[:B], case.cache, Hq), Hq)


def test_steps_captured_and_replayed(gpu):
    """Plan, append in place and attention of two layers as one graph, replayed on requests and rows that change, with
    eager work between, every replay against the eager calls bit for bit; two graphs use one workspace in turn."""
    from tokamak_amd import attn
    B, Hq, Hkv, D, page, dtype, rows = 5, 8, 2, 128, 64, "bf16", 96
    r, _ = rope_of(128, "halves", "bands")
    k = [randn((300, Hkv, page // 32, D // 32, 32, 32), dtype, s).to(gpu) for s in range(4)]
    x = randn((2, rows, (Hq + 2 * Hkv) * D), dtype, 9).to(gpu)
    want = torch.zeros(B, dtype=torch.int32, device=gpu)

    def world():
        table, length = torch.full((B, 50), -1, dtype=torch.int32, device=gpu), torch.zeros(B, dtype=torch.int32, device=gpu)
        layers = [attn.KvCache(k[2 * i].clone(), k[2 * i + 1].clone(), table, length) for i in range(2)]
        return layers, attn.KvPages.all_free(layers[0]), attn.KvPlan.empty(B, rows, gpu)

    ws = torch.empty(attn.chunk_workspace_bytes(world()[0][0], rows, Hq), dtype=torch.uint8, device=gpu)
    assert ws.numel() > 0

    def step(layers, pages, plan):
        attn.kv_plan(layers[0], pages, want, plan=plan)
        outs = []
        for i, c in enumerate(layers):
            qkv = x[i].clone()
            attn.kv_append_rows(qkv, c, Hq, plan, rope=r, q=qkv)
            outs += [qkv, *attn.gqa_chunk(qkv, c, Hq, plan.row_start, plan.n_new, out=torch.zeros(rows, Hq * D, dtype=DT[dtype], device=gpu),
                                          lse=torch.zeros(rows, Hq, device=gpu), workspace=ws)]
        return outs

    def state(w):
        layers, pages, plan = w
        return [layers[0].table, layers[0].kv_len, pages.free[:int(pages.n_free)], pages.n_free, pages.held, plan.n_new, plan.row_start, plan.seq, plan.pos,
                plan.slot] + [t for c in layers for t in (c.k, c.v)]

    step(*world())
    worlds, graphs, outs = [world(), world()], [], []
    for w in worlds:
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(*w))
        graphs.append(g)
    eager = world()
    for i, n in enumerate([[60, 0, 30, 1, 0], [1, 50, 1, 1, 0], [0, 1, 1, 40, 1], [1, 1, 1, 1, 1], [20, 20, 20, 20, 20]]):
        want.copy_(i32(n, gpu))
        x.normal_()
        ref = step(*eager)
        torch.cuda.synchronize()
        for w, g, out in zip(worlds, graphs, outs):
            g.replay()
            torch.cuda.synchronize()
            for a, b in zip(out + state(w), ref + state(eager)):
                assert torch.equal(a, b), i
    assert int(eager[2].row_start[-1]) == 80       # of 100 rows in a plan of 96


def test_step_on_streams_of_their_own(gpu):
    """Chunks of one cache on streams of their own at once, and a step on a stream that is not the current one."""
    from tokamak_amd import attn
    case = Case(gpu, [3000, 777, 2048], 4, 64, 64, "bf16")
    n = i32([30, 9, 200], gpu)
    start = i32([0, 30, 39], gpu)
    qs = [queries(239, 16, 4, 64, "bf16", gpu, seed=s) for s in range(4)]
    ref = [attn.gqa_chunk(q, case.cache, 16, start, n) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    got = [attn.gqa_chunk(q, case.cache, 16, start, n, stream=s) for _ in range(4) for q, s in zip(qs, streams)]
    torch.cuda.synchronize()
    for i, (o, lse) in enumerate(got):
        assert torch.equal(o, ref[i % 4][0]) and torch.equal(lse, ref[i % 4][1])
    r, _ = rope_of(64, "halves", None)
    small = Case(gpu, [0, 0], 4, 64, 64, "bf16", spare=8, extra_pages=4)
    pages, x = attn.KvPages.all_free(small.cache), queries(50, 16, 4, 64, "bf16", gpu)
    rot = attn.rope_fwd(x, r, 16, 4, 64, pos=torch.arange(50, dtype=torch.int32, device=gpu) % 30)
    torch.cuda.synchronize()
    with torch.cuda.stream(streams[0]):
        plan = attn.kv_plan(small.cache, pages, i32([30, 20], gpu), rows=50)
        q = attn.kv_append_rows(x, small.cache, 16, plan, rope=r)
        o, lse = attn.gqa_chunk(q, small.cache, 16, plan.row_start, plan.n_new)
    torch.cuda.synchronize()
    assert torch.equal(q, rot[:, :16 * 64])
    for b, at in ((0, slice(0, 30)), (1, slice(30, 50))):
        small.k[b], small.v[b] = small.held(b)
        assert torch.equal(small.k[b].transpose(0, 1).reshape(-1, 256), rot[at, 1024:1280].cpu().double())
    check_chunk(small, [30, 20], [30, 20], q, o, lse, 16)


def test_step_beyond_32_bit_offsets(gpu):
    """A pool of 5 GB of K and as much of V, the sequences' pages at its end: the same results as from a small one."""
    from tokamak_amd import attn
    case = Case(gpu, [700, 90], 8, 128, 256, "bf16", weights=True, spare=4)
    c, n = case.cache, 9600
    shape = (n,) + tuple(c.k.shape[1:])
    big = attn.KvCache(torch.empty(shape, dtype=c.dtype, device=gpu), torch.empty(shape, dtype=c.dtype, device=gpu),
                       torch.where(c.table >= 0, c.table + (n - c.num_pages), c.table), c.kv_len.clone(), c.weight.clone())
    assert big.k.numel() * 2 > 4 << 30
    big.k[-c.num_pages:], big.v[-c.num_pages:] = c.k, c.v
    r, _ = rope_of(128, "pairs", None)
    for rows, want in ((3, [2, 1]), (1200, [40, 160])):
        x, got = queries(rows, 16, 8, 128, "bf16", gpu), []
        for one in (c, big):
            held = i32([(int(m) + 255) // 256 for m in one.kv_len], gpu)
            free = torch.zeros(one.num_pages, dtype=torch.int32, device=gpu)
            used = one.table[one.table >= 0].tolist()
            left = [p for p in range(one.num_pages - c.num_pages, one.num_pages) if p not in used]
            free[:len(left)] = i32(left, gpu)
            plan = attn.kv_plan(one, attn.KvPages(free, i32([len(left)], gpu), held), i32(want, gpu), rows=rows)
            assert plan.n_new.tolist() == want
            q = attn.kv_append_rows(x, one, 16, plan, rope=r)
            o, lse = attn.gqa_chunk(q, one, 16, plan.row_start, plan.n_new)
            total = sum(want)
            got.append((q[:total], o[:total], lse[:total], one.weight, one.kv_len, *case.held(0, one), *case.held(1, one)))
        for a, b in zip(*got):
            assert torch.equal(a, b)


@pytest.mark.parametrize("Hq,Hkv,D,dtype,window", [(4, 1, 128, "bf16", 0), (2, 2, 64, "f16", 0), (4, 2, 64, "bf16", 40000)])
def test_chunk_of_a_long_sequence(gpu, Hq, Hkv, D, dtype, window):
    from tokamak_amd import attn
    print(f"[case] long Hq{Hq} Hkv{Hkv} D{D} {dtype} window {window}", flush=True)
    lens, n_new = [131085, 5], [13, 2]
    case = Case(gpu, lens, Hkv, D, 256, dtype)
    q = queries(15, Hq, Hkv, D, dtype, gpu)
    o, lse = attn.gqa_chunk(q, case.cache, Hq, i32([0, 13], gpu), i32(n_new, gpu), window=window)
    check_chunk(case, lens, n_new, q, o, lse, Hq, window=window)


@pytest.mark.parametrize("layout,rot", [("halves", 64), ("halves", 40), ("halves", 18), ("halves", 126), ("pairs", 50)])
@pytest.mark.parametrize("rows", [5, 3000])
def test_rope_in_place_is_rope(gpu, layout, rot, rows):
    """In place as into another tensor, where the other sides of a pair come from a thread's neighbours, in rows that are
    further apart than they are long; the way back is the gradient's, up to two roundings."""
    from tokamak_amd import attn
    r = attn.Rope(rot, layout=layout)
    x = queries(rows, 6, 2, 128, "bf16", gpu)
    wide = torch.full((rows, 10 * 128 + 24), 3.0, dtype=torch.bfloat16, device=gpu)
    wide[:, :1280] = x
    y = attn.rope_fwd(x, r, 6, 2, 128, S=rows)
    assert attn.rope_fwd(wide[:, :1280], r, 6, 2, 128, S=rows, out=wide[:, :1280]) is not None
    assert torch.equal(wide[:, :1280], y) and (wide[:, 1280:] == 3.0).all()
    back = attn.rope_bwd(y, r, 6, 2, 128, S=rows).float().cpu()
    # a side is at most |x0| + |x1|, and so is the sum of both; each rounding is of that times 2^-8, twice and once more
    x = x.float().cpu()
    heads = x.reshape(rows, 10, 128)
    i = torch.arange(rot // 2)
    i0, i1 = (i, i + rot // 2) if layout == "halves" else (2 * i, 2 * i + 1)
    size = torch.zeros_like(heads)
    size[:, :8, i0] = size[:, :8, i1] = heads[:, :8, i0].abs() + heads[:, :8, i1].abs()
    assert ((back - x).abs() <= (2.0 ** -8 * 3.1 * size).reshape(x.shape)).all()


def test_the_binding_refuses(gpu):
    from tokamak_amd import attn
    case = Case(gpu, [5, 9], 1, 64, 64, "f16", spare=6, extra_pages=3)
    c, dt = case.cache, torch.int32
    n = c.num_pages

    def z(*shape, d=dt):
        return torch.zeros(*shape, dtype=d, device=gpu)

    for args in ((z(n, d=torch.int64), z(1), z(2)), (z(n), z(2), z(2)), (z(n), z(1), z(2, d=torch.int64))):
        with pytest.raises(ValueError, match="dtype|elements"):
            attn.KvPages(*args)
    slot = z(4, d=torch.int64)
    for args in ((z(2), z(2), z(4), z(4), slot), (z(2), z(3), z(3), z(4), slot), (z(2), z(3), z(4), z(5), slot), (z(2), z(3), z(4), z(4), z(4))):
        with pytest.raises(ValueError, match="dtype|elements"):
            attn.KvPlan(*args)
    plan, pages, want = attn.KvPlan.empty(2, 4, gpu), attn.KvPages.all_free(c), z(2)
    for pg, kw, match in ((pages, {}, "how many"), (pages, dict(rows=3, plan=plan), "4 rows"), (attn.KvPages(z(n), z(1), z(3)), dict(plan=plan), "2 sequences"),
                          (attn.KvPages(z(n - 1), z(1), z(2)), dict(plan=plan), "pages"), (pages, dict(plan=attn.KvPlan.empty(3, 4, gpu)), "2 sequences"),
                          (pages, dict(plan=plan, start=z(3)), "start")):
        with pytest.raises(ValueError, match=match):
            attn.kv_plan(c, pg, want, **kw)
    with pytest.raises(ValueError, match="want"):
        attn.kv_plan(c, pages, z(2, d=torch.int64), plan=plan)
    x = z(4, 3 * 64, d=torch.float16)
    for bad, match in ((x[:3], "plan must be"), (x[:, :128], "192"), (x.float(), "float16"), (z(192, 4, d=torch.float16).t(), "contiguous")):
        with pytest.raises(ValueError, match=match):
            attn.kv_append_rows(bad, c, 1, plan)
    with pytest.raises(ValueError, match="rows, expected"):
        attn.kv_append_rows(x, c, 1, plan, q=x[:2])
    for q, kw, match in ((x[0], {}, "rows"), (x, dict(row_start=z(1), n_new=z(2)), "row_start"), (x, dict(n_new=z(3)), "n_new"),
                         (x, dict(out=z(4, 128, d=torch.float16)), "out"), (x, dict(lse=z(4, d=torch.float16)), "lse"),
                         (x, dict(workspace=z(3, 2, d=torch.uint8).t()), "workspace")):
        with pytest.raises(ValueError, match=match):
            attn.gqa_chunk(q, c, 1, **kw)
    r = attn.Rope(64)
    for bad, kw, match in ((x, {}, "positions"), (x[:, :64], dict(S=4), "192"), (x, dict(pos=z(3)), "pos"), (x, dict(S=4, out=x[:3]), "rows, expected"),
                           (x, dict(pos=z(4, d=torch.int64)), "pos")):
        with pytest.raises(ValueError, match=match):
            attn.rope_fwd(bad, r, 1, 1, 64, **kw)
    assert case.held(0)[0].shape[1] == 5 and c.kv_len.tolist() == [5, 9]


@pytest.mark.parametrize("B,extra,dtype", [(1100, 20, "f16"), (2300, 40, "bf16")])
def test_chunk_of_many_sequences(gpu, B, extra, dtype):
    """More sequences, and items, than a workgroup has threads."""
    from tokamak_amd import attn
    print(f"[case] {B} sequences", flush=True)
    lens, n_new = [(7 * i) % 50 + 2 for i in range(B)], [i % 3 for i in range(B)]
    lens[B - 1], n_new[B - 1] = 900, 300
    case = Case(gpu, lens, 1, 64, 64, dtype, extra_pages=extra)
    q = queries(sum(n_new), 2, 1, 64, dtype, gpu)
    row_start = [sum(n_new[:b]) for b in range(B + 1)]
    for window in (0, 20):
        o, lse = attn.gqa_chunk(q, case.cache, 2, i32(row_start, gpu), i32(n_new, gpu), window=window)
        check_chunk(case, lens, n_new, q, o, lse, 2, window=window)


def test_chunk_of_rows_that_sequences_share(gpu):
    """Rows that several sequences name, which the call does not promise anything of, leave what is beside o, lse and the
    workspace alone."""
    from tokamak_amd import attn
    case = Case(gpu, [310] * 60, 2, 64, 64, "f16", extra_pages=20)
    q = queries(300, 4, 2, 64, "f16", gpu)
    need = attn.chunk_workspace_bytes(case.cache, 300, 4)
    assert need > 0
    ws = torch.full((need + 8192,), 0x5a, dtype=torch.uint8, device=gpu)
    out, lse = torch.full((340, 256), 4.0, dtype=torch.float16, device=gpu), torch.full((340, 4), 4.0, device=gpu)
    attn.gqa_chunk(q, case.cache, 4, i32([0] * 60, gpu), i32([300] * 60, gpu), out=out[20:320], lse=lse[20:320], workspace=ws[4096:4096 + need])
    assert (ws[:4096] == 0x5a).all() and (ws[4096 + need:] == 0x5a).all()
    for t in (out, lse):
        assert (t[:20] == 4.0).all() and (t[320:] == 4.0).all()
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("lens,n_new,Hq,Hkv,D,page,dtype,window", [
    ([1900, 700], [1900, 200], 32, 4, 64, 64, "bf16", 0), ([1000, 33, 0, 900, 1000], [1000, 1, 0, 500, 900], 16, 16, 128, 32, "f16", 0),
    ([5000, 3000, 64], [1200, 900, 3], 16, 2, 64, 128, "bf16", 300), ([2500, 1300], [1250, 1300], 24, 24, 64, 64, "f16", 1000)])
def test_chunk_of_many_rows_in_one_launch(gpu, lens, n_new, Hq, Hkv, D, page, dtype, window):
    """Prompts whose items are workgroups enough, and short enough, that none is split."""
    from tokamak_amd import attn
    print(f"[case] {lens} Hq{Hq} Hkv{Hkv} D{D} {dtype} window {window}", flush=True)
    case = Case(gpu, lens, Hkv, D, page, dtype)
    q = queries(sum(n_new), Hq, Hkv, D, dtype, gpu)
    row_start = [sum(n_new[:b]) for b in range(len(lens) + 1)]
    o, lse = attn.gqa_chunk(q, case.cache, Hq, i32(row_start, gpu), i32(n_new, gpu), window=window)
    assert attn.last_kernels() == ["chunk"]
    check_chunk(case, lens, n_new, q, o, lse, Hq, window=window)
