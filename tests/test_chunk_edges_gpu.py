"""gqa_chunk on the GPU at the ends of its arguments' ranges, and with infinite values, against the operator in 64 bits."""
import math

import pytest
import torch

from kv_cases import DT, HALF, TINY, Case
from step_cases import check_chunk
from test_kv_odd_values_gpu import LENS, formula, plant, same_kind

pytestmark = pytest.mark.gpu

INT_MAX = (1 << 31) - 1


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def randn(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(DT[dtype])


@pytest.mark.parametrize("Hq,Hkv,D,page,dtype", [(4, 2, 64, 32, "f16"), (16, 2, 128, 64, "bf16"), (7, 1, 64, 64, "bf16")])
@pytest.mark.parametrize("extra", [1, 60])
def test_windows_as_wide_as_an_int(gpu, Hq, Hkv, D, page, dtype, extra):
    """A window of all that a table holds or more is none, also for sequences of more rows than tokens, whose first rows
    stand before position 0 and see nothing."""
    from tokamak_amd import attn
    print(f"[case] Hq{Hq} Hkv{Hkv} D{D} page{page} {dtype} extra {extra}", flush=True)
    lens, n_new = [50, 20, 0, 300], [60, 23, 4, 7]
    case = Case(gpu, lens, Hkv, D, page, dtype, extra_pages=extra)
    total, cap = sum(n_new), case.max_pages * page
    q = randn((total, Hq * D), dtype, 1).to(gpu)
    where = i32([sum(n_new[:b]) for b in range(5)], gpu), i32(n_new, gpu)
    o, lse = attn.gqa_chunk(q, case.cache, Hq, *where)
    check_chunk(case, lens, n_new, q, o, lse, Hq)
    for window in (INT_MAX, INT_MAX - 1, 1 << 30, cap + 1, cap):
        wo, wl = attn.gqa_chunk(q, case.cache, Hq, *where, window=window)
        assert torch.equal(wo, o) and torch.equal(wl, lse), window
    for window in (301, 300, 294, 293, 20):      # ends inside the sequences
        check_chunk(case, lens, n_new, q, *attn.gqa_chunk(q, case.cache, Hq, *where, window=window), Hq, window=window)


@pytest.mark.parametrize("D,dtype,G", [(64, "f16", 3), (128, "bf16", 33), (64, "bf16", 8), (128, "f16", 2)])
@pytest.mark.parametrize("cap,window", [("tight", 0), ("tight", 200), ("wide", 0), ("wide", 500)])
@pytest.mark.parametrize("q0", ["up", "mixed"])
def test_infinities_are_those_of_decoding(gpu, D, dtype, G, cap, window, q0):
    """Infinities and NaN among keys and values go where the formula takes them, in tiles that all rows see and in those on
    an edge, in calls of one launch and of three: which outputs are NaN, or infinite, agrees with gqa_decode's formula for
    each row over what it sees, and the others are within its bounds."""
    from tokamak_amd import attn
    print(f"[case] D{D} {dtype} G{G} {cap} window {window} {q0}", flush=True)
    Hkv, Hq, scale = 2, 2 * G, 1.0 / math.sqrt(D)
    lens, n_new = LENS[cap], [1, 3, 9, 4, 1, 13, 5, 2]
    case = Case(gpu, lens, Hkv, D, 64, dtype, extra_pages=100 if cap == "wide" else 0)
    plant(case)
    total, row_start = sum(n_new), [sum(n_new[:b]) for b in range(len(lens) + 1)]
    q = randn((total, Hkv, G, D), dtype, G)
    q[..., 0] = 0.5
    if q0 == "mixed":
        q[:, :, 1, 0] = -0.5         # -inf keys give +inf
        if G > 2:
            q[:, :, 2, 0] = 0.0      # and 0 * inf = NaN
    o, lse = attn.gqa_chunk(q.reshape(total, -1).to(gpu), case.cache, Hq, i32(row_start, gpu), i32(n_new, gpu), window=window)
    assert window or ("join" in attn.last_kernels()) == (cap == "wide")       # a window can make items short
    o, lse = o.cpu().double().reshape(total, Hkv, G, D), lse.cpu().double().reshape(total, Hkv, G)
    worst = [0.0, 0.0]
    for b, n in enumerate(n_new):
        for i in range(n):
            r, up = row_start[b] + i, lens[b] - n + i + 1
            lo = max(0, up - window) if window else 0
            for h in range(Hkv):
                ro, rl, _, eo, el, _ = [x.cpu() for x in formula(*(x.to(gpu) for x in (q[r, h].double(), case.k[b][h, lo:up], case.v[b][h, lo:up])), scale)]
                assert same_kind(lse[r, h], rl), (b, i, h)
                assert same_kind(o[r, h], ro), (b, i, h, torch.nonzero(o[r, h].isnan() != ro.isnan()).tolist()[:9])
                some = torch.isfinite(ro)
                worst[0] = max([worst[0], *((o[r, h] - ro).abs() / (eo + HALF[dtype] * (ro.abs() + eo) + TINY[dtype]))[some].tolist()])
                worst[1] = max([worst[1], *((lse[r, h] - rl).abs() / el)[torch.isfinite(rl)].tolist()])
    print("    o %.3f, lse %.3f of their bounds" % tuple(worst), flush=True)
    assert max(worst) <= 1.0


@pytest.mark.parametrize("Hq,Hkv,D,page,dtype", [(4, 2, 64, 32, "f16"), (16, 2, 128, 64, "bf16")])
@pytest.mark.parametrize("extra", [1, 60])
def test_padded_rows_are_clamped(gpu, Hq, Hkv, D, page, dtype, extra):
    """A batch of S rows a sequence, of which n_new says more: S of them, as kv_append stores them, and none of the next
    sequence's."""
    from tokamak_amd import attn
    print(f"[case] Hq{Hq} Hkv{Hkv} D{D} page{page} {dtype} extra {extra}", flush=True)
    lens, S = [100, 33, 400, 20], 11
    case = Case(gpu, lens, Hkv, D, page, dtype, extra_pages=extra)
    q = randn((4 * S, Hq * D), dtype, 2).to(gpu)
    o, lse = attn.gqa_chunk(q, case.cache, Hq)
    check_chunk(case, lens, [S] * 4, q, o, lse, Hq)
    for n in ([S + 1] * 4, [4 * S, INT_MAX, S, S + 5], [INT_MAX] * 4):
        for _ in range(3):
            co, cl = attn.gqa_chunk(q, case.cache, Hq, n_new=i32(n, gpu))
            assert torch.equal(co, o) and torch.equal(cl, lse), n
    out = torch.full_like(o, 4.0)
    co, cl = attn.gqa_chunk(q, case.cache, Hq, n_new=i32([S + 9, -3, 5, INT_MAX], gpu), out=out)
    check_chunk(case, lens, [S, 0, 5, S], q, co, cl, Hq, row_start=[0, S, 2 * S, 3 * S])
    assert (out[S:2 * S] == 4.0).all() and (out[2 * S + 5:3 * S] == 4.0).all()
