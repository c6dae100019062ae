"""Attention of one new token over caches that hold infinities and NaN among a sequence's own keys and values, against
the formula in 64 bits: which outputs are NaN or infinite has to agree, the others within kv_cases' bounds, and so the
weights.  Each sequence has a kv head with odd values and one without, whose results show that nothing else is reached."""
import math

import pytest
import torch

from kv_cases import HALF, TINY, Case, blocks

pytestmark = pytest.mark.gpu
inf, nan = float("inf"), float("nan")
LENS = {"tight": [300, 250, 600, 333, 500, 610, 611, 97], "wide": [700, 650, 2100, 333, 500, 900, 611, 97]}


def formula(q, k, v, scale):
    """o [G, D], lse [G], weights [n] and bounds on their errors (kv_cases.decode_ref, of the finite values alone) for
    q [G, D], k and v [n, D], all fp64."""
    n, D = k.shape
    s = (q[:, None] * k[None]).sum(2) * scale
    m = s.amax(1, keepdim=True)
    m = torch.where(m == -inf, torch.zeros_like(m), m)
    p = torch.exp(s - m)
    total = p.sum(1, keepdim=True)
    lse = (m + torch.log(total))[:, 0]
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    o = (p[:, :, None] * v[None]).sum(1)
    kz, vz, pz, sz, lz = (x.nan_to_num(0.0, 0.0, 0.0) for x in (k, v, p, s, lse))
    ds = ((D + 2) * 2.0 ** -24 * scale * (q.abs() @ kz.abs().T) + 2.0 ** -23 * sz.abs()).amax(1) + 8 * 2.0 ** -23
    el = ds + n * 2.0 ** -24 + 4 * 2.0 ** -24 * (lz.abs() + 16)
    eo = (2 * ds + n * 2.0 ** -23 + 2.0 ** -21)[:, None] * (pz @ vz.abs())
    some = torch.isfinite(lse)[:, None]
    w = torch.where(some, pz, torch.zeros_like(pz))
    return o, lse, w.sum(0), eo, el, ((ds + el + 2.0 ** -21)[:, None] * w).sum(0)


def plant(case):
    """The odd values, into case.k and case.v (fp64) of each sequence's kv head 0 or 1; q's dim 0 is the caller's."""
    for b in range(1, case.B):
        h, n, k, v = b % 2, case.lens[b], case.k[b], case.v[b]
        if b == 1:
            k[h, :, 0] = -inf                        # every score -inf, or (with q0 < 0) +inf
        elif b == 2:
            k[h, : n // 2, 0] = -inf                 # whole tiles and pieces of -inf ahead of ordinary ones
        elif b == 3:
            k[h, n // 3:, 0] = -inf                  # and behind them
        elif b == 4:
            k[h, 77, 3] = nan
        elif b == 5:
            v[h, 40, 5], v[h, n - 1, 6] = inf, -inf
            v[h, 40, 7], v[h, 590, 7] = inf, -inf
            v[h, 123, 8], v[h, 124, 9], v[h, 600, 9] = nan, nan, inf
            v[h, ::2, 10] = inf                      # many of them
            v[h, :, 11] = -inf
        elif b == 6:
            k[h, 10:300, 0] = -inf
            v[h, 11, 5] = inf                        # 0 * inf
            v[h, 12, 6], v[h, 500, 6] = inf, inf     # and once more with an ordinary score
            v[h, 400, 7] = -inf
        else:
            k[h, n - 1, 0], v[h, n - 2, 1] = -inf, inf
            v[h, n - 1, 2] = 1.0
    for b in range(case.B):                          # to the device
        pages = case.cache.table[b, :(case.lens[b] + case.page - 1) // case.page].long()
        for pool, x, isv in ((case.cache.k, case.k[b], False), (case.cache.v, case.v[b], True)):
            full = torch.full((case.Hkv, len(pages) * case.page, case.D), nan, dtype=torch.float64)
            full[:, :case.lens[b]] = x
            pool[pages] = blocks(full, case.page, isv).to(pool.dtype).to(pool.device)


def same_kind(got, ref):
    return torch.equal(got.isnan(), ref.isnan()) and torch.equal(got == inf, ref == inf) and torch.equal(got == -inf, ref == -inf)


@pytest.mark.parametrize("D,dtype", [(64, "f16"), (128, "bf16"), (64, "bf16")])
@pytest.mark.parametrize("G", [3, 33, 70])
@pytest.mark.parametrize("cap,add", [("tight", False), ("tight", True), ("wide", False), ("wide", True)])
@pytest.mark.parametrize("q0", ["up", "mixed"])
def test_formula(gpu, D, dtype, G, cap, add, q0):
    """tight: tables for which a workgroup has a row, of up to 64 query heads; wide: the split form, joined by workgroups,
    or by waves where there are over 512 query heads."""
    from tokamak_amd import attn
    Hkv, Hq, scale = 2, 2 * G, 1.0 / math.sqrt(D)
    case = Case(gpu, LENS[cap], Hkv, D, 64, dtype, weights=True, extra_pages=100 if cap == "wide" else 0)
    plant(case)
    g = torch.Generator().manual_seed(G)
    q = torch.randn(case.B, Hkv, G, D, generator=g).to(case.cache.dtype)
    q[..., 0] = 0.5
    if q0 == "mixed":
        q[:, :, 1, 0], q[:, :, 2, 0] = -0.5, 0.0     # -inf keys give +inf and 0 * inf = NaN
    o, lse = attn.gqa_decode(q.reshape(case.B, -1).to(gpu), case.cache, Hq, add_weights=add)
    kinds = attn.last_kernels()
    assert ("join" in kinds) == (cap == "wide" or G > 64), kinds
    o, lse = o.cpu().double().reshape(case.B, Hkv, G, D), lse.cpu().double().reshape(case.B, Hkv, G)
    weight, worst = case.cache.weight.cpu().double(), [0.0, 0.0, 0.0]
    for b in range(case.B):
        for h in range(Hkv):
            n = case.lens[b]
            ro, rl, rw, eo, el, ew = [x.cpu() for x in formula(*(x.to(gpu) for x in (q[b, h].double(), case.k[b][h], case.v[b][h])), scale)]
            assert same_kind(lse[b, h], rl), (b, h)
            assert same_kind(o[b, h], ro), (b, h, torch.nonzero(o[b, h].isnan() != ro.isnan()).tolist()[:9])
            d, some = (o[b, h] - ro).abs(), torch.isfinite(ro)
            worst[0] = max([worst[0], *(d / (eo + HALF[dtype] * (ro.abs() + eo) + TINY[dtype]))[some].tolist()])
            worst[1] = max([worst[1], *((lse[b, h] - rl).abs() / el)[torch.isfinite(rl)].tolist()])
            before = case.weight[b, h].double()
            if add:
                ref = before[:n] + rw
                worst[2] = max(worst[2], ((weight[b, h, :n] - ref).abs() / (ew + 2.0 ** -23 * ref + 1e-30)).max().item())
                assert torch.equal(weight[b, h, n:], before[n:])
            else:
                assert torch.equal(weight[b, h], before)
    print("    o %.3f, lse %.3f, weights %.3f of their bounds" % tuple(worst), flush=True)
    assert max(worst) <= 1.0
