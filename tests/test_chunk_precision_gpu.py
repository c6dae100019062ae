"""The weights of gqa_chunk's second product on the GPU: as many bits as gqa_decode's, which reads the same cache."""
import math

import pytest
import torch

from kv_cases import DT, HALF, TINY, Case, blocks, decode_ref

pytestmark = pytest.mark.gpu

# two parts of fp16 hold 22 bits of a weight, three of bf16 its 24
PART = {"f16": 2.0 ** -22, "bf16": 2.0 ** -24}


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("Hq,Hkv,D,page,dtype", [(8, 2, 64, 32, "f16"), (8, 1, 64, 64, "bf16"), (4, 4, 128, 32, "f16"), (16, 2, 128, 64, "bf16")])
@pytest.mark.parametrize("extra", [0, 60])
def test_difference_of_two_weights(gpu, Hq, Hkv, D, page, dtype, extra):
    """Three tokens of scores 0, -d and c and values 1, -1 and 0: o = (1 - e^-d) / (1 + e^-d + e^c), a difference of weights
    that are alike in their first 14 bits.

    Bounds: the argument of an exponential is below 8 and rounded once, 2^-22 * ln 2 of a weight; the exponential itself is
    off by 2^-22 at most; then the parts' bits, PART.  Together below 3 * 2^-22 of each of the two weights (2^-22 (0.7 + 1 +
    1) in fp16).  The sums add 4 * 2^-24 of each, the quotient 2^-22 of o, which is rounded once on its way out."""
    from tokamak_amd import attn
    print(f"[case] Hq{Hq} Hkv{Hkv} D{D} page{page} {dtype} extra {extra}", flush=True)
    B, dt, g = 200, DT[dtype], torch.Generator().manual_seed(3)
    k, v = torch.zeros(Hkv, page, D), torch.zeros(Hkv, page, D)
    k[:, 1, 0], k[:, 2, 1] = -1.0, 1.0
    v[:, 0], v[:, 1] = 1.0, -1.0
    table = torch.zeros(B, 1 + extra, dtype=torch.int32, device=gpu)
    cache = attn.KvCache(blocks(k.to(dt), page, False).to(gpu), blocks(v.to(dt), page, True).to(gpu), table, i32([3] * B, gpu))
    q = torch.zeros(B, Hq, D)
    q[..., 0] = 2.0 ** (-18 + 4 * torch.rand(B, Hq, generator=g))
    q[..., 1] = 0.3 + 1.7 * torch.rand(B, Hq, generator=g)
    q = q.to(dt)
    o, lse = attn.gqa_chunk(q.reshape(B, Hq * D).to(gpu), cache, Hq, scale=1.0)
    s = torch.stack((torch.zeros(B, Hq, dtype=torch.float64), -q[..., 0].double(), q[..., 1].double()))
    top = torch.logsumexp(s, 0)
    w = torch.exp(s - top)
    ref = (torch.expm1(s[0] - s[1]) * w[1])[..., None]
    tol = (w[0] + w[1])[..., None] * (3 * 2.0 ** -22 + 4 * 2.0 ** -24) + (HALF[dtype] + 2.0 ** -22) * ref.abs() + TINY[dtype]
    worst = ((o.cpu().double().reshape(B, Hq, D) - ref).abs() / tol).max().item()
    print(f"    o {worst:.3f} of its bound", flush=True)
    assert worst <= 1.0
    assert ((lse.cpu().double() - top).abs() <= 2.0 ** -20 * (1 + top.abs())).all()


@pytest.mark.parametrize("Hq,Hkv,D,page,dtype", [(8, 2, 64, 32, "f16"), (12, 4, 128, 64, "f16"), (3, 1, 64, 256, "bf16"), (16, 2, 128, 32, "bf16")])
@pytest.mark.parametrize("extra", [1, 200])
@pytest.mark.parametrize("window", [0, 100])
def test_rows_have_the_precision_of_decoding(gpu, Hq, Hkv, D, page, dtype, extra, window):
    """Drafts, prompts and single rows against gqa_decode's bounds (kv_cases.decode_ref), which leave 2^-21 for the parts of
    a weight; and the single rows against gqa_decode itself, within both calls' bounds."""
    from tokamak_amd import attn
    print(f"[case] Hq{Hq} Hkv{Hkv} D{D} page{page} {dtype} extra {extra} window {window}", flush=True)
    lens, n_new = [700, 2049, 96, 40, 1300], [1, 60, 17, 40, 1]
    case = Case(gpu, lens, Hkv, D, page, dtype, extra_pages=extra)
    total, scale = sum(n_new), 1.0 / math.sqrt(D)
    q = torch.randn(total, Hq * D, generator=torch.Generator().manual_seed(5)).to(DT[dtype])
    row_start = [sum(n_new[:b]) for b in range(len(lens) + 1)]
    o, lse = attn.gqa_chunk(q.to(gpu), case.cache, Hq, i32(row_start, gpu), i32(n_new, gpu), window=window)
    ks, vs = [], []
    for b, (length, n) in enumerate(zip(lens, n_new)):
        for i in range(n):
            hi = length - n + i + 1
            lo = max(0, hi - window) if window else 0
            ks.append(case.k[b][:, lo:hi])
            vs.append(case.v[b][:, lo:hi])
    ro, rl, _, eo, el = decode_ref(q.double().reshape(total, Hq, D), ks, vs, Hkv, scale)
    go, gl = o.cpu().double().reshape(total, Hq, D), lse.cpu().double()
    tol = eo + HALF[dtype] * (ro.abs() + eo) + TINY[dtype]
    worst, worst_l = ((go - ro).abs() / tol).max().item(), ((gl - rl).abs() / el).max().item()
    print(f"    o {worst:.3f}, lse {worst_l:.3f} of their bounds", flush=True)
    assert worst <= 1.0 and worst_l <= 1.0
    if not window:
        alone = torch.stack([q[row_start[b]] if n_new[b] == 1 else torch.zeros(Hq * D, dtype=DT[dtype]) for b in range(len(lens))])
        d, dl = attn.gqa_decode(alone.to(gpu), case.cache, Hq)
        for b in (0, 4):
            r = row_start[b]
            assert ((d[b].cpu().double().reshape(Hq, D) - go[r]).abs() <= 2 * tol[r]).all()
            assert ((dl[b].cpu().double() - gl[r]).abs() <= 2 * el[r]).all()
