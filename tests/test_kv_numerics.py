"""How exactly a decoding step holds the softmax weights P between its two products: keys whose P are the worst for a
split into 16-bit parts, and values that cancel, so that the output is small and shows the error of the sums alone."""
import pytest
import torch

from kv_cases import DT, HALF, TINY, blocks


def two_parts(p, dt):
    """What is left of fp32 p behind two 16-bit parts, relative to p."""
    hi = p.to(dt).float()
    return ((p - hi) - (p - hi).to(dt).float()).double() / p.double()


def worst_scores(dt, n):
    """Scores in (-0.69, 0) that dt holds, whose P = 64 exp(score) leave most behind two bf16 parts: n that leave a
    positive rest and n a negative one.  P is off by 1.6 * 2^-22 at most where it is computed in fp32 (see the bound
    below): scores are taken whose neighbours at +-2^-21 leave as much."""
    s = -torch.arange(1, 177, dtype=torch.float64) / 256
    s = s[s.to(dt).double() == s]
    p = torch.exp(s) * 64
    rests = torch.stack([two_parts((p * (1 + d)).float(), torch.bfloat16) for d in (-2.0 ** -21, 0.0, 2.0 ** -21)])
    low, high = rests.amin(0), rests.amax(0)
    return s[low.argsort(descending=True)[:n]], s[high.argsort()[:n]]


def cancelling(dt, Hkv, D, seed):
    """K and V [Hkv, 7, D] of a sequence and the scores [7] that a query (1, 0, 0, ..) gives: two keys whose P leave a
    positive rest with positive values, two that leave a negative one with negative values, and three of score 0 (a P
    of one bit) that take the sum away, each to half a step of what the one before left."""
    g = torch.Generator().manual_seed(seed)
    up, down = worst_scores(dt, 2)
    s = torch.cat((up, down, torch.zeros(3, dtype=torch.float64)))
    v = (1 + torch.rand(Hkv, 7, D, generator=g)).to(dt).double()
    v[:, 2:4] *= -1
    p = torch.exp(s)[:, None]
    for i in range(4, 7):
        v[:, i] = (-(p[:i] * v[:, :i]).sum(1)).to(dt).double()
    k = torch.zeros(Hkv, 7, D, dtype=torch.float64)
    k[:, :, 0] = s
    order = torch.randperm(7, generator=g)
    return k[:, order], v[:, order], s[order]


def test_two_bf16_parts_of_p_are_not_enough():
    """Such P lose over 1.3 * 2^-18 of themselves, each to the side that its value adds up on: together more than the
    bound below, 0.82 * 2^-18 of the sum of absolute values."""
    for dt in DT.values():
        up, down = worst_scores(dt, 2)
        for s, sign in ((up, 1), (down, -1)):
            assert (sign * two_parts((torch.exp(s) * 64).float(), torch.bfloat16)).min() > 1.3 * 2.0 ** -18
        k, v, s = cancelling(dt, 3, 64, 0)
        p = torch.exp(s)[:, None] * 64
        rest = (two_parts(p.float(), torch.bfloat16) * p * v).sum(1).abs() / (p * v.abs()).sum(1)
        assert rest.min() > 1.1 * 2.0 ** -18
        assert ((p * v).sum(1).abs() / (p * v.abs()).sum(1)).max() < 2.0 ** -24


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv,D", [(2, 2, 64), (8, 2, 128), (20, 1, 128), (70, 1, 64)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("pages", [1, 200])
@pytest.mark.parametrize("add", [False, True])
def test_p_keeps_the_bits_of_fp32(gpu, Hq, Hkv, D, dtype, pages, add):
    """The bound, relative to sum p |v| / sum p.  Scores are exact; their factor log2(e) and the product with it are
    rounded (2 * 0.69 * 2^-24), the difference to the maximum too (half a step of [4, 8), times ln 2: 0.69 * 2^-22),
    exp2 is good to 2^-23: 1.54 * 2^-22, and P's parts leave 2^-22 at most (fp16's two): 0.16 * 2^-18.  Seven tokens
    of up to three parts are added in fp32, 2^-23 an addition however it rounds: 0.66 * 2^-18.  Then the output's own
    rounding."""
    from tokamak_amd import attn
    dt = DT[dtype]
    k, v, s = cancelling(dt, Hkv, D, Hq)
    pool = torch.zeros(2, 1, Hkv, 1, D // 32, 32, 32, dtype=dt)
    for i, x in enumerate((k, v)):
        full = torch.zeros(Hkv, 32, D, dtype=torch.float64)
        full[:, :7] = x
        pool[i] = blocks(full, 32, i == 1).to(dt)
    table = torch.zeros(1, pages, dtype=torch.int32, device=gpu)      # many pages: the split form
    cache = attn.KvCache(pool[0].to(gpu), pool[1].to(gpu), table, torch.full((1,), 7, dtype=torch.int32, device=gpu),
                         torch.zeros(1, Hkv, pages * 32, device=gpu))
    q = torch.zeros(1, Hq, D, dtype=dt, device=gpu)
    q[:, :, 0] = 1
    o, _ = attn.gqa_decode(q.reshape(1, Hq * D), cache, Hq, scale=1.0, add_weights=add)
    p = torch.softmax(s, 0)[:, None]
    ref, size = (p * v).sum(1, keepdim=True), (p * v.abs()).sum(1, keepdim=True)      # [Hkv, 1, D]
    got = o.cpu().double().reshape(Hkv, Hq // Hkv, D)
    worst = ((got - ref).abs() / (0.82 * 2.0 ** -18 * size + HALF[dtype] * ref.abs() + TINY[dtype])).max().item()
    print(f"    {worst:.3f} of the bound", flush=True)
    assert worst <= 1.0
