"""The weights of a decoding step at scales that make the scores flat, ordinary, or so steep that a few positions of a
row gather everything and most get exactly 0."""
import pytest
import torch

from kv_cases import HALF, TINY, Case
from test_kv_odd_values_gpu import formula

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [1e-6, 0.02, 3.0, 40.0])
@pytest.mark.parametrize("extra", [1, 200])
@pytest.mark.parametrize("D,dtype", [(64, "f16"), (128, "bf16")])
def test_weights(gpu, scale, extra, D, dtype):
    """Positions whose exp(score - LSE) is below fp32's 2^-126 may get 0 (extra = 200: the split form)."""
    from tokamak_amd import attn
    lens, G, Hkv = [70, 1000, 1, 0], 4, 2
    case = Case(gpu, lens, Hkv, D, 32, dtype, weights=True, extra_pages=extra)
    g = torch.Generator().manual_seed(9)
    q = torch.randn(4, Hkv, G, D, generator=g).to(case.cache.dtype)
    o, lse = attn.gqa_decode(q.reshape(4, -1).to(gpu), case.cache, Hkv * G, scale=scale, add_weights=True)
    o, lse = o.cpu().double().reshape(4, Hkv, G, D), lse.cpu().double().reshape(4, Hkv, G)
    got, worst = case.cache.weight.cpu().double(), [0.0, 0.0, 0.0]
    for b, n in enumerate(lens):
        for h in range(Hkv if n else 0):
            ro, rl, rw, eo, el, ew = formula(q[b, h].double(), case.k[b][h], case.v[b][h], float(torch.tensor(scale, dtype=torch.float32)))
            ref = case.weight[b, h, :n].double() + rw
            off = ((o[b, h] - ro).abs() / (eo + HALF[dtype] * (ro.abs() + eo) + TINY[dtype])).max().item()
            off_w = ((got[b, h, :n] - ref).abs() / (ew + 2.0 ** -23 * ref + G * 2.0 ** -126)).max().item()
            worst = [max(x, y) for x, y in zip(worst, (off, ((lse[b, h] - rl).abs() / el).max().item(), off_w))]
        assert torch.equal(got[b, :, n:], case.weight[b, :, n:].double())
    print("    o %.3f, lse %.3f, weights %.3f of their bounds" % tuple(worst), flush=True)
    assert max(worst) <= 1.0
