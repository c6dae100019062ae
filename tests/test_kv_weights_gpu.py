"""What a position has gathered is large and what a step adds is small: the query heads' weights are summed before they
are added, so that the sum is rounded once, and none of them is lost to the size of what it is added to."""
import pytest
import torch

from kv_cases import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,D", [(2500, 64), (600, 128), (5000, 64), (9000, 128)])
@pytest.mark.parametrize("G", [4, 32, 70])
def test_small_weights_add_up(gpu, n, D, G):
    """Queries of zeros weigh all n positions alike, exactly 1/n a head, which alone is under half a step of what is
    there already.  A head's weight is off by 8 * 2^-23 of itself (the bound of LSE and exp2 in kv_cases.py) and n 2^-24
    (the sum of n), the heads' sum by 2^-24 a head, and the result by half a step."""
    from tokamak_amd import attn
    big = 2.0 ** (24 - int(n).bit_length() + 2)         # half a step of it is 4 / 2^bit_length(n), over 1/n
    case = Case(gpu, [n, 1, 0], 2, D, 32, "f16", weights=True, extra_pages=0 if n <= 2500 else 300)
    case.cache.weight.fill_(big)
    q = torch.zeros(3, 2 * G * D, dtype=torch.float16, device=gpu)
    attn.gqa_decode(q, case.cache, 2 * G, add_weights=True)
    assert ("join" in attn.last_kernels()) == (n > 2500 or G > 64)
    got = case.cache.weight.cpu().double()
    for b, k in ((0, n), (1, 1)):
        w = G / k
        bound = (8 * 2.0 ** -23 + (k + G) * 2.0 ** -24) * w + 2.0 ** -24 * big
        print(f"    {k}: off by {(got[b, :, :k] - (big + w)).abs().max().item() / bound:.3f} of the bound", flush=True)
        assert ((got[b, :, :k] - (big + w)).abs() <= bound).all()
        assert (got[b, :, k:] == big).all()
