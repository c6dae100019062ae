"""gqa_chunk on the GPU at the ends of its arguments' ranges, and with infinite values, against the operator in 64 bits."""
import math

import pytest
import torch

from kv_cases import DT, Case
from step_cases import check_chunk

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
