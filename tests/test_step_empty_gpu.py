"""A serving step without rows, on the GPU: sequences end, and no call of the step is refused."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rope", [False, True])
def test_step_without_rows(gpu, rope):
    from tokamak_amd import attn
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)
    Hq, Hkv, D = 4, 2, 64
    cache = attn.KvCache.empty(2, 40, 5, Hkv, D, page=32, device=gpu)
    pages = attn.KvPages.all_free(cache)
    assert attn.kv_plan(cache, pages, i32([40, 3]), rows=50).n_new.tolist() == [40, 3]
    plan = attn.kv_plan(cache, pages, i32([0, 0]), rows=0, start=i32([0, 0]))
    assert pages.n_free.tolist() == [5] and plan.row_start.tolist() == [0, 0, 0] and cache.kv_len.tolist() == [0, 0]
    x = torch.empty(0, (Hq + 2 * Hkv) * D, dtype=torch.float16, device=gpu)
    q = attn.kv_append_rows(x, cache, Hq, plan, rope=attn.Rope(D) if rope else None)
    for row_start, n_new in ((plan.row_start, plan.n_new), (None, None)):
        o, lse = attn.gqa_chunk(q, cache, Hq, row_start, n_new)
        assert o.shape == (0, Hq * D) and lse.shape == (0, Hq) and o.dtype == torch.float16
    with pytest.raises(ValueError):
        attn.gqa_chunk(q, cache, Hq, plan.row_start, i32([0, 0, 0]))
