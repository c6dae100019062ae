"""kv_append_rows in place through a view of the Q heads, on the GPU."""
import pytest
import torch

from kv_cases import DT

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 2, 5])
@pytest.mark.parametrize("rot", [0, 64])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_view_of_the_query_heads(gpu, rows, rot, dtype):
    """q is the rows' own Q heads: they are rotated where they are, as in a tensor of their own, K and V stay."""
    from tokamak_amd import attn
    print(f"[case] rows {rows} rot {rot} {dtype}", flush=True)
    Hq, Hkv, D, W = 4, 2, 64, 8 * 64
    cache = attn.KvCache.empty(1, 2, 2, Hkv, D, page=32, dtype=DT[dtype], device=gpu)
    plan = attn.kv_plan(cache, attn.KvPages.all_free(cache), torch.tensor([rows], dtype=torch.int32, device=gpu), rows=rows)
    rope = attn.Rope(rot) if rot else None
    x = torch.randn(rows, W, generator=torch.Generator().manual_seed(rows)).to(DT[dtype]).to(gpu)
    want = torch.zeros(rows, Hq * D, dtype=DT[dtype], device=gpu)
    attn.kv_append_rows(x, cache, Hq, plan, rope=rope, q=want)
    k, v = cache.k.clone(), cache.v.clone()
    for wide in (x.clone(), torch.cat((x, x), 1)[:, :W]):         # rows of the heads' width, and further apart
        view = wide[:, :Hq * D]
        assert attn.kv_append_rows(wide, cache, Hq, plan, rope=rope, q=view) is view
        assert torch.equal(wide[:, :Hq * D], want) and torch.equal(wide[:, Hq * D:], x[:, Hq * D:])
        assert torch.equal(cache.k[0, :, 0, :, :rows], k[0, :, 0, :, :rows]) and torch.equal(cache.v[0, :, 0, :, :, :rows], v[0, :, 0, :, :, :rows])
