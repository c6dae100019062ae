"""Sequences that share the pages of a common beginning, which are only read, against the same sequences with pages of
their own, bit for bit: decoding, rows appended behind the shared part, eviction into another table."""
import pytest
import torch

from kv_cases import DT, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,dtype,extra", [(64, "f16", 0), (128, "bf16", 120)])
def test_shared_beginning(gpu, D, dtype, extra):
    from tokamak_amd import attn
    page, Hkv, Hq, B, pages = 32, 2, 6, 4, 5
    case = Case(gpu, [5 * page], Hkv, D, page, dtype, spare=40)
    k, v, first = case.cache.k, case.cache.v, case.cache.table[0, :3]
    k[case.free], v[case.free] = torch.randn_like(k[case.free].float()).to(k.dtype), torch.randn_like(v[case.free].float()).to(v.dtype)
    spare = case.free.to(torch.int32).to(gpu)
    shared, own = (torch.full((B, pages + extra), -1, dtype=torch.int32, device=gpu) for _ in range(2))
    shared[:, :3], own[0, :3] = first, first             # three pages of the beginning, for all
    shared[:, 3:5] = own[:, 3:5] = spare[:2 * B].reshape(B, 2)
    own[1:, :3] = spare[2 * B:2 * B + 3 * (B - 1)].reshape(B - 1, 3)
    lens = torch.tensor([96, 100, 128, 97], dtype=torch.int32, device=gpu)
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(B, 7, (Hq + 2 * Hkv) * D, generator=g).to(DT[dtype]).to(gpu)
    got = []
    for table in (shared, own):
        pool = [x.clone() for x in (k, v)]
        for x in pool:
            x[own[1:, :3].long()] = x[first.long()].unsqueeze(0)
        w = torch.zeros(B, Hkv, (pages + extra) * page, device=gpu)
        c = attn.KvCache(pool[0], pool[1], table.clone(), lens.clone(), w)
        attn.kv_append(qkv, c, Hq)
        o, lse = attn.gqa_decode(qkv[:, 6], c, Hq, add_weights=True)
        d = attn.KvCache.empty(B, 3, 3 * B, Hkv, D, page, DT[dtype], gpu, weights=True)
        d.table.copy_(torch.arange(3 * B).reshape(B, 3).to(torch.int32))
        kept = attn.kv_evict(c, 70, sink=2, recent=9, dst=d)
        at = torch.arange(70, device=gpu)
        K = d.k[d.table.long()][:, at // page, :, 0, :, at % page]
        V = d.v[d.table.long()][:, at // page, :, 0, :, :, at % page]
        got.append((o, lse, w, kept, d.kv_len, d.weight[:, :, :70], K, V, c.kv_len))
    assert got[0][8].tolist() == [103, 107, 135, 104]
    for x, y in zip(*got):
        assert torch.equal(x, y)
