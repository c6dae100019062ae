"""Calls whose launches would have 2^32 threads or more, which HIP refuses: they are refused before anything is
launched.  A refused first kernel followed by the second would move tokens by positions that nothing wrote."""
import pytest

from test_kv_cpu import EUNSUPPORTED, P, append, decode, evict, kv, ref
from tokamak_amd import attn

OTHER = dict(table=9 * P, len=10 * P, weight=11 * P)


@pytest.mark.parametrize("kw,S", [(dict(B=1 << 24, Hkv=1), 1), (dict(B=1, Hkv=1), (1 << 29) - 30), (dict(B=1 << 12, Hkv=16), 1 << 13),
                                  (dict(B=1 << 24, Hkv=1), 2)])
def test_append(kw, S):
    assert append(kv(**kw), S=S, Hq=kw["Hkv"]) == EUNSUPPORTED
    assert b"grid" in attn.lib().tkm_attn_last_error() and attn.lib().tkm_attn_last_kernels() == 0


@pytest.mark.parametrize("kw,add", [
    (dict(B=1 << 23, Hkv=1), 0),                                              # a workgroup of 512 a row
    (dict(B=1 << 21, Hkv=1, page=256, max_pages=32), 1),                      # the weights, 1024 positions a workgroup
])
def test_decode(kw, add):
    c = kv(**kw)
    assert attn.lib().tkm_attn_decode_workspace_bytes(ref(c), kw["Hkv"], add) == 0
    assert decode(c, Hq=kw["Hkv"], stride=64, add=add, wsb=1 << 50) == EUNSUPPORTED
    assert b"grid" in attn.lib().tkm_attn_last_error() and attn.lib().tkm_attn_last_kernels() == 0


@pytest.mark.parametrize("kw,budget,place", [
    (dict(B=1 << 24, Hkv=1, max_pages=1), 1, 0),                              # choosing, 256 threads a row
    (dict(B=1 << 22, Hkv=1, page=256, max_pages=16), 200, 0),                 # choosing, 1024
    (dict(B=1 << 22, Hkv=1, page=256, max_pages=8), 2048, 1),                 # moving in place, 32 dims of K or V
    (dict(B=1 << 20, Hkv=1, page=256, max_pages=16), 4096, 0),                # moving, 256 tokens a workgroup
])
def test_evict(kw, budget, place):
    assert evict(kv(**kw), dst=None if place else kv(**{**kw, **OTHER}), budget=budget) == EUNSUPPORTED
    assert b"grid" in attn.lib().tkm_attn_last_error() and attn.lib().tkm_attn_last_kernels() == 0
