"""The paged key-value cache's entry points without a GPU: what they refuse before anything is launched, and the
helpers that the GPU tests compare with."""
import ctypes

import pytest
import torch

from kv_cases import blocks, decode_ref, dense, evict_ref
from tokamak_amd import attn

OK, EINVAL, EUNSUPPORTED, EALIGN, EWORKSPACE = 0, -1, -2, -3, -4
P = 0x10000                     # aligned fake device addresses: nothing below reaches a HIP call


def kv(**kw):
    c = dict(k=P, v=2 * P, table=3 * P, len=4 * P, weight=5 * P, B=2, Hkv=2, D=64, page=64, max_pages=4, num_pages=8, dtype=0)
    c.update(kw)
    return attn._Kv(*(c[n] for n, _ in attn._Kv._fields_))


def ref(c):
    return None if c is None else ctypes.byref(c)


def append(c, qkv=P, S=3, Hq=4, start=None, n_new=None):
    return attn.lib().tkm_attn_kv_append(ref(c), qkv, S, Hq, start, n_new, None)


def decode(c, q=P, stride=256, o=2 * P, lse=None, Hq=4, scale=0.125, add=0, ws=P, wsb=None):
    L = attn.lib()
    wsb = L.tkm_attn_decode_workspace_bytes(ref(c), Hq, add) if wsb is None else wsb
    return L.tkm_attn_decode(ref(c), q, stride, o, lse, Hq, scale, add, ws, wsb, None)


def evict(c, dst=None, kept=P, budget=100, sink=0, recent=0):
    return attn.lib().tkm_attn_kv_evict(ref(c), ref(dst), kept, budget, sink, recent, None)


BAD_CACHE = [
    (dict(k=None), EINVAL, b"non-null"), (dict(v=None), EINVAL, b"non-null"), (dict(table=None), EINVAL, b"non-null"),
    (dict(len=None), EINVAL, b"non-null"), (dict(B=0), EINVAL, b"positive"), (dict(Hkv=-1), EINVAL, b"positive"),
    (dict(num_pages=0), EINVAL, b"positive"), (dict(max_pages=0), EINVAL, b"positive"), (dict(D=96), EUNSUPPORTED, b"head dim"),
    (dict(page=16), EUNSUPPORTED, b"pages of"), (dict(page=48), EUNSUPPORTED, b"pages of"), (dict(page=512), EUNSUPPORTED, b"pages of"),
    (dict(dtype=2), EUNSUPPORTED, b"dtype"), (dict(max_pages=1 << 25), EUNSUPPORTED, b"too large"),
    (dict(B=1 << 20, Hkv=32), EUNSUPPORTED, b"too large"), (dict(k=P + 8), EALIGN, b"aligned"), (dict(v=P + 2), EALIGN, b"aligned"),
    (dict(table=P + 2), EALIGN, b"aligned"), (dict(len=P + 1), EALIGN, b"aligned"), (dict(weight=P + 2), EALIGN, b"aligned"),
]


@pytest.mark.parametrize("kw,status,msg", BAD_CACHE)
@pytest.mark.parametrize("call", [append, decode, evict])
def test_every_call_refuses_a_bad_cache(call, kw, status, msg):
    assert call(kv(**kw)) == status
    assert msg in attn.lib().tkm_attn_last_error()
    assert attn.lib().tkm_attn_last_kernels() == 0


@pytest.mark.parametrize("call", [append, decode, evict])
def test_every_call_refuses_no_cache(call):
    assert call(None) == EINVAL


@pytest.mark.parametrize("kw,status,msg", [
    (dict(qkv=None), EINVAL, b"qkv"), (dict(S=0), EINVAL, b"positive"), (dict(Hq=3), EINVAL, b"multiple"), (dict(Hq=0), EINVAL, b"positive"),
    (dict(qkv=P + 8), EALIGN, b"aligned"), (dict(start=P + 2), EALIGN, b"aligned"), (dict(n_new=P + 1), EALIGN, b"aligned"),
    (dict(n_new=4 * P), EINVAL, b"own len"), (dict(S=1 << 29), EUNSUPPORTED, b"grid"),
])
def test_append_refuses(kw, status, msg):
    assert append(kv(), **kw) == status
    assert msg in attn.lib().tkm_attn_last_error()


@pytest.mark.parametrize("kw,status,msg", [
    (dict(q=None), EINVAL, b"non-null"), (dict(o=None), EINVAL, b"non-null"), (dict(Hq=3), EINVAL, b"multiple"),
    (dict(stride=248), EINVAL, b"q_stride"), (dict(stride=260), EINVAL, b"q_stride"), (dict(q=P + 8), EALIGN, b"aligned"),
    (dict(o=P + 8), EALIGN, b"aligned"), (dict(lse=P + 2), EALIGN, b"aligned"), (dict(scale=0.0), EINVAL, b"scale"),
    (dict(scale=float("nan")), EINVAL, b"scale"), (dict(scale=float("inf")), EINVAL, b"scale"), (dict(add=2), EINVAL, b"add_weights"),
    (dict(Hq=1 << 24), EUNSUPPORTED, b"too large"),
])
def test_decode_refuses(kw, status, msg):
    assert decode(kv(), **kw) == status
    assert msg in attn.lib().tkm_attn_last_error()


def test_decode_refuses_weights_without_room_for_them():
    assert decode(kv(weight=None), add=1, wsb=1 << 30) == EINVAL and b"add_weights" in attn.lib().tkm_attn_last_error()
    assert decode(kv(max_pages=1 << 22, page=256, B=64), wsb=1 << 40) == EUNSUPPORTED


@pytest.mark.parametrize("kw,status,msg", [
    (dict(ws=None), EWORKSPACE, b"workspace"), (dict(wsb=16), EWORKSPACE, b"workspace"), (dict(ws=P + 4), EALIGN, b"aligned")])
@pytest.mark.parametrize("add", [0, 1])
def test_decode_refuses_a_workspace(kw, status, msg, add):
    assert decode(kv(max_pages=100 if not add else 1), add=add, **kw) == status
    assert msg in attn.lib().tkm_attn_last_error()


def test_decode_workspace():
    L = attn.lib()
    small, large = kv(max_pages=1), kv(max_pages=1000)
    assert 0 == L.tkm_attn_decode_workspace_bytes(ref(small), 4, 0) < L.tkm_attn_decode_workspace_bytes(ref(large), 4, 0)
    assert L.tkm_attn_decode_workspace_bytes(ref(large), 4, 0) <= 256 * 8 * 2 * 66 * 4 + 4096
    assert L.tkm_attn_decode_workspace_bytes(ref(small), 4, 1) >= 2 * 4 * 65 * 4
    assert L.tkm_attn_decode_workspace_bytes(ref(kv(D=80)), 4, 0) == 0
    assert L.tkm_attn_decode_workspace_bytes(ref(small), 5, 0) == 0


@pytest.mark.parametrize("kw,status,msg", [
    (dict(kept=None), EINVAL, b"kept"), (dict(kept=P + 2), EALIGN, b"kept"), (dict(budget=0), EINVAL, b"budget"),
    (dict(sink=-1), EINVAL, b"sink"), (dict(recent=-1), EINVAL, b"recent"), (dict(sink=60, recent=41), EINVAL, b"recent"),
    (dict(sink=2147483647, recent=2147483647), EINVAL, b"sink"), (dict(budget=257), EINVAL, b"exceeds"),
    (dict(dst=kv(table=9 * P, len=10 * P, weight=11 * P, D=128)), EINVAL, b"same"), (dict(dst=kv(len=9 * P)), EINVAL, b"in place"),
    (dict(dst=kv(table=9 * P)), EINVAL, b"its own"), (dict(dst=kv(table=9 * P, len=10 * P)), EINVAL, b"its own"),
    (dict(dst=kv(table=9 * P, len=10 * P, weight=11 * P, max_pages=1)), EINVAL, b"exceeds"),
    (dict(dst=kv(page=7)), EUNSUPPORTED, b"pages of"),
])
def test_evict_refuses(kw, status, msg):
    assert evict(kv(), **kw) == status
    assert msg in attn.lib().tkm_attn_last_error()


def test_evict_refuses_a_cache_without_weights():
    assert evict(kv(weight=None)) == EINVAL and b"weights" in attn.lib().tkm_attn_last_error()


def test_python_refuses():
    k = torch.zeros(4, 2, 2, 2, 32, 32, dtype=torch.float16)
    table, n = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="on cpu"):      # no device tensors here: the first check of placement
        attn.KvCache(k, k.clone(), table, n)
    with pytest.raises(ValueError, match="32, 32"):
        attn.KvCache(k[..., :16], k[..., :16], table, n)
    with pytest.raises(ValueError, match="max_pages"):
        attn.KvCache(k, k.clone(), table[0], n)
    with pytest.raises(TypeError, match="float16"):
        attn.KvCache(k.float(), k.float(), table, n)


def test_layout_helpers_are_inverse():
    x = torch.randn(3, 128, 64)
    for v in (False, True):
        p = blocks(x, 64, v)
        assert p.shape == (2, 3, 2, 2, 32, 32) and torch.equal(dense(p, v), x)
    assert blocks(x, 64, False)[1, 2, 1, 0, 5, 7] == x[2, 64 + 32 + 5, 7]
    assert blocks(x, 64, True)[1, 2, 1, 1, 7, 5] == x[2, 64 + 32 + 5, 32 + 7]


def test_references_by_hand():
    q = torch.tensor([[[1.0, 0.0], [0.0, 2.0]]], dtype=torch.float64)
    k, v = torch.tensor([[[0.0, 0.0], [1.0, 1.0]]], dtype=torch.float64), torch.tensor([[[1.0, 2.0], [3.0, 4.0]]], dtype=torch.float64)
    o, lse, w, _, _ = decode_ref(q, [k], [v], 1, 1.0)
    e = torch.tensor([1.0, 2.0], dtype=torch.float64).exp()
    p = e / (1 + e)                                           # of the second key
    assert torch.allclose(o[0], torch.stack((1 + 2 * p, 2 + 2 * p), 1)) and torch.allclose(lse[0], (1 + e).log())
    assert torch.allclose(w[0][0], torch.stack(((1 - p).sum(), p.sum())))
    assert evict_ref([0.0, 3.0, 1.0, 3.0, float("nan"), 2.0], 6, 3, 1, 1) == [0, 1, 5]
    assert evict_ref([0.0, 1.0, 1.0, 1.0, 0.0], 5, 3, 0, 1) == [1, 2, 4]
    assert evict_ref([5.0, 1.0], 2, 3, 0, 0) == [0, 1]
