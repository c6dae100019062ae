"""The calls of a serving step without a GPU: what they refuse before anything is launched, the frequencies of rotary
positions, and the helpers that the GPU tests compare with."""
import ctypes
import math

import numpy as np
import pytest
import torch

from step_cases import chunk_ref, freqs_ref, plan_ref, rope_ref, visible
from test_kv_cpu import BAD_CACHE, P, kv, ref
from tokamak_amd import attn, prep

OK, EINVAL, EUNSUPPORTED, EALIGN, EWORKSPACE = 0, -1, -2, -3, -4


def rope(rot=64, layout=0):
    r = attn._Rope()
    r.rot, r.layout, r.factor = rot, layout, 1.0
    return r


def plan(**kw):
    c = dict(n_new=P, row_start=2 * P, seq=3 * P, pos=4 * P, slot=5 * P)
    c.update(kw)
    return attn._Plan(*(c[n] for n, _ in attn._Plan._fields_))


def pages(**kw):
    c = dict(free=6 * P, n_free=7 * P, held=8 * P)
    c.update(kw)
    return attn._Pages(*(c[n] for n, _ in attn._Pages._fields_))


def call_plan(c, pg=None, want=9 * P, start=None, pl=None, rows=5):
    return attn.lib().tkm_attn_kv_plan(ref(c), ref(pages() if pg is None else pg), want, start, ref(plan() if pl is None else pl), rows, None)


def call_append(c, r=None, qkv=P, stride=512, q=2 * P, q_stride=256, pl=None, rows=5, Hq=4):
    return attn.lib().tkm_attn_kv_append_rows(ref(c), ref(r), qkv, stride, q, q_stride, ref(plan() if pl is None else pl), rows, Hq, None)


def call_chunk(c, q=P, stride=256, row_start=None, n_new=None, rows=6, o=2 * P, lse=None, Hq=4, scale=0.125, causal=1, window=0, ws=P, wsb=None):
    L = attn.lib()
    wsb = L.tkm_attn_chunk_workspace_bytes(ref(c), rows, Hq) if wsb is None else wsb
    return L.tkm_attn_chunk(ref(c), q, stride, row_start, n_new, rows, o, lse, Hq, scale, causal, window, ws, wsb, None)


def call_rope(r=None, x=P, xs=512, y=2 * P, ys=512, pos=3 * P, S=1, rows=5, Hq=4, Hkv=2, D=64, dtype=0, inverse=0):
    return attn.lib().tkm_attn_rope_rows(ref(rope() if r is None else r), x, xs, y, ys, pos, S, rows, Hq, Hkv, D, dtype, inverse, None)


@pytest.mark.parametrize("kw,status,msg", BAD_CACHE)
@pytest.mark.parametrize("call", [call_plan, call_append, call_chunk])
def test_every_call_refuses_a_bad_cache(call, kw, status, msg):
    assert call(kv(**kw)) == status
    assert msg in attn.lib().tkm_attn_last_error()
    assert attn.lib().tkm_attn_last_kernels() == 0


@pytest.mark.parametrize("call", [call_plan, call_append, call_chunk])
def test_every_call_refuses_no_cache(call):
    assert call(None) == EINVAL


@pytest.mark.parametrize("kw,status,msg", [
    (dict(pg=pages(free=None)), EINVAL, b"free"), (dict(pg=pages(n_free=None)), EINVAL, b"n_free"), (dict(pg=pages(held=None)), EINVAL, b"held"),
    (dict(want=None), EINVAL, b"want"), (dict(rows=-1), EINVAL, b"rows"), (dict(pl=plan(n_new=None)), EINVAL, b"n_new"),
    (dict(pl=plan(row_start=None)), EINVAL, b"row_start"), (dict(pl=plan(seq=None)), EINVAL, b"seq"), (dict(pl=plan(slot=None)), EINVAL, b"slot"),
    (dict(pl=plan(slot=P + 4)), EALIGN, b"slot"), (dict(pl=plan(pos=P + 2)), EALIGN, b"4-byte"), (dict(want=P + 2), EALIGN, b"4-byte"),
    (dict(start=P + 1), EALIGN, b"4-byte"), (dict(pg=pages(held=P + 2)), EALIGN, b"4-byte"), (dict(want=P), EINVAL, b"another"),
    (dict(want=4 * P), EINVAL, b"another"), (dict(start=9 * P), EINVAL, b"another"),
])
def test_plan_refuses(kw, status, msg):
    assert call_plan(kv(), **kw) == status
    assert msg in attn.lib().tkm_attn_last_error()


@pytest.mark.parametrize("kw,status,msg", [
    (dict(qkv=None), EINVAL, b"qkv"), (dict(rows=-1), EINVAL, b"positive"), (dict(Hq=3), EINVAL, b"multiple"), (dict(Hq=0), EINVAL, b"positive"),
    (dict(stride=504), EINVAL, b"stride"), (dict(stride=516), EINVAL, b"stride"), (dict(q_stride=248), EINVAL, b"q_stride"),
    (dict(q_stride=260), EINVAL, b"q_stride"), (dict(q=P), EINVAL, b"in place"), (dict(qkv=P + 8), EALIGN, b"aligned"), (dict(q=P + 8), EALIGN, b"aligned"),
    (dict(pl=plan(seq=None)), EINVAL, b"seq"), (dict(pl=plan(pos=None)), EINVAL, b"pos"), (dict(pl=plan(slot=None)), EINVAL, b"slot"),
    (dict(pl=plan(slot=P + 4)), EALIGN, b"slot"), (dict(r=rope(66)), EINVAL, b"rot"), (dict(r=rope(63)), EINVAL, b"rot"), (dict(r=rope(0)), EINVAL, b"rot"),
    (dict(r=rope(64, 2)), EINVAL, b"layout"), (dict(Hq=1 << 26, stride=1 << 32), EUNSUPPORTED, b"wide"), (dict(rows=(1 << 31) - 1), EUNSUPPORTED, b"grid"),
])
def test_append_rows_refuses(kw, status, msg):
    assert call_append(kv(), **kw) == status
    assert msg in attn.lib().tkm_attn_last_error()


@pytest.mark.parametrize("kw,status,msg", [
    (dict(x=None), EINVAL, b"non-null"), (dict(y=None), EINVAL, b"non-null"), (dict(rows=-1), EINVAL, b"positive"), (dict(Hq=0), EINVAL, b"positive"),
    (dict(Hkv=-1), EINVAL, b"positive"), (dict(D=96), EUNSUPPORTED, b"head dim"), (dict(dtype=2), EUNSUPPORTED, b"dtype"), (dict(inverse=2), EINVAL, b"inverse"),
    (dict(pos=None, S=0), EINVAL, b"positions"), (dict(xs=504), EINVAL, b"stride"), (dict(ys=516), EINVAL, b"stride"), (dict(y=P, ys=1024), EINVAL, b"in place"),
    (dict(x=P + 8), EALIGN, b"aligned"), (dict(pos=P + 2), EALIGN, b"aligned"), (dict(r=rope(66)), EINVAL, b"rot"), (dict(r=rope(64, -1)), EINVAL, b"layout"),
    (dict(Hq=1 << 25, xs=1 << 32, ys=1 << 32), EUNSUPPORTED, b"wide"), (dict(rows=(1 << 31) - 1), EUNSUPPORTED, b"grid"),
])
def test_rope_refuses(kw, status, msg):
    assert call_rope(**kw) == status
    assert msg in attn.lib().tkm_attn_last_error()


@pytest.mark.parametrize("kw,status,msg", [
    (dict(q=None), EINVAL, b"non-null"), (dict(o=None), EINVAL, b"non-null"), (dict(rows=0), EINVAL, b"positive"), (dict(Hq=3), EINVAL, b"multiple"),
    (dict(Hq=0), EINVAL, b"positive"), (dict(row_start=P), EINVAL, b"n_new"), (dict(rows=5), EINVAL, b"same number"), (dict(causal=2), EINVAL, b"causal"),
    (dict(window=-1), EINVAL, b"window"), (dict(causal=0, window=3), EINVAL, b"window"), (dict(stride=248), EINVAL, b"q_stride"), (dict(stride=260), EINVAL, b"q_stride"),
    (dict(q=P + 8), EALIGN, b"aligned"), (dict(o=P + 8), EALIGN, b"aligned"), (dict(lse=P + 2), EALIGN, b"aligned"), (dict(n_new=P + 2), EALIGN, b"aligned"),
    (dict(row_start=P + 2, n_new=P), EALIGN, b"aligned"), (dict(scale=0.0), EINVAL, b"scale"), (dict(scale=float("nan")), EINVAL, b"scale"),
    (dict(scale=3e38), EINVAL, b"scale"), (dict(ws=None), EWORKSPACE, b"workspace"), (dict(wsb=64), EWORKSPACE, b"workspace"), (dict(ws=P + 4), EALIGN, b"workspace"),
    (dict(rows=1 << 30, wsb=1 << 60), EUNSUPPORTED, b"too large"),
])
def test_chunk_refuses(kw, status, msg):
    assert call_chunk(kv(max_pages=100), **kw) == status
    assert msg in attn.lib().tkm_attn_last_error()
    assert attn.lib().tkm_attn_last_kernels() == 0


def test_chunk_workspace():
    L = attn.lib()
    small, large = kv(max_pages=4), kv(max_pages=1000)
    assert L.tkm_attn_chunk_workspace_bytes(ref(small), 6, 4) == 0 < L.tkm_attn_chunk_workspace_bytes(ref(large), 6, 4)
    assert L.tkm_attn_chunk_workspace_bytes(ref(large), 1 << 20, 4) <= 1024 * 2 * 128 * 66 * 4 + (1 << 20)      # its pieces, and lists
    for kw, rows, Hq in ((dict(D=80), 6, 4), ({}, 6, 5), ({}, -1, 4)):
        assert L.tkm_attn_chunk_workspace_bytes(ref(kv(max_pages=1000, **kw)), rows, Hq) == 0


def test_nothing_to_do_launches_nothing():
    assert call_rope(rows=0, x=None, y=None) == OK and call_append(kv(), rows=0, qkv=None) == OK
    assert attn.lib().tkm_attn_last_kernels() == 0
    assert attn.lib().tkm_attn_chunk_workspace_bytes(ref(kv()), 0, 4) == 0


@pytest.mark.parametrize("kw", [
    dict(rot=63), dict(rot=0), dict(rot=130), dict(rot=64, layout="thirds"), dict(rot=64, scaling="cubic"), dict(rot=64, theta=0.5), dict(rot=64, theta=float("inf")),
    dict(rot=64, scaling="linear", scale=0.5), dict(rot=64, scaling="ntk", scale=float("nan")), dict(rot=64, scaling="bands", scale=2, low=4, high=1),
    dict(rot=64, scaling="yarn", scale=2, original=0), dict(rot=64, scaling="yarn", scale=2, theta=1.0), dict(rot=64, factor=-1.0), dict(rot=64, factor=1e39),
    dict(rot=64, freqs=[1.0] * 31), dict(rot=64, freqs=[1.0] * 31 + [float("nan")]), dict(rot=64, freqs=[1e11] * 32), dict(rot=64, freqs=[1.0] * 32, scaling="ntk")])
def test_rope_is_not_made_of(kw):
    with pytest.raises((ValueError, attn.AttnError)):
        attn.Rope(**kw)


@pytest.mark.parametrize("rot", [2, 4, 20, 64, 100, 128])
@pytest.mark.parametrize("theta", [1.0, 100.0, 10000.0, 5e5, 1e8])
@pytest.mark.parametrize("scaling,kw", [(None, {}), ("linear", dict(scale=4.0)), ("ntk", dict(scale=8.0)), ("bands", dict(scale=8.0)),
                                        ("bands", dict(scale=3.0, original=4096.0, low=2.0, high=7.5)), ("yarn", dict(scale=16.0)),
                                        ("yarn", dict(scale=1.0)), ("yarn", dict(scale=4.0, original=32.0, low=0.5, high=2.0))])
def test_frequencies(rot, theta, scaling, kw):
    """A frequency's turns in units of 2^-64 are those of the formula in 80 bits: both sides round a power, a few
    products and a quotient in 64 bits of mantissa, 16 roundings of 2^-64 at most, of numbers of 2 radians at most."""
    if scaling == "yarn" and theta == 1.0:
        return
    r = attn.Rope(rot, theta=theta, scaling=scaling, **kw)
    f, factor = freqs_ref(rot, theta, scaling, **kw)
    want = f / (2 * np.longdouble("3.14159265358979323846264338327950288")) * np.longdouble(2.0) ** 64
    for i in range(rot // 2):
        got = np.longdouble(r._c.turns[i])
        assert abs(got - want[i]) <= 32, (i, got, want[i])
    assert r.factor == np.float32(factor) and r.rot == rot
    # 32 units of 2 pi 2^-64 are 1.1e-17, and a frequency of 1e-8 has 1e-9 of that: an absolute bound, not a relative one
    assert np.allclose(r.freqs(), [float(x) for x in f], rtol=1e-14, atol=1.1e-17)


def test_given_frequencies_wrap():
    r = attn.Rope(4, freqs=[2 * math.pi * 3 + 1.0, -0.5], factor=2.0)
    assert r.freqs()[0] == pytest.approx(1.0, abs=1e-14) and r.freqs()[1] == pytest.approx(2 * math.pi - 0.5, abs=1e-14)
    assert r.factor == 2.0


def test_rope_of_a_prep_descriptor():
    d = prep.make_desc(2, 1, 64, 100, rope=True, theta=500.0, scale=4.0)
    r = attn.Rope.of_prep(d)
    assert r.rot == 64 and r._c.layout == attn.Rope.LAYOUTS["pairs"] and r.factor == 1.0
    assert r.freqs()[0] == pytest.approx(1.0) and r.freqs()[1] == pytest.approx(500.0 ** (-1 / 64), rel=1e-6)
    with pytest.raises(attn.AttnError):
        attn.Rope.of_prep(prep.make_desc(2, 1, 64, 100))


def test_helpers():
    x = torch.randn(3, 2, 64, dtype=torch.float64)
    for layout in ("halves", "pairs"):
        y, _ = rope_ref(x, [0, 5, 70000], freqs_ref(20, 10000.0)[0], 2.0, layout)
        back, _ = rope_ref(y, [0, 5, 70000], freqs_ref(20, 10000.0)[0], 0.5, layout, inverse=True)
        assert torch.allclose(back, x, atol=1e-12) and torch.equal(y[..., 20:], x[..., 20:]) and torch.allclose(y[0, :, :20], 2 * x[0, :, :20])
    seen = visible(5, 3, True, 2)
    assert seen.tolist() == [[False, True, True, False, False], [False, False, True, True, False], [False, False, False, True, True]]
    assert visible(2, 3, True, 0)[0].sum() == 0
    k, v = torch.randn(1, 5, 64, dtype=torch.float64), torch.randn(1, 5, 64, dtype=torch.float64)
    o, lse, _, _ = chunk_ref(x, k, v, seen, 1, 0.1, "f16")
    p = torch.softmax(x[1, 1] @ k[0, 2:4].T * 0.1, 0)
    assert torch.allclose(o[1, 1], p @ v[0, 2:4]) and lse[1, 1] == pytest.approx(torch.logsumexp(x[1, 1] @ k[0, 2:4].T * 0.1, 0).item())


def test_plan_by_a_loop():
    """Two sequences grow, one ends, one finds too few pages, the one behind it needs none."""
    p = plan_ref([[5, -1, -1], [6, 7, -1], [8, -1, -1], [9, -1, -1]], [1, 2, 0, 0, 0], 2, [1, 2, 1, 1], [40, 0, 90, 3], [30, 0, 20, 4],
                 32, 10, 60)
    assert p["n_new"] == [40, 0, 0, 3] and p["row_start"] == [0, 40, 40, 40, 43] and p["kv_len"] == [70, 0, 20, 7]
    assert p["table"] == [[5, 7, 6], [-1, -1, -1], [8, -1, -1], [9, -1, -1]] and p["n_free"] == [2] and p["held"] == [3, 0, 1, 1]
    assert p["slot"][:4] == [5 * 32 + 30, 5 * 32 + 31, 7 * 32, 7 * 32 + 1] and p["slot"][40:44] == [9 * 32 + 4, 9 * 32 + 5, 9 * 32 + 6, -1]


def test_tensors_off_the_gpu_are_refused():
    import torch
    x, dt = torch.zeros(4, 3 * 64, dtype=torch.float16), torch.int32
    with pytest.raises(ValueError, match="GPU"):
        attn.rope_fwd(x, attn.Rope(64), 1, 1, 64, S=4)
    with pytest.raises(ValueError, match="must be on"):
        attn.KvPages(torch.zeros(8, dtype=dt), torch.zeros(1, dtype=dt), torch.zeros(2, dtype=dt))
    with pytest.raises(ValueError, match="must be on"):
        attn.KvPlan.empty(2, 4, "cpu")
