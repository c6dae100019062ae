"""tkm_hip_sample without a GPU: its refusals, and the 64-bit draw that the GPU tests compare with."""
import ctypes

import numpy as np
import pytest
import torch

from sample_cases import draw_ref
from tokamak_amd import runtime as R

P = 0x10000


def call(null=False, **kw):
    a = dict(logits=P, row_stride=100, rows=3, vocab=100, dtype=0, draws=3, row_index=None, temperature=None, top_k=None, top_p=None,
             min_p=None, u=P, token=P)
    a.update(kw)
    s = R._SampleArgs(*(a[n] for n, _ in R._SampleArgs._fields_))
    return R.lib().tkm_hip_sample(None if null else ctypes.byref(s), None)


@pytest.mark.parametrize("kw,status,msg", [
    (dict(null=True), -1, b"non-null"), (dict(logits=None), -1, b"non-null"), (dict(u=None), -1, b"non-null"), (dict(token=None), -1, b"non-null"),
    (dict(rows=0), -1, b"positive"), (dict(draws=0), -1, b"positive"), (dict(vocab=-1), -1, b"positive"), (dict(draws=4), -1, b"row_index"),
    (dict(dtype=3), -2, b"dtype"), (dict(vocab=524289, row_stride=1 << 20), -2, b"vocab"), (dict(row_stride=99), -1, b"row_stride"),
    (dict(logits=P + 1), -3, b"aligned"), (dict(logits=P + 2, dtype=2), -3, b"aligned"), (dict(top_k=P + 2), -3, b"aligned"),
    (dict(token=P + 1), -3, b"aligned"), (dict(row_index=P + 2, draws=9), -3, b"aligned"),
])
def test_refusals(kw, status, msg):
    assert call(**kw) == status
    assert msg in R.lib().tkm_attn_last_error()


def test_runtime_sample_refuses_no_runtime():
    s = R._SampleArgs()
    assert R.lib().tkm_runtime_sample(None, None, ctypes.byref(s)) == -1


def test_python_refuses():
    x, u = torch.zeros(2, 8), torch.zeros(2)
    with pytest.raises(TypeError, match="float16"):
        R.sample(x.double(), u)
    with pytest.raises(ValueError, match="device"):
        R.sample(x, u)


def test_reference_by_hand():
    x = np.log([1.0, 4.0, 2.0, 2.0, 1.0])                   # of 10: running 1, 5, 7, 9, 10
    for u, token in ((0.0, 0), (0.0999, 0), (0.1001, 1), (0.4999, 1), (0.5001, 2), (0.8999, 3), (0.95, 4), (1.0, 4)):
        assert draw_ref(x, u)[0] == token
    assert [draw_ref(x, u, top_k=2)[0] for u in (0.0, 0.66, 0.67, 0.99)] == [1, 1, 2, 2]      # 4, 2 (the first of the twos)
    assert [draw_ref(x, u, top_p=0.41)[0] for u in (0.0, 0.66, 0.67)] == [1, 1, 2]            # 4 of 10 is not enough
    assert draw_ref(x, 0.99, top_p=0.39)[0] == 1 and draw_ref(x, 0.99, top_p=0.0)[0] == 1
    assert draw_ref(x, 0.99, min_p=0.4)[0] == 3 and draw_ref(x, 0.99, min_p=0.6)[0] == 1
    assert draw_ref(x, 0.5, temperature=0.0)[0] == 1 and draw_ref([-np.inf, np.nan], 0.5)[0] == -1
