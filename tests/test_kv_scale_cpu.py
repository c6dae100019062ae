"""Decode multiplies scores by scale * log2(e): a scale whose product is not finite would make NaN of scores of 0."""
import pytest

from test_kv_cpu import EINVAL, decode, kv
from tokamak_amd import attn


@pytest.mark.parametrize("scale", [2.4e38, 3.4e38])
def test_refused(scale):
    assert decode(kv(), scale=scale) == EINVAL
    assert b"scale" in attn.lib().tkm_attn_last_error()
