"""More draws than a launch of fewer than 2^32 threads (HIP's limit) has are refused, not launched."""
import pytest

from test_sample_cpu import P, call
from tokamak_amd import runtime as R


@pytest.mark.parametrize("draws", [1 << 22, 1 << 24, (1 << 31) - 1])
def test_draws(draws):
    assert call(draws=draws, row_index=P) == -2
    assert b"draws" in R.lib().tkm_attn_last_error()
