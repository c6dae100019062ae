"""Limits of a serving step's calls without a GPU, with results written out by hand."""
import pytest
import torch

from step_cases import plan_ref
from test_step_cpu import EINVAL, OK, call_rope
from tokamak_amd import attn


@pytest.mark.parametrize("rows,want,n_new", [(10, [8, 5, 2], [8, 0, 0]), (10, [8, 2, 5], [8, 2, 0]), (10, [30, 1, 1], [0, 0, 0]),
                                             (10, [-1, 11, 1], [0, 0, 0]), (40, [33, 300, 7], [33, 0, 7])])
def test_rows_that_do_not_fit_hold_up_those_behind(rows, want, n_new):
    """What the helper of the GPU tests gives is what include/tkm_attn.h says."""
    p = plan_ref([[-1] * 4 for _ in range(3)], [2, 1, 0], 3, [0, 0, 0], want, [0, 0, 0], 32, 3, rows)
    assert p["n_new"] == n_new and p["row_start"] == [0, n_new[0], n_new[0] + n_new[1], sum(n_new)]


@pytest.mark.parametrize("inverse", [-1, 2, 3, 255, 258, 512, 1 | 512])
def test_rope_knows_no_other_flags(inverse):
    assert call_rope(inverse=inverse) == EINVAL
    assert b"inverse" in attn.lib().tkm_attn_last_error()


@pytest.mark.parametrize("inverse", [256, 257])
def test_rope_takes_the_flag(inverse):
    assert call_rope(inverse=inverse, rows=0, x=None, y=None) == OK


@pytest.mark.parametrize("kw", [{}, {"scaling": "yarn", "scale": 4.0}, {"freqs": [1.0] * 32}])
def test_rope_factors_that_vanish_in_fp32(kw):
    """They would make every rotated dim 0; 0 itself stands for the scaling's own."""
    for factor in (1e-60, 7e-46):          # half of the least fp32, and below: rounded to 0
        with pytest.raises(attn.AttnError, match="factor"):
            attn.Rope(64, factor=factor, **kw)
    assert attn.Rope(64, factor=1e-45, **kw).factor > 0.0
    assert attn.Rope(64, factor=0.0, **kw).factor == attn.Rope(64, **kw).factor


@pytest.mark.parametrize("cls,name", [(attn.KvPages, "n_free"), (attn.KvPages, "held"), (attn.KvPlan, "slot"), (attn.KvPlan, "row_start")])
def test_tensors_of_handles_are_written_not_replaced(cls, name):
    """The C structs hold the first tensor's address, whatever the attribute says.  (Handles made without their
    constructors, which take device tensors alone.)"""
    h, t = cls.__new__(cls), torch.tensor([3, 4])
    setattr(h, name, t)
    setattr(h, name, getattr(h, name).add_(1))       # what h.name += 1 ends in
    assert getattr(h, name) is t and t.tolist() == [4, 5]
    with pytest.raises(AttributeError, match="cannot be replaced"):
        setattr(h, name, torch.tensor([4, 5]))
    assert getattr(h, name) is t
