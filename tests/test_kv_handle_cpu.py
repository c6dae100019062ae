"""A cache's tensors are written, not replaced: also by augmented assignment, which ends in an assignment of the same
tensor.  (The handle is made without its constructor, which takes device tensors alone.)"""
import pytest
import torch

from tokamak_amd import attn


def handle():
    c = attn.KvCache.__new__(attn.KvCache)
    c.kv_len, c.weight, c.page = torch.tensor([3, 4]), torch.ones(2, 2), 64
    return c


def test_augmented_assignment_writes_the_tensor():
    c = handle()
    n, w = c.kv_len, c.weight
    c.kv_len += 1
    c.weight *= 0.5
    c.kv_len = n
    assert c.kv_len is n and n.tolist() == [4, 5] and c.weight is w and w.tolist() == [[0.5, 0.5], [0.5, 0.5]]


@pytest.mark.parametrize("name,value", [("kv_len", torch.tensor([3, 4])), ("weight", None), ("page", 32)])
def test_another_value_is_refused(name, value):
    c = handle()
    with pytest.raises(AttributeError, match="cannot be replaced"):
        setattr(c, name, value)
    assert c.kv_len.tolist() == [3, 4] and c.weight is not None and c.page == 64
