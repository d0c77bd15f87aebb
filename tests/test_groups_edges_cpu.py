"""Attention over shared prefixes, decode attention over pages with scores and eviction, CPU forms: calls at the borders of what their documentation allows."""
import pytest
import torch

from groups_refusals import ints, packed
from nanorlhf_b200 import ops


@pytest.mark.parametrize("groups", [0, 2])
def test_rows_without_any_sequence(groups):
    """they are behind the last one: 0, and so are their gradients"""
    q, k, v, dout, cu, _ = packed([[5]], 4, 2)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = ops.attention_shared_prefix(*leaves, cu[:1], ints(*[0] * (groups + 1)))
    for x in (out, *torch.autograd.grad(out, leaves, dout)):
        assert torch.equal(x, torch.zeros_like(x))
