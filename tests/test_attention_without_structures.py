"""Rows of no structure give zeros and take no gradient, whatever they hold, where a batch has no structure with atoms."""
import pytest
import torch

from xnn_b200.ops import structure_attention


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("ptr", [[0], [0, 0], [3, 3], [1, 1, 1]])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_unowned_rows_do_not_reach_the_result(device, ptr, value):
    q, k, v = (torch.full((3, h, 8), value, device=device, requires_grad=True) for h in (2, 1, 1))
    o = structure_attention(q, k, v, torch.tensor(ptr, device=device))
    assert torch.equal(o, torch.zeros_like(q))
    do = torch.full_like(q, value).requires_grad_()
    first = torch.autograd.grad(o, (q, k, v), do, create_graph=True)
    assert all(torch.equal(g, torch.zeros_like(t)) for g, t in zip(first, (q, k, v)))
