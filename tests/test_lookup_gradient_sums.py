"""Sums of many rows in one: the error of a table row's gradient does not grow with the number of its ids.

Whatever their number, a row's sum is off by fewer than 100 roundings of half a step, relative to the sum of its terms'
magnitudes: trees of eight (3), chains of at most 512 / 8 of them and 14 single terms, partial sums by compensated
summation (3 + 2) and those of a block's warps (3 + 4), the scale (1). Equal terms are the worst case of a plain chain, since
each step of it rounds to the same side."""
import pytest
import torch

from xnn_b200.ops import embedding_lookup

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _check(ids, rows, gy, scale=1.0):
    table = torch.zeros(rows, gy.shape[1], dtype=gy.dtype, device=gy.device, requires_grad=True)
    (grad,) = torch.autograd.grad(embedding_lookup(table, ids, scale), table, gy)
    wide = torch.zeros(rows, gy.shape[1], dtype=torch.float64, device=gy.device)
    want = scale * wide.index_add(0, ids, gy.double())
    size = abs(scale) * wide.index_add(0, ids, gy.double().abs())
    assert float(((grad.double() - want).abs() - 100 * torch.finfo(gy.dtype).eps / 2 * size).max()) <= 0


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("value", [0.7, 1.1, 0.1])
@pytest.mark.parametrize("n,rows,width", [(8192, 3, 16), (8000, 60, 7), (100000, 4, 8)])
def test_equal_terms(device, value, n, rows, width):
    _check(torch.full((n,), rows - 1, device=device), rows, torch.full((n, width), value, device=device), 0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("value", [0.7, 1.1, None])
@pytest.mark.parametrize("n,rows,width", [(4_000_000, 2, 4), (4_000_003, 200, 3), (2_000_000, 87, 16)])
def test_many_terms(value, n, rows, width):
    g = torch.Generator("cuda").manual_seed(n)
    ids = torch.randint(0, rows, (n,), generator=g, device="cuda")
    ids[: n // 2] = rows - 1
    gy = torch.rand(n, width, generator=g, device="cuda") if value is None else torch.full((n, width), value, device="cuda")
    _check(ids, rows, gy)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n", [3000, 30000])
def test_infinite_terms_stay_infinite(device, n):
    ids = torch.arange(n, device=device) % 5
    gy = torch.ones(n, 4, device=device)
    gy[5 * 100, 0], gy[5 * 101 + 1, 1], gy[5 * 102 + 2, 2] = float("inf"), float("-inf"), float("nan")
    gy[5 * 103 + 3, 3], gy[5 * 400 + 3, 3] = float("inf"), float("-inf")
    table = torch.zeros(5, 4, device=device, requires_grad=True)
    (grad,) = torch.autograd.grad(embedding_lookup(table, ids), table, gy)
    want = torch.full((5, 4), n / 5.0, device=device)
    want[0, 0], want[1, 1], want[2, 2], want[3, 3] = float("inf"), float("-inf"), float("nan"), float("nan")
    assert torch.equal(grad.nan_to_num(nan=-1.0), want.nan_to_num(nan=-1.0))
