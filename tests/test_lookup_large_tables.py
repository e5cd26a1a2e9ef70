"""Few ids of a large table: the gradient is right on both sides of the rule that skips the sort, and costs no more than
that of many ids."""
import pytest
import torch

from xnn_b200.ops import embedding_lookup


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("rows", [16383, 16384, 16385, 65537])
@pytest.mark.parametrize("width", [1, 3, 8])
def test_gradients(device, rows, width):
    ids = torch.tensor([0, rows - 1, 5, rows, -1, 5, rows - 1, rows // 2], device=device)
    table = torch.randn(rows, width, device=device, requires_grad=True)
    g = torch.randn(ids.numel(), width, device=device)
    (grad,) = torch.autograd.grad(embedding_lookup(table, ids), table, g)
    want = torch.zeros(rows, width, device=device)
    want[0], want[5], want[rows - 1], want[rows // 2] = g[0], g[2] + g[5], g[1] + g[6], g[7]
    assert torch.equal(grad, want)              # two terms at most: one rounding in any order


@pytest.mark.gpu
def test_few_ids_cost_no_more_than_many():
    rows = 1 << 20
    table = torch.randn(rows, 64, device="cuda", requires_grad=True)
    times = []
    for n in (16, 10000):                       # the second is sorted by any rule
        ids = torch.randint(0, rows, (n,), device="cuda")
        g = torch.randn(n, 64, device="cuda")
        best = float("inf")
        for _ in range(8):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            y = embedding_lookup(table, ids)
            a.record()
            torch.autograd.grad(y, table, g)
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        times.append(best)
    assert times[0] < 2 * times[1], times
