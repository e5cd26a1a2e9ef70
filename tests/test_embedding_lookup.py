"""Rows by id and their gradient by sorted ids against sums in 64 bits.

A sum of n numbers is off by at most (n - 1) roundings of half a step each, relative to the sum of their
magnitudes; the scale adds one more."""
import pytest
import torch

from xnn_b200.ops import ScaledEmbedding, embedding_lookup

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _ids(n, rows, kind, g):
    if kind == "same":
        return torch.full((n,), rows - 1)
    if kind == "few":
        return torch.randint(0, 3, (n,), generator=g).clamp(max=rows - 1)
    if kind == "outside":
        return torch.randint(-3, rows + 3, (n,), generator=g)
    if kind == "sorted":
        return torch.randint(0, rows, (n,), generator=g).sort().values
    return torch.randint(0, rows, (n,), generator=g)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("n,rows,width,kind", [
    (1, 1, 1, "same"), (5, 3, 7, "outside"), (611, 87, 64, "any"), (4096, 100, 33, "few"), (4097, 100, 32, "few"),
    (4500, 87, 64, "same"), (5000, 255, 128, "any"), (5000, 256, 20, "outside"), (9000, 257, 130, "sorted"),
    (20000, 7569, 16, "any"), (30011, 70000, 4, "outside"), (40000, 5, 300, "few"), (700, 9000, 12, "any"), (60000, 148, 130, "any"),
    (60000, 149, 3, "few"), (50001, 4, 257, "same"),
    (8192, 2000, 16, "any"), (8192, 40, 16, "same"), (8192, 40, 17, "same"), (8193, 5, 3, "few"), (1023, 30, 128, "few")])
def test_values_and_gradients(device, dtype, n, rows, width, kind):
    g = torch.Generator().manual_seed(n + rows)
    table = torch.randn(rows, width, generator=g, dtype=torch.float64).to(dtype).to(device).requires_grad_()
    ids = _ids(n, rows, kind, g).to(device)
    gy = torch.randn(n, width, generator=g, dtype=torch.float64).to(dtype).to(device).requires_grad_()
    on = (ids >= 0) & (ids < rows)
    out = embedding_lookup(table, ids, 0.5)
    assert torch.equal(out, torch.where(on[:, None], 0.5 * table[torch.where(on, ids, 0)], 0.0))
    (grad,) = torch.autograd.grad(out, table, gy, create_graph=True)
    wide = torch.zeros(rows, width, dtype=torch.float64)
    want = 0.5 * wide.index_add(0, ids[on].cpu(), gy[on].detach().double().cpu())
    size = 0.5 * wide.index_add(0, ids[on].cpu(), gy[on].detach().double().abs().cpu())
    count = torch.bincount(ids[on].cpu(), minlength=rows)[:, None].double()
    assert bool(((grad.detach().double().cpu() - want).abs() <= (count + 1) * torch.finfo(dtype).eps / 2 * size).all())
    (back,) = torch.autograd.grad(grad, gy, table)
    assert torch.equal(back, out)
    assert torch.equal(embedding_lookup(table, ids.int(), 0.5), out)
    if device == "cuda":
        again = torch.autograd.grad(embedding_lookup(table, ids.int(), 0.5), table, gy)[0]
        assert torch.equal(again, grad)


@pytest.mark.parametrize("device", DEVICES)
def test_shapes_and_strides(device):
    table = torch.randn(9, 12, device=device)
    ids = torch.randint(0, 9, (6, 4), device=device)
    assert torch.equal(embedding_lookup(table, ids), table[ids])
    assert torch.equal(embedding_lookup(table, ids.t()), table[ids.t()])
    assert torch.equal(embedding_lookup(table[:, 1:8], ids), table[:, 1:8][ids])
    odd = torch.randn(9 * 8 + 1, device=device)[1:].view(9, 8).requires_grad_()
    out = embedding_lookup(odd, ids[0])
    assert torch.equal(out, odd[ids[0]])
    (g,) = torch.autograd.grad(out.sum(), odd)          # an expanded gradient
    assert torch.equal(g.sum(1), 8.0 * torch.bincount(ids[0], minlength=9))
    for empty in (ids[:0], torch.zeros(0, dtype=torch.int32, device=device)):
        t = table.clone().requires_grad_()
        out = embedding_lookup(t, empty)
        assert out.shape == tuple(empty.shape) + (12,)
        assert not torch.autograd.grad(out.sum(), t)[0].any()
    assert not embedding_lookup(table[:0], ids).any()


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    table, ids = torch.zeros(3, 4, device=device), torch.zeros(2, dtype=torch.int64, device=device)
    for bad in ((table.half(), ids), (table[0], ids), (table, ids.float()), (table, ids.short())):
        with pytest.raises(TypeError):
            embedding_lookup(*bad)
    with pytest.raises(ValueError):
        ScaledEmbedding(3, 4, padding_idx=1)
    if device == "cuda":
        with pytest.raises(ValueError):
            embedding_lookup(table, ids.cpu())


def test_module_refuses_what_it_would_ignore():
    for wrong in (dict(padding_idx=0), dict(padding_idx=2), dict(max_norm=1.0), dict(sparse=True), dict(scale_grad_by_freq=True)):
        with pytest.raises(ValueError):
            ScaledEmbedding(3, 4, **wrong)
    assert ScaledEmbedding(3, 4, padding_idx=None, sparse=False).weight.shape == (3, 4)


def test_module_keeps_the_parameter_name():
    m = ScaledEmbedding(5, 3, scale=2.0)
    assert list(m.state_dict()) == ["weight"]
    ids = torch.tensor([4, 0, 4])
    assert torch.equal(m(ids), 2.0 * m.weight[ids])


@pytest.mark.gpu
def test_captured():
    table = torch.randn(300, 64, device="cuda", requires_grad=True)
    ids = torch.randint(0, 300, (20000,), device="cuda")
    gy = torch.randn(20000, 64, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (grad,) = torch.autograd.grad(embedding_lookup(table, ids), table, gy)
    ids.copy_(torch.randint(0, 300, (20000,), device="cuda"))
    graph.replay()
    assert torch.equal(grad, torch.autograd.grad(embedding_lookup(table, ids), table, gy)[0])
