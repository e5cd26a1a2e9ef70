"""Dropout from a counter: the generator's published vectors, the mask's law, sharing, gradients, devices."""
import pytest
import torch

from xnn_b200.ops import CounterDropout, counter_dropout
from xnn_b200.ops.dropout import philox

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def test_generator_vectors():
    """The known answers that its authors publish for ten rounds."""
    zero = philox(torch.zeros(1, dtype=torch.int64), torch.zeros(2, dtype=torch.int64))[0]
    assert [hex(int(w)) for w in zero] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]
    ones = philox(torch.full((1,), -1, dtype=torch.int64), torch.full((2,), -1, dtype=torch.int64))[0]
    assert [hex(int(w)) for w in ones] == ["0x408f276d", "0x41c83b0e", "0xa20bc7c6", "0x6d5451fd"]


def _mask(shape, p, rng, shared):
    sizes = [1 if d in shared else s for d, s in enumerate(shape)]
    n = 1
    for s in sizes:
        n *= s
    words = philox(torch.arange((n + 3) // 4), torch.tensor(rng)).reshape(-1)[:n]
    return (words >= int(p * 2 ** 32)).view(sizes).expand(shape)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("shape,shared", [((1,), ()), ((7,), ()), ((33, 8), ()), ((1201, 8), ()), ((5, 49, 128), (1,)),
                                          ((6, 9, 13), (1,)), ((300, 4, 3), (1,)), ((4, 5, 6, 7), (1, 2)), ((2, 1, 9), (1,)),
                                          ((40, 16), (1,)), ((40, 16), (0,)), ((3, 2), (0, 1)), ((5000, 49, 4), (1,)),
                                          ((4099,), ()), ((129, 3, 37), (1,)), ((3, 2, 301), (1,))])
def test_values_and_gradients(device, dtype, shape, shared):
    rng = (2 ** 61 + 12345, 2 ** 40 + 7)
    x = torch.randn(shape, dtype=dtype, device=device, requires_grad=True)
    g = torch.randn(shape, dtype=dtype, device=device, requires_grad=True)
    keep = _mask(shape, 0.3, rng, shared).to(device)
    y = counter_dropout(x, 0.3, rng, shared)
    assert torch.equal(y, torch.where(keep, x * (1.0 / (1.0 - 0.3)), 0.0))
    (dx,) = torch.autograd.grad(y, x, g, create_graph=True)
    assert torch.equal(dx, torch.where(keep, g * (1.0 / (1.0 - 0.3)), 0.0))
    (gg,) = torch.autograd.grad(dx, g, x)
    assert torch.equal(gg, y)
    held = torch.tensor(rng, device=device)
    assert torch.equal(counter_dropout(x, 0.3, held, [d - len(shape) for d in shared]), y)


@pytest.mark.parametrize("device", DEVICES)
def test_law(device):
    """Kept shares within five standard deviations; another seed or offset gives an independent mask."""
    n = 1 << 18
    x = torch.ones(n, device=device)
    for p in (0.05, 0.5, 0.9):
        a, b, c = (counter_dropout(x, p, r) != 0 for r in ((1, 0), (1, 1), (2, 0)))
        for m in (a, b, c):
            assert abs(float(m.double().mean()) - (1 - p)) < 5 * (p * (1 - p) / n) ** 0.5
        for m in (b, c):
            both = (1 - p) ** 2
            assert abs(float((a & m).double().mean()) - both) < 5 * (both * (1 - both) / n) ** 0.5
    assert torch.equal(counter_dropout(x, 0.0, (1, 0)), x)
    assert not counter_dropout(x, 1.0, (1, 0)).any()
    bad = torch.full((64,), float("nan"), device=device)
    assert bool(((counter_dropout(bad, 0.5, (3, 0)) == 0) == ~_mask((64,), 0.5, (3, 0), ()).to(device)).all())


@pytest.mark.parametrize("device", DEVICES)
def test_strided_inputs(device):
    x = torch.randn(12, 10, device=device)
    for view in (x.t(), x[:, 1:], x[1:, 2:6], x.view(-1)[1:]):
        want = counter_dropout(view.contiguous().clone(), 0.4, (5, 6))
        assert torch.equal(counter_dropout(view, 0.4, (5, 6)), want)


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    x = torch.zeros(3, 4, 5, device=device)
    for kw, kind in ((dict(p=1.5), ValueError), (dict(p=-0.1), ValueError), (dict(p=float("nan")), ValueError),
                     (dict(shared=(3,)), ValueError), (dict(shared=(0, 2)), ValueError),
                     (dict(rng=torch.zeros(2, device=device)), ValueError),
                     (dict(rng=torch.zeros(3, dtype=torch.int64, device=device)), ValueError)):
        with pytest.raises(kind):
            counter_dropout(x, **{"p": 0.1, "rng": (1, 2), **kw})
    with pytest.raises(TypeError):
        counter_dropout(x.half(), 0.1, (1, 2))
    assert counter_dropout(x[:0], 0.1, (1, 2)).shape == (0, 4, 5)
    with pytest.raises(ValueError):
        CounterDropout(2.0)


@pytest.mark.parametrize("device", DEVICES)
def test_module(device):
    a, b = CounterDropout(0.5, seed=4).to(device), CounterDropout(0.5, seed=4).to(device)
    x = torch.randn(100, 8, device=device)
    first, second = a(x), a(x)
    assert not torch.equal(first, second)
    assert torch.equal(first, b(x)) and torch.equal(second, b(x))
    assert a.eval()(x) is x and CounterDropout(0.0)(x) is x
    assert not a.state_dict()


@pytest.mark.gpu
def test_captured_replays_draw_new_masks():
    drop = CounterDropout(0.5, seed=9).cuda()
    x = torch.ones(4096, device="cuda", requires_grad=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = drop(x)
        (g,) = torch.autograd.grad(y, x, torch.ones_like(y))
    seen = []
    for step in range(3):
        graph.replay()
        assert torch.equal(y, g)                 # the backward pass has the forward pass's mask
        assert torch.equal(y, counter_dropout(x, 0.5, (9, step)))
        seen.append(y.detach().clone())
    assert not torch.equal(seen[0], seen[1])


def test_module_refuses_a_recomputed_pass():
    """The second run of a checkpointed pass would meet another offset; the function with its numbers repeats its mask."""
    from torch.utils.checkpoint import checkpoint
    x = torch.randn(64, requires_grad=True)
    drop = CounterDropout(0.5, seed=3)
    y = checkpoint(lambda t: drop(t).square(), x, use_reentrant=False)
    with pytest.raises(RuntimeError, match="counter_dropout"):
        y.sum().backward()
    y = checkpoint(lambda t: counter_dropout(t, 0.5, (3, 7)).square(), x, use_reentrant=False)
    (g,) = torch.autograd.grad(y.sum(), x)
    kept = counter_dropout(torch.ones(64), 0.5, (3, 7))
    assert torch.equal(g, 2 * x.detach() * kept * kept)
