"""Derivatives and transforms that the CUDA kernels of the transformer operators do not have are refused, not dropped."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from xnn_b200.ops import counter_dropout, embedding_lookup, structure_attention


def _calls(device):
    ptr = torch.tensor([0, 9, 50], device=device)
    ids = torch.tensor([3, 0, 3, -1], device=device)
    other = torch.randn(50, 2, 16, device=device)
    return {"attention": (lambda t: structure_attention(t, t, t, ptr), (50, 2, 16)),
            "attention_keys": (lambda t: structure_attention(other, t, other, ptr), (50, 2, 16)),
            "attention_values": (lambda t: structure_attention(other, other, t, ptr), (50, 2, 16)),
            "dropout": (lambda t: counter_dropout(t, 0.3, (1, 2)), (50, 2, 16)),
            "lookup": (lambda t: embedding_lookup(t, ids), (5, 16))}


NAMES = ["attention", "attention_keys", "attention_values", "dropout", "lookup"]


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("leaf", [False, True])
def test_tangents_are_refused(name, leaf):
    fn, shape = _calls("cuda")[name]
    x = torch.randn(shape, device="cuda").requires_grad_(leaf)
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            fn(forward_ad.make_dual(x, torch.ones_like(x)))
    assert fn(x).shape[-1] == 16                # an ordinary call afterwards is served


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("graph", [False, True])
def test_tangents_of_incoming_gradients_are_refused(name, graph):
    fn, shape = _calls("cuda")[name]
    x = torch.randn(shape, device="cuda", requires_grad=True)
    y = fn(x)
    with forward_ad.dual_level():
        g = forward_ad.make_dual(torch.randn_like(y), torch.ones_like(y))
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(y, x, g, create_graph=graph)


def test_tangents_on_the_cpu():
    """The formula of attention carries them, the other two refuse them."""
    calls = _calls("cpu")
    fn, shape = calls["attention"]
    x, u = torch.randn(shape, dtype=torch.float64), torch.randn(shape, dtype=torch.float64)
    with forward_ad.dual_level():
        tangent = forward_ad.unpack_dual(fn(forward_ad.make_dual(x, u))).tangent
    step = 1e-6
    # central differences: the remainder is of size step^2, a value's rounding is divided by step
    assert float((tangent - (fn(x + step * u) - fn(x - step * u)) / (2 * step)).abs().max()) < 1e-8
    for name in ("dropout", "lookup"):
        fn, shape = calls[name]
        with forward_ad.dual_level(), pytest.raises(NotImplementedError):
            fn(forward_ad.make_dual(torch.randn(shape), torch.ones(shape)))


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("leaf", [False, True])
def test_traces_are_refused(name, leaf):
    """A trace would keep the example's result whatever its inputs are later."""
    fn, shape = _calls("cuda")[name]
    x = torch.randn(shape, device="cuda").requires_grad_(leaf)
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda t: fn(t) + t.sum(), (x,), check_trace=False)
    assert fn(x).shape[-1] == 16


def test_traced_attention_on_the_cpu():
    """Longer structures than the example's, shorter ones and other counts."""
    def inputs(lens):
        n = sum(lens)
        return (torch.randn(n, 2, 4), torch.randn(n, 1, 4), torch.randn(n, 1, 4), torch.tensor([0] + lens).cumsum(0))
    traced = torch.jit.trace(structure_attention, inputs([5, 3]), check_trace=False)
    for lens in ([5, 3], [9, 2, 7], [1], [4, 0, 2, 30]):
        args = inputs(lens)
        assert torch.equal(traced(*args), structure_attention(*args))


@pytest.mark.gpu
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("lens", [[9, 20], [50]])
def test_third_derivative_through_the_incoming_gradient_is_refused(turned, lens):
    """Refused on the path through the cotangent of the output too, contiguous or not."""
    n = sum(lens)
    ptr = torch.tensor([0] + lens).cumsum(0).cuda()
    q, k, v = (torch.randn(n, 2, 16, device="cuda", requires_grad=True) for _ in range(3))
    y = torch.randn((16, 2, n) if turned else (n, 2, 16), device="cuda", requires_grad=True)
    do = y.square().permute(2, 1, 0) if turned else y.square()
    (dq,) = torch.autograd.grad(structure_attention(q, k, v, ptr), q, do, create_graph=True)
    second = torch.autograd.grad(dq, (q, k, v), torch.ones_like(dq), create_graph=True)
    with pytest.raises(RuntimeError, match="not three times"):
        torch.autograd.grad(sum(t.sum() for t in second), y, allow_unused=True)
