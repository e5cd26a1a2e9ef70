"""The transformer operators where models use them, and a training step through all of them together."""
import pytest
import torch
from torch import nn

from xnn_b200.data import collate, structure_to_graph, synthetic
from xnn_b200.models import ForceStressOutput
from xnn_b200.models.equiformer_v2 import EquiformerV2
from xnn_b200.models.spookynet import NonlocalInteraction, PackedAtoms, SpookyNet, structure_slots
from xnn_b200.ops import CounterDropout, ScaledEmbedding, structure_attention

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


class Block(nn.Module):
    """Elements looked up, attention over each structure's atoms, dropout, an energy per structure."""

    def __init__(self, width=32, heads=2):
        super().__init__()
        self.table = ScaledEmbedding(20, width, scale=0.5)
        self.qkv = nn.Linear(width, 3 * width)
        self.drop = CounterDropout(0.25, seed=11)
        self.out = nn.Linear(width, 1)
        self.heads = heads

    def forward(self, z, pos, ptr, most):
        x = self.table(z) + torch.cos(pos @ pos.new_ones(3, 1) * torch.arange(32, device=pos.device) * 0.1)
        q, k, v = self.qkv(x).view(-1, 3, self.heads, 32 // self.heads).unbind(1)
        return self.out(x + self.drop(structure_attention(q, k, v, ptr, max_len=most).flatten(1))).sum()


def _step(block, z, pos, ptr, most):
    """Energy, forces and the parameters' gradients of a loss on both: one dropout mask, two derivatives."""
    pos = pos.detach().requires_grad_()
    e = block(z, pos, ptr, most)
    (f,) = torch.autograd.grad(e, pos, create_graph=True)
    loss = e * 0.01 + f.square().sum()
    return [e, f] + list(torch.autograd.grad(loss, list(block.parameters())))


@pytest.mark.parametrize("lens", [[7, 12, 3], [80, 40, 150]])
@pytest.mark.parametrize("device", DEVICES)
def test_together(device, lens):
    torch.manual_seed(3)
    block = Block().to(device)
    wide = Block().double()
    wide.load_state_dict(block.state_dict())
    n = sum(lens)
    z, pos, ptr = torch.randint(-1, 20, (n,)), torch.randn(n, 3), torch.tensor([0] + lens).cumsum(0)
    got = _step(block, z.to(device), pos.to(device), ptr.to(device), max(lens))
    want = _step(wide, z, pos.double(), ptr, max(lens))
    for x, y in zip(got, want):
        # some ten operations of at most a hundred independent roundings each, and sums over up to 270 atoms that
        # cancel to a tenth of their terms
        assert float((x.detach().double().cpu() - y.detach()).norm()) <= 1e4 * torch.finfo(torch.float32).eps / 2 * max(float(y.detach().norm()), 1e-2)


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[7, 12, 3], [80, 40, 150]])
def test_captured_step(lens):
    """A captured training step replays: each time with a new mask, the same as the eager step that draws it. (No
    eager graph over the parameters may live during the capture: PyTorch ties their gradient nodes to the stream
    that first met them, whatever the operators.)"""
    block = Block().cuda()
    n = sum(lens)
    z, pos = torch.randint(-1, 20, (n,), device="cuda"), torch.randn(n, 3, device="cuda")
    ptr = torch.tensor([0] + lens).cumsum(0).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            _step(block, z, pos, ptr, max(lens))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(block, z, pos, ptr, max(lens))
    for _ in range(2):
        at = block.drop.rng.clone()
        graph.replay()
        after = block.drop.rng.clone()
        block.drop.rng.copy_(at)
        eager = _step(block, z, pos, ptr, max(lens))
        assert torch.equal(block.drop.rng, after)
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


def _molecules(count, seed=0):
    return collate([structure_to_graph(s, 4.5) for s in synthetic.organic_molecules(count, seed=seed)])


def _spooky(dtype=torch.float64, **kw):
    torch.manual_seed(1)
    m = SpookyNet(n_features=16, n_interactions=2, n_rbf=6, cutoff=4.5, d4_dispersion=False, attention="softmax", **kw)
    with torch.no_grad():
        for p in m.parameters():
            p.add_(0.05 * torch.randn_like(p))
    return m.to(dtype)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("heads", [1, 4])
def test_nonlocal_interaction(device, heads):
    """One structure at a time by the definition; structures in any order in the batch."""
    torch.manual_seed(0)
    net = NonlocalInteraction(16, 1, None, heads=heads).double().to(device)
    with torch.no_grad():
        for p in net.parameters():
            p.add_(0.3 * torch.randn_like(p))
    batch = torch.tensor([2, 0, 0, 1, 2, 1, 0, 2, 2]).to(device)
    x = torch.randn(9, 16, dtype=torch.float64, device=device)
    for b in (batch, batch.sort().values, torch.zeros_like(batch)):
        g = int(b.max()) + 1
        slot, most = structure_slots(b, g)
        got = net(x, b, g, slot, most)
        q, k, v = (m(x).view(9, heads, -1) for m in (net.resmlp_q, net.resmlp_k, net.resmlp_v))
        for s in range(g):
            on = b == s
            w = torch.softmax(torch.einsum("ihc,jhc->hij", q[on], k[on]) / (16 // heads) ** 0.5, -1)
            assert torch.allclose(got[on], torch.einsum("hij,jhc->ihc", w, v[on]).flatten(1), rtol=0, atol=1e-12)


def test_packed_atoms():
    """First rows, order and places, for one structure without reading anything back."""
    one = PackedAtoms(torch.zeros(5, dtype=torch.long), 1, torch.arange(5), 5)
    assert one.ptr.tolist() == [0, 5] and one.ptr.dtype == torch.int64 and one.order is None
    mixed = PackedAtoms(torch.tensor([1, 0, 1, 2, 0]), 4, torch.tensor([0, 0, 1, 0, 1]), 2)
    assert mixed.ptr.tolist() == [0, 2, 4, 5, 5]
    assert mixed.order.tolist() == [1, 4, 0, 2, 3] and mixed.place.tolist() == [2, 0, 3, 4, 1]


@pytest.mark.gpu
def test_one_structure_is_captured():
    torch.manual_seed(3)
    layer = NonlocalInteraction(16, 1, None, heads=2).cuda()
    for mlp in (layer.resmlp_q, layer.resmlp_k, layer.resmlp_v):
        for p in mlp.parameters():
            torch.nn.init.normal_(p, std=0.3)
    x, batch, slot = torch.randn(40, 16, device="cuda"), torch.zeros(40, dtype=torch.long, device="cuda"), torch.arange(40, device="cuda")
    run = lambda: layer(x, batch, 1, slot, 40)  # noqa: E731
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        x.copy_(torch.randn(40, 16, device="cuda"))
        graph.replay()
        assert torch.equal(out, run()) and bool(out.any())


def test_spookynet_options():
    for kw in (dict(attention_heads=3), dict(attention_heads=0)):
        with pytest.raises(ValueError):
            SpookyNet(n_features=16, attention="softmax", d4_dispersion=False, **kw)
    with pytest.raises(ValueError):
        SpookyNet(n_features=16, attention="exact", attention_heads=2, d4_dispersion=False)
    a, b = _spooky(), SpookyNet(n_features=16, n_interactions=2, n_rbf=6, cutoff=4.5, d4_dispersion=False, attention="exact")
    assert {k: v.shape for k, v in a.state_dict().items()} == {k: v.shape for k, v in b.state_dict().items()}


@pytest.mark.gpu
def test_spookynet_force_training_on_gpu():
    """Energies, forces and the gradients of a force loss in float64: kernels against the CPU's formula."""
    results = []
    for device in ("cpu", "cuda"):
        model = ForceStressOutput(_spooky(attention_heads=2).to(device)).train()
        data = _molecules(3).to(device)
        out = model(data)
        loss = out["energy"].square().sum() + out["forces"].square().sum()
        results.append([out["energy"], out["forces"]] + list(torch.autograd.grad(loss, [p for p in model.parameters() if p.requires_grad], allow_unused=True)))
    for x, y in zip(*results):
        assert (x is None) == (y is None)
        if x is not None:
            assert float((x - y.cpu()).norm()) <= 1e-9 * max(1.0, float(x.norm()))


def _equiformer(**kw):
    torch.manual_seed(2)
    return EquiformerV2(n_features=8, n_interactions=1, cutoff=4.5, n_rbf=8, l_max=2, m_max=2, num_heads=2, attn_hidden_channels=8,
                        attn_alpha_channels=8, attn_value_channels=4, ffn_hidden_channels=8, edge_channels=8, **kw)


def test_equiformer_sorted_lookup():
    """The same parameters, outputs and gradients."""
    a, b = _equiformer().double(), _equiformer(sorted_lookup=True).double()
    b.load_state_dict(a.state_dict())
    data = _molecules(2)
    for m in (a, b):
        m(data)["energy"].sum().backward()
    assert torch.equal(a(data)["energy"], b(data)["energy"])
    for x, y in zip(a.parameters(), b.parameters()):
        assert (x.grad is None) == (y.grad is None)
        if x.grad is not None:
            assert torch.allclose(x.grad, y.grad, rtol=1e-12, atol=1e-14)
    with pytest.raises(ValueError):
        _equiformer(dropout_rng="other")


@pytest.mark.gpu
def test_equiformer_counter_dropout_on_gpu():
    """The same masks on both devices: a training pass with dropout agrees with the CPU's, a second one differs."""
    outs = []
    for device in ("cpu", "cuda"):
        torch.manual_seed(4)
        m = _equiformer(dropout_rng="counter", sorted_lookup=True, alpha_drop=0.2, proj_drop=0.3).double().to(device).train()
        data = _molecules(2).to(device)
        first, second = m(data)["energy"], m(data)["energy"]
        grads = torch.autograd.grad(first.sum(), [p for p in m.parameters() if p.requires_grad], allow_unused=True)
        assert not torch.equal(first, second)
        outs.append([first, second] + [g for g in grads if g is not None])
        # without dropout the same energies, but for the order of the model's other sums over edges
        m.eval()
        assert torch.allclose(m(data)["energy"], m(data)["energy"], rtol=0, atol=1e-12)
    for x, y in zip(*outs):
        assert float((x - y.cpu()).norm()) <= 1e-9 * max(1.0, float(x.norm()))
