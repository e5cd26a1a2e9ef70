"""Attention over the atoms of each structure against its definition in 64 bits: outputs, gradients and second
gradients over head layouts, widths, lengths from none to long, masks and strides.

Tolerances count roundings of the operands' type, half a step (``eps / 2``) each, in the 2-norm of the
whole result: an output element passes the products of its score, the exponential, the running sums
and the final division. With scores of a few units and sums whose roundings are independent that is
below 64 of them for outputs and gradients and below 128 for second gradients, which chain two such
expressions."""
import pytest
import torch

from xnn_b200.ops import structure_attention

CASES = [
    # lengths, heads, key heads, width, masked share, rows behind the last structure
    ([1], 1, 1, 64, 0.0, 0),
    ([21], 1, 1, 64, 0.0, 0),
    ([0, 5, 0, 0, 2], 2, 1, 8, 0.0, 0),
    ([32, 1, 33, 31], 4, 2, 20, 0.0, 3),
    ([9, 17, 29, 12, 3], 1, 1, 64, 0.3, 0),
    ([64, 65, 63], 2, 2, 32, 0.0, 0),
    ([128, 129, 127, 1], 2, 2, 128, 0.0, 5),
    ([200, 3, 0, 31], 8, 2, 50, 0.1, 0),
    ([300, 70], 3, 1, 1, 0.0, 0),
    ([77, 140], 2, 1, 100, 0.2, 0),
    ([700], 1, 1, 64, 0.0, 0),
    ([1200], 2, 1, 33, 0.05, 1),
    ([400, 500], 4, 4, 64, 0.0, 0),
    ([150] + [4] * 60, 2, 2, 32, 0.1, 0),
]


def _inputs(case, dtype, device, seed=0):
    lens, h, hk, d, masked, tail = case
    g = torch.Generator().manual_seed(seed)
    n = sum(lens) + tail
    ptr = torch.tensor([0] + lens).cumsum(0)
    make = lambda heads: torch.randn(n, heads, d, generator=g, dtype=torch.float64).to(dtype).to(device)  # noqa: E731
    q, k, v, do, a, b, c = make(h), make(hk), make(hk), make(h), make(h), make(hk), make(hk)
    mask = None
    if masked:
        mask = torch.rand(n, generator=g) >= masked
        mask[:lens[0]] = len(lens) == 1          # a whole structure that nobody attends to
        mask = mask.to(device)
    return q, k, v, do, a, b, c, ptr.to(device), mask


def _definition(q, k, v, ptr, mask, scale):
    out = []
    wide = torch.arange(q.shape[1], device=q.device) // (q.shape[1] // k.shape[1])
    bounds = ptr.tolist()
    for lo, hi in zip(bounds[:-1], bounds[1:]):
        keys = torch.arange(lo, hi, device=q.device)
        if mask is not None:
            keys = keys[mask[lo:hi]]
        if hi == lo:
            continue
        if keys.numel() == 0:
            out.append(torch.zeros_like(q[lo:hi]))
            continue
        s = scale * torch.einsum("ihd,jhd->hij", q[lo:hi], k[keys][:, wide])
        out.append(torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), v[keys][:, wide]))
    out.append(torch.zeros_like(q[bounds[-1]:]))
    return torch.cat(out)


def _all(fn, q, k, v, do, a, b, c, second=True):
    q, k, v, do = (t.detach().requires_grad_() for t in (q, k, v, do))
    o = fn(q, k, v)
    first = torch.autograd.grad(o, (q, k, v), do, create_graph=second, allow_unused=True, materialize_grads=True)
    if not second or not any(f.requires_grad for f in first):
        return (o,) + first
    more = torch.autograd.grad(first, (q, k, v, do), (a, b, c), allow_unused=True, materialize_grads=True)
    return (o,) + first + more


def _check(got, want, dtype, counts):
    for i, (x, y) in enumerate(zip(got, want)):
        y = y.double()
        # What is zero by cancellation (a single key: dq, dk and all second gradients) is compared with the size of
        # its terms. With normal inputs and scale = D^-1/2, dP and E are of size D^1/2 and T of size 2^1/2, so the
        # terms scale dP k and do P of the gradients are of size 1 an element, and scale (T dP + E) k, T do, T v of
        # the second ones of size 3^1/2, 2^1/2, 2^1/2: one per element is below all of them.
        size = max(float(y.detach().norm()), float(y.numel()) ** 0.5)
        off = float((x.detach().double() - y).norm())
        assert off <= counts[i] * torch.finfo(dtype).eps / 2 * size, (i, off / size)


COUNTS = (64,) * 4 + (128,) * 4


def _run(case, dtype, device):
    q, k, v, do, a, b, c, ptr, mask = _inputs(case, dtype, device)
    scale = q.shape[2] ** -0.5
    most = max(case[0])
    got = _all(lambda *t: structure_attention(*t, ptr, max_len=most, key_mask=mask), q, k, v, do, a, b, c)
    want = _all(lambda *t: _definition(*t, ptr, mask, scale), *(t.double() for t in (q, k, v, do, a, b, c)))
    _check(got, want, dtype, COUNTS)
    return got


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_formula(case, dtype):
    _run(case, dtype, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_kernels(case, dtype):
    got = _run(case, dtype, "cuda")
    again = _run(case, dtype, "cuda")
    assert all(torch.equal(x, y) for x, y in zip(got, again))


def _refusals(device):
    q, k, v, *_, ptr, _ = _inputs(([4, 3], 2, 1, 8, 0.0, 0), torch.float32, device)
    ok = dict(ptr=ptr, max_len=4)
    mask = torch.ones(7, dtype=torch.bool, device=device)
    assert structure_attention(q, k, v, **ok, key_mask=mask).shape == (7, 2, 8)
    for bad, kind in (
            ((q[0], k, v), ValueError), ((q, k.double(), v), TypeError), ((q.half(), k.half(), v.half()), TypeError),
            ((q, k[:5], v[:5]), ValueError), ((q, k, v[..., :4]), ValueError),
            ((q, k.expand(-1, 3, -1), v.expand(-1, 3, -1)), ValueError), ((q, k[:, :0], v[:, :0]), ValueError)):
        with pytest.raises(kind):
            structure_attention(*bad, **ok)
    for wrong in (dict(ptr=ptr.int()), dict(ptr=ptr[None]), dict(ptr=ptr[:0]), dict(max_len=-1),
                  dict(key_mask=mask.int()), dict(key_mask=mask[:3])):
        with pytest.raises(ValueError):
            structure_attention(q, k, v, **{**ok, **wrong})


def test_refusals():
    _refusals("cpu")
    q, k, v, *_, ptr, _ = _inputs(([4, 3], 2, 1, 8, 0.0, 0), torch.float32, "cpu")
    for wrong in (dict(max_len=3), dict(ptr=torch.tensor([0, 5, 4])), dict(ptr=torch.tensor([0, 9])), dict(ptr=torch.tensor([-1, 4]))):
        with pytest.raises(ValueError):
            structure_attention(q, k, v, **{"ptr": ptr, **wrong})


@pytest.mark.gpu
def test_refusals_gpu():
    _refusals("cuda")
    q = torch.zeros(4, 1, 130, device="cuda")
    ptr = torch.tensor([0, 4], device="cuda")
    with pytest.raises(ValueError):
        structure_attention(q, q, q, ptr)
    with pytest.raises(ValueError):
        structure_attention(q[..., :8], q[..., :8], q[..., :8], ptr.cpu())
    x = torch.randn(4, 1, 8, device="cuda", requires_grad=True)
    g = torch.autograd.grad(structure_attention(x, x, x, ptr).square().sum(), x, create_graph=True)[0]
    g2 = torch.autograd.grad(g.square().sum(), x, create_graph=True)[0]
    with pytest.raises(RuntimeError):           # the third derivative is refused, not wrong
        torch.autograd.grad(g2.sum(), x)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_empty_batches(device):
    for n, ptr in ((0, [0]), (0, [0, 0, 0]), (3, [0]), (3, [0, 0]), (3, [3, 3])):
        q = torch.randn(n, 2, 8, device=device, requires_grad=True)
        o = structure_attention(q, q, q, torch.tensor(ptr, device=device))
        (g,) = torch.autograd.grad(o.sum(), q)
        assert o.shape == q.shape and not o.any() and not g.any()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("lens", [[20, 11, 25], [90, 70, 200], [300, 260, 513]])
def test_hidden_values_do_not_spread(device, lens):
    """NaN and infinities of masked atoms, of another structure and of the padding rows stay there."""
    q, k, v, do, a, b, c, ptr, mask = _inputs((lens, 2, 2, 16, 0.3, 4), torch.float32, device)
    mask[lens[0]] = True
    run = lambda *t: structure_attention(*t, ptr, max_len=max(lens), key_mask=mask)  # noqa: E731
    clean = _all(run, q, k, v, do, a, b, c)
    last = slice(lens[0] + lens[1], None)
    k[~mask], v[~mask] = float("nan"), float("inf")
    b[~mask], c[~mask] = float("inf"), float("nan")
    for t in (q, k, v, do, a, b, c):
        t[last] = float("nan")
    dirty = _all(run, q, k, v, do, a, b, c)
    kept = slice(0, lens[0] + lens[1])
    for x, y in zip(clean, dirty):
        assert torch.equal(x[kept], y[kept])
        assert not y[sum(lens):].any()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("lens,width", [([20, 11], 16), ([90, 70], 16), ([90, 70], 72), ([400], 64)])
def test_no_gradient_where_no_key_is(device, dtype, lens, width):
    """Rows without an allowed key, with NaN as queries and as incoming gradients (0 / 0 of a padded row), get zeros, and
    so do masked keys next to valid ones."""
    q, k, v, do, a, b, c, ptr, _ = _inputs((lens, 2, 1, width, 0.0, 0), dtype, device)
    mask = torch.ones(sum(lens), dtype=torch.bool, device=device)
    mask[:lens[0]] = False                       # the first structure has no key
    mask[lens[0] + 1::3] = False
    q[:lens[0]], do[:lens[0]] = float("nan"), float("nan")
    run = lambda *t: structure_attention(*t, ptr, max_len=max(lens), key_mask=mask)  # noqa: E731
    _, *first = _all(run, q, k, v, do, a, b, c, second=False)
    _, *both = _all(run, q, k, v, do, a, b, c)
    for x in first + both:
        assert not x[:lens[0]].any() and not x.isnan().any()
    do[lens[0]:] = float("nan")                  # what a masked key hides from the queries, it does not take from them
    for x in _all(run, q, k, v, do, a, b, c, second=False)[2:]:
        assert not x[~mask].any()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_large_scores(device):
    """Scores of thousands: the running maximum keeps every power in range, and one key takes all."""
    q, k, v, do, *_, ptr, _ = _inputs(([150, 40], 1, 1, 32, 0.0, 0), torch.float64, device)
    q = q * 1e3
    got = structure_attention(q, k, v, ptr)
    want = _definition(q, k, v, ptr, None, 32 ** -0.5)
    # a score of 1e4 is off by 1e4 * 64 halves of a step, and so is the exponential's relative error
    assert float((got - want).norm() / want.norm()) < 64e4 * torch.finfo(torch.float64).eps / 2


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("lens", [[30, 7, 22], [150, 333]])
def test_strides(dtype, lens):
    """Views of one packed projection, rows on odd addresses, expanded heads and gradients."""
    n, h, d = sum(lens), 2, 24
    ptr = torch.tensor([0] + lens).cumsum(0).cuda()
    g = torch.Generator("cuda").manual_seed(1)
    packed = torch.randn(n, 3, h, d, generator=g, device="cuda", dtype=dtype)
    odd = torch.randn(n * 3 * h * d + 1, generator=g, device="cuda", dtype=dtype)[1:].view(n, h, 3, d)
    one = torch.randn(n, 1, d, generator=g, device="cuda", dtype=dtype)
    for q, k, v in (packed.unbind(1), odd.unbind(2), (packed[:, 0], one.expand(-1, h, -1), one.expand(-1, h, -1)),
                    (packed[:, 0].transpose(1, 2).contiguous().transpose(1, 2), packed[:, 1], packed[:, 2])):
        do = torch.ones((), device="cuda", dtype=dtype).expand(n, h, d)
        a, b, c = (torch.randn(n, h, d, generator=g, device="cuda", dtype=dtype) for _ in range(3))
        got = _all(lambda *t: structure_attention(*t, ptr, max_len=max(lens)), q, k, v, do, a, b, c)
        want = _all(lambda *t: _definition(*t, ptr, None, d ** -0.5), *(t.double() for t in (q, k, v, do, a, b, c)))
        _check(got, want, dtype, COUNTS)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("lens", [[33] + [2] * 40, [3] * 500 + [1000] + [1] * 300 + [33, 34, 0, 64, 65, 32, 128, 129], [4] * 90 + [70, 0, 63]])
@pytest.mark.parametrize("before", [0, 5, 70])
def test_few_long_among_many_short(dtype, lens, before):
    """Both classes in one batch, with rows in front of the first structure and behind the last."""
    h, d, behind = 2, 16, 40
    n = before + sum(lens) + behind
    ptr = torch.tensor([before] + lens).cumsum(0).cuda()
    g = torch.Generator("cuda").manual_seed(2)
    q, k, v, do, a, b, c = (torch.randn(n, h, d, generator=g, device="cuda", dtype=dtype) for _ in range(7))
    got = _all(lambda *t: structure_attention(*t, ptr, max_len=max(lens)), q, k, v, do, a, b, c)
    inner = slice(before, n - behind)
    want = _all(lambda *t: _definition(*t, ptr - before, None, d ** -0.5), *(t[inner].double() for t in (q, k, v, do, a, b, c)))
    _check([x[inner] for x in got], want, dtype, COUNTS)
    assert not any(x[:before].any() or x[n - behind:].any() for x in got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("width", [3, 31, 64, 65, 96, 113, 128])
@pytest.mark.parametrize("heads", [(1, 1), (6, 2)])
def test_short_structures_at_every_width(dtype, width, heads):
    _run(([3, 32, 1, 17, 0, 30, 8], *heads, width, 0.2, 2), dtype, "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[12, 30], [40, 600], [500, 900]])
def test_wrong_bound_is_loud_or_right(lens):
    """A structure longer than ``max_len``: its gradients are right or NaN, the others' are right."""
    q, k, v, do, *_, ptr, _ = _inputs((lens, 1, 1, 32, 0.0, 0), torch.float32, "cuda")
    right = _all(lambda *t: structure_attention(*t, ptr), q, k, v, do, *[None] * 3, second=False)
    got = _all(lambda *t: structure_attention(*t, ptr, max_len=10), q, k, v, do, *[None] * 3, second=False)
    for i, (x, y) in enumerate(zip(got, right)):
        fine = x.isnan() | ((x - y).abs() <= 256 * torch.finfo(torch.float32).eps * y.abs().max())
        assert bool(fine.all()), i
    assert not got[0].isnan().any()


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[9, 25, 14], [130, 61], [900]])
def test_captured_and_on_another_stream(lens):
    case = (lens, 2, 1, 32, 0.0, 0)
    q, k, v, do, a, b, c, ptr, _ = _inputs(case, torch.float32, "cuda")
    run = lambda: _all(lambda *t: structure_attention(*t, ptr, max_len=max(lens)), q, k, v, do, a, b, c)  # noqa: E731
    eager = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(eager, other))
    graphs = []
    for _ in range(2):                          # two graphs with their own workspaces
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        graphs.append((graph, out))
    fresh = _inputs(case, torch.float32, "cuda", seed=5)
    for old, new in zip((q, k, v, do, a, b, c), fresh):
        old.copy_(new)
    eager = run()
    for graph, _ in graphs:
        graph.replay()
    for _, out in graphs:
        assert all(torch.equal(x, y) for x, y in zip(eager, out))


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_gradients_against_differences(device):
    q, k, v, *_, ptr, mask = _inputs(([5, 3, 7], 2, 1, 4, 0.2, 1), torch.float64, device)
    inputs = tuple(t.requires_grad_() for t in (q, k, v))
    fn = lambda *t: structure_attention(*t, ptr, key_mask=mask)  # noqa: E731
    assert torch.autograd.gradcheck(fn, inputs)
    assert torch.autograd.gradgradcheck(fn, inputs)
