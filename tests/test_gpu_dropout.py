"""Dropout and the dropped Gaussians' activations against the generator's restatement, in 64 bits.

Tolerances: the factor 1 / (1 - T / 2^32) is rounded to float32 (2^-24), the product once more (2^-24) and the result to
its type (half a step: 2^-24, 2^-8, 2^-11); zeros are exact."""
import pytest
import torch

from tests import _draws

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = list(HALF)


def _x(shape, dtype, dev, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(dev)


def _check(y, x, keep, factor, spare=0.0):
    y, x = y.detach().cpu(), x.detach().cpu()
    keep = torch.as_tensor(keep).view([*y.shape[:y.dim()]]) if keep.size == y.numel() else torch.as_tensor(keep)
    want = torch.where(keep, x.double() * factor, 0.0)
    assert y.dtype == x.dtype and y.shape == x.shape
    assert bool((y[~keep.expand(y.shape)] == 0).all())
    bound = (HALF[y.dtype] + 2 * U + spare) * want.abs() + (2.0 ** -25 if y.dtype == torch.float16 else 0.0)
    assert bool(((y.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 63, 255, 4095, 4096, 4097, 100_003])
def test_elements(dev, dtype, n):
    from xsimgs_amd import rendering

    x = _x((n,), dtype, dev, n)
    for p, seed, stream in ((0.1, 5, 0), (0.73, 2 ** 63 - 1, 2 ** 31 - 1)):
        keep, factor = _draws.kept(n, p, seed, stream)
        _check(rendering.dropout(x, p, seed, stream=stream), x, keep, factor)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape, shared", [((5, 3), 1), ((1000, 3), 1), ((1000, 4), 1), ((77, 7), 1), ((513, 8), 1),
                                           ((300, 9), 1), ((1001, 16, 3), 2), ((33, 16, 3), 1), ((9, 4095), 1),
                                           ((7, 4096), 1), ((5, 4097), 1), ((3, 20_001), 1), ((11, 5), 2), ((40, 1), 1),
                                           ((6, 5, 4), 3), ((12, 100, 2), 0)])
def test_rows(dev, dtype, shape, shared):
    """Rows shorter and longer than a thread's eight elements and a workgroup's span."""
    from xsimgs_amd import rendering

    x = _x(shape, dtype, dev, 3)
    lead = shape[:len(shape) - shared]
    n = 1
    for k in lead:
        n *= k
    keep, factor = _draws.kept(n, 0.4, 99, 2)
    keep = torch.as_tensor(keep).view(*lead, *[1] * shared).expand(shape).numpy()
    dirty = x.clone()
    dirty[~torch.as_tensor(keep).to(dev)] = float("nan")     # what a dropped place holds does not matter
    y = rendering.dropout(dirty, 0.4, 99, stream=2, shared=shared)
    _check(y, x, keep, factor)


def test_ties_take_the_lower_bits(dev):
    """A threshold at a value's own 32 bits keeps it, one above drops it: the upper 16 alone do not tell."""
    from xsimgs_amd import rendering

    u = _draws.draws(0, 4000, 31)
    x = torch.ones(4000, device=dev)
    picked = [i for i in range(3, 4000, 211) if int(u[i]) & 0xFFFF not in (0, 0xFFFF)]
    assert len(picked) > 10
    for i in picked:
        for t, stays in ((int(u[i]), True), (int(u[i]) + 1, False)):
            y = rendering.dropout(x, t / 2 ** 32, 31).cpu().numpy()
            assert (y[i] != 0) == stays and ((y != 0) == (u >= t)).all()


def test_probabilities_at_the_ends(dev):
    from xsimgs_amd import rendering

    x = torch.full((1000,), float("inf"), device=dev, requires_grad=True)
    assert rendering.dropout(x, 0.0, 1) is x
    y = rendering.dropout(x, 1.0, 1)
    assert bool((y == 0).all())
    assert bool((torch.autograd.grad(y.sum(), x)[0] == 0).all())
    assert bool((rendering.drop_mask(1000, 1.0, 1, device=dev).view(torch.int32) == 0).all())
    words = rendering.drop_mask(1000, 0.0, 1, device=dev).cpu().view(torch.int32).numpy()
    assert (words[:31] == -1).all() and words[31] == 0xFF
    assert torch.equal(rendering.dropout(x.detach(), 1e-12, 1), x.detach())     # less than half a step of 2^-32
    for p in (-0.1, 1.1, float("nan")):
        for call in (lambda: rendering.dropout(x, p, 1), lambda: rendering.drop_mask(4, p, 1, device=dev),
                     lambda: rendering.activate_gaussians(torch.zeros(4, 3, device=dev), torch.zeros(4, device=dev), drop=p)):
            with pytest.raises(RuntimeError, match="probability"):
                call()


@pytest.mark.parametrize("dtype", TYPES)
def test_gradient_is_the_same_draws(dev, dtype):
    from xsimgs_amd import rendering

    x = _x((301, 7), dtype, dev).requires_grad_()
    g = _x((301, 7), dtype, dev, 9)
    keep, factor = _draws.kept(x.numel(), 0.3, 12)
    y = rendering.dropout(x, 0.3, 12)
    _check(torch.autograd.grad(y, x, g, retain_graph=True)[0], g, keep, factor)
    # a gradient that is broadcast, and one that is strided
    _check(torch.autograd.grad(y.sum(), x, retain_graph=True)[0], torch.ones_like(x), keep, factor)
    t = g.t().contiguous().t()
    _check(torch.autograd.grad(y, x, t)[0], g, keep, factor)


def test_strides_offsets_and_empty(dev):
    from xsimgs_amd import rendering

    big = _x((40, 33), torch.bfloat16, dev)
    for view in (big[:, 1:], big[1:, :32], big.t(), big[::2], big[:1].expand(5, 33), big.view(-1)[3:1000]):
        keep, factor = _draws.kept(view.numel(), 0.25, 4)
        _check(rendering.dropout(view, 0.25, 4), view, keep.reshape(view.shape), factor)
    for shape in ((0,), (0, 3), (4, 0)):
        for shared in range(len(shape) + 1):
            x = torch.zeros(shape, device=dev, requires_grad=True)
            y = rendering.dropout(x, 0.5, 1, shared=shared)
            assert y.shape == shape
            y.sum().backward()
            assert x.grad.shape == shape
    one = torch.full((), 3.0, device=dev)
    keep, factor = _draws.kept(1, 0.5, 8)
    _check(rendering.dropout(one, 0.5, 8), one, keep, factor)


def test_numbers_past_32_bits(dev):
    """Elements behind the first 2^32 and a row of more than 2^31."""
    from xsimgs_amd import rendering

    n = 2 ** 32 + 1000
    y = rendering.dropout(torch.ones(n, dtype=torch.bfloat16, device=dev), 0.5, 3)
    for first in (0, 2 ** 31 - 64, 2 ** 32 - 64, n - 100):
        keep, _ = _draws.kept(100, 0.5, 3, first=first)
        assert ((y[first:first + 100] != 0).cpu().numpy() == keep).all(), first
    del y
    row = 2 ** 31 + 5
    x = torch.ones(2 * row, dtype=torch.bfloat16, device=dev).view(2, row)
    seed = next(s for s in range(100) if _draws.kept(2, 0.5, s)[0].tolist() == [True, False])
    y = rendering.dropout(x, 0.5, seed, shared=1)
    assert bool((y[0] == 2).all()) and bool((y[1] == 0).all())


def test_other_types_and_places_are_refused(dev):
    from xsimgs_amd import rendering

    x = torch.zeros(8, device=dev)
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        rendering.dropout(x.double(), 0.5, 1)
    for seed, says in ((torch.zeros(2, dtype=torch.int64, device=dev), "one int64"),
                       (torch.zeros(1, device=dev), "one int64"), (torch.zeros(1, dtype=torch.int64), "must be on")):
        with pytest.raises(RuntimeError, match=says):
            rendering.dropout(x, 0.5, seed)
    for stream in (-1, 2 ** 31):
        with pytest.raises(RuntimeError, match="stream"):
            rendering.dropout(x, 0.5, 1, stream=stream)


@pytest.mark.parametrize("n", [1, 3, 4, 8, 9, 31, 1000, 10_001])
@pytest.mark.parametrize("shape", [(), (1,)])
def test_gaussians(dev, n, shape):
    """sigmoid and exp are good to a few units of float32 (8 U taken), 1 - s to one of 1."""
    from xsimgs_amd import rendering

    a = _x((n, 3), torch.float32, dev, 1).requires_grad_()
    o = _x((n, *shape), torch.float32, dev, 2).requires_grad_()
    keep, factor = _draws.kept(n, 0.35, 17, 5)
    keep = torch.as_tensor(keep).view(o.shape)
    scales, opac = rendering.activate_gaussians(a, o, drop=0.35, seed=17, stream=5)
    plain = rendering.activate_gaussians(a.detach(), o.detach())
    assert torch.equal(scales.detach(), plain[0])
    s = torch.sigmoid(o.detach().cpu().double())
    want = torch.where(keep, s * factor, 0.0)
    assert bool(((opac.detach().cpu().double() - want).abs() <= 10 * U * want).all())
    va, vo = _x(a.shape, torch.float32, dev, 3), _x(o.shape, torch.float32, dev, 4)
    ga, go = torch.autograd.grad([scales, opac], [a, o], [va, vo], retain_graph=True)
    assert torch.equal(ga, va * plain[0])
    want = torch.where(keep, vo.cpu().double() * factor * s * (1 - s), 0.0)
    assert bool(((go.cpu().double() - want).abs() <= 16 * U * vo.cpu().double().abs() * factor * s).all())
    assert bool((go.cpu()[~keep] == 0).all())
    # one output alone
    assert torch.equal(torch.autograd.grad(opac, o, vo, retain_graph=True)[0], go)
    assert torch.equal(torch.autograd.grad(scales, a, va)[0], ga)
    bits = rendering.drop_mask(n, 0.35, 17, stream=5, device=dev).cpu().view(torch.int32)
    got = (bits.long().view(-1, 1) >> torch.arange(32)) & 1
    assert torch.equal(got.view(-1)[:n].bool(), keep.view(-1)) and not bool(got.view(-1)[n:].any())


def test_gaussians_strided(dev):
    from xsimgs_amd import rendering

    both = _x((501, 4), torch.float32, dev, 6)
    a, o = both[:, 1:].clone().requires_grad_(), both[:, 0].clone().requires_grad_()
    va, vo = _x((501, 3), torch.float32, dev, 7), _x((501,), torch.float32, dev, 8)
    wide = both.clone().requires_grad_()
    one = rendering.activate_gaussians(a, o, drop=0.2, seed=3)
    two = rendering.activate_gaussians(wide[:, 1:], wide[:, 0], drop=0.2, seed=3)
    assert all(torch.equal(x, y) for x, y in zip(one, two))
    ga, go = torch.autograd.grad(one, [a, o], [va, vo])
    gw, = torch.autograd.grad(two, wide, [va, vo])
    assert torch.equal(gw[:, 1:], ga) and torch.equal(gw[:, 0], go)
    # buffers at an odd place
    flat = _x((4 * 501 + 1,), torch.float32, dev, 6)
    odd = rendering.activate_gaussians(flat[1:1504].view(501, 3), flat[1504:], drop=0.2, seed=3)
    even = rendering.activate_gaussians(flat[1:1504].view(501, 3).clone(), flat[1504:].clone(), drop=0.2, seed=3)
    assert all(torch.equal(x, y) for x, y in zip(odd, even))


def test_seed_on_the_gpu_and_graphs(dev):
    """A captured forward and backward draw anew when the seed's tensor changes between replays."""
    from xsimgs_amd import rendering

    x = _x((1003,), torch.float32, dev).requires_grad_()
    g = _x((1003,), torch.float32, dev, 1)
    seed = torch.full((1,), 40, dtype=torch.int64, device=dev)
    assert torch.equal(rendering.dropout(x, 0.3, seed), rendering.dropout(x, 0.3, 40))
    assert torch.equal(rendering.drop_mask(99, 0.3, seed).view(torch.int32), rendering.drop_mask(99, 0.3, 40, device=dev).view(torch.int32))

    def both():
        y = rendering.dropout(x, 0.3, seed)
        return y.detach(), torch.autograd.grad(y, x, g)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for s in (40, 41, 2 ** 40 + 3, 40):
        seed.fill_(s)
        graph.replay()
        torch.cuda.synchronize()
        keep, factor = _draws.kept(1003, 0.3, s)
        _check(out[0], x, keep, factor)
        _check(out[1], g, keep, factor)
    y = rendering.dropout(x, 0.3, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_streams(dev):
    from xsimgs_amd import rendering

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        x = torch.randn(1_000_003, device=dev)
        y = rendering.dropout(x, 0.5, 6)
        z = y * 1.0
    side.synchronize()
    keep, factor = _draws.kept(1_000_003, 0.5, 6)
    _check(z, x, keep, factor)
