"""The training step's operators where their kernels go different ways: lists longer than a launch's arguments
hold (with more masks and rates than a piece of their table), more data than the caches hold, rows of every
length under a mask, tensors that start anywhere in a buffer, and the edges between small and ordinary calls.
Each against float64, with the tolerances of test_gpu_optim."""
import math

import numpy as np
import pytest
import torch

from tests.test_gpu_optim import (BETAS, EPS, HALF_ULP, SMALLEST, TYPES, U, _adam64, _adam_bounds, _check_update, _close,
                                  _f64, _norm64, _pack, _state, _values)

pytestmark = pytest.mark.gpu


def _keep(n, share, seed):
    return np.random.default_rng(seed).random(n) < share


@pytest.mark.parametrize("count", [51, 52, 53, 88, 89, 130, 700])
def test_long_lists_with_many_masks_and_rates(dev, count):
    """Every third tensor has a mask of its own, every one its own rate and every fifth decays."""
    from xsimgs_amd import optim

    sizes = [(1 + (i * 53) % 90, 1 + i % 7) if i % 11 else (0, 3) for i in range(count)]
    ptypes, gtypes = [TYPES[i % 3] for i in range(count)], [TYPES[(i // 3) % 3] for i in range(count)]
    before = _state(sizes, ptypes, gtypes, 9, dev)
    keeps = [torch.from_numpy(_keep(s[0], 0.4, i)) if i % 3 == 0 else torch.ones(s[0], dtype=torch.bool)
             for i, s in enumerate(sizes)]
    for i, (g, keep) in enumerate(zip(before[1], keeps)):
        g[~keep] = float("nan")
    masks = [_pack(k.numpy()).to(dev) if i % 3 == 0 else None for i, k in enumerate(keeps)]
    p, g, m, v = ([x.to(dev) for x in xs] for xs in before)
    kept = [_f64(x)[k] for x, k in zip(before[1], keeps)]
    norm = _norm64(kept, 2.0)
    total, each = optim.grad_norm(g, masks=masks, per_tensor=True)
    _close(total, norm, 2 * U)
    for i, x in enumerate(kept):
        _close(each[i], _norm64([x], 2.0), 2 * U, i)
    lr, decay = [1e-3 * (1 + i) / count for i in range(count)], [0.1 if i % 5 == 0 else 0.0 for i in range(count)]
    step = torch.full((1,), 3, dtype=torch.int64, device=dev)
    got = optim.adam_step_(p, g, m, v, step, lr=lr, betas=BETAS, eps=EPS, weight_decay=decay, max_norm=0.5 * norm,
                           masks=masks, skip_nonfinite=True)
    _close(got, norm, 2 * U)
    c = 0.5 * norm / (norm + 1e-6)
    _check_update((p, m, v), before, 4, lr, decay, c, keeps)
    _close(optim.clip_grads_(g, 0.5 * norm, masks=masks), norm, 2 * U)
    for x, old, keep in zip(g, before[1], keeps):
        off = (_f64(x)[keep] - c * _f64(old)[keep]).abs()
        assert bool((off <= (3 * U + 1.001 * HALF_ULP[x.dtype]) * c * _f64(old)[keep].abs() + 2 * SMALLEST[x.dtype]).all())
        assert bool(x.cpu()[~keep].isnan().all())


@pytest.mark.parametrize("row", [1, 2, 3, 4, 7, 8, 48, 127, 128, 129, 200, 1500])
@pytest.mark.parametrize("offset", [0, 1, 2, 4])
def test_rows_of_any_length_anywhere(dev, row, offset):
    """Masked tensors that start `offset` elements into a buffer; what lies around them stays."""
    from xsimgs_amd import optim

    n = 1 + 6000 // row if row < 1000 else 9
    kept = _keep(n, 0.3, row)
    kept[[0, -1]] = True, False
    keep = torch.from_numpy(kept)
    mask = _pack(kept).to(dev)
    for dtype in (torch.float32, torch.float16):
        before = _state([(n, row)], [dtype], [dtype], 17, dev)
        before[1][0][~keep] = float("inf")
        arenas = [torch.full((n * row + 8,), 77.0, dtype=x[0].dtype, device=dev) for x in before]
        p, g, m, v = ([a[offset:offset + n * row].view(n, row)] for a in arenas)
        for new, old in zip((p, g, m, v), before):
            new[0].copy_(old[0])
        norm = _norm64([_f64(before[1][0])[keep]], 2.0)
        _close(optim.grad_norm(g, masks=mask), norm, 2 * U)
        step = torch.full((1,), 20, dtype=torch.int64, device=dev)
        optim.adam_step_(p, g, m, v, step, lr=1e-2, betas=BETAS, eps=EPS, max_norm=0.5 * norm, masks=mask)
        c = 0.5 * norm / (norm + 1e-6)
        _check_update((p, m, v), before, 21, [1e-2], [0.0], c, [keep])
        optim.clip_grads_(g, 0.5 * norm, masks=mask)
        x, old = _f64(g[0]), _f64(before[1][0])
        off = (x[keep] - c * old[keep]).abs()
        assert bool((off <= (3 * U + 1.001 * HALF_ULP[dtype]) * c * old[keep].abs() + 2 * SMALLEST[dtype]).all())
        assert bool(torch.isinf(x[~keep]).all())
        for a in arenas:
            assert bool((a[:offset] == 77).all()) and bool((a[offset + n * row:] == 77).all())


def test_arrays_aligned_differently(dev):
    """The four arrays of a parameter each start elsewhere."""
    from xsimgs_amd import optim

    n = 5003
    before = _state([(n,)], [torch.float32], [torch.bfloat16], 3, dev)
    arenas = [torch.zeros(n + 8, dtype=x[0].dtype, device=dev) for x in before]
    p, g, m, v = ([a[o:o + n]] for a, o in zip(arenas, (0, 3, 1, 2)))
    for new, old in zip((p, g, m, v), before):
        new[0].copy_(old[0])
    step = torch.full((1,), 20, dtype=torch.int64, device=dev)
    optim.adam_step_(p, g, m, v, step, lr=1e-2, betas=BETAS, eps=EPS)
    _check_update((p, m, v), before, 21, [1e-2], [0.0], 1.0)


@pytest.mark.parametrize("count,size", [(1, 1), (16, 1024), (17, 1024), (64, 256), (65, 256), (64, 257), (51, 256), (24, 4)])
@pytest.mark.parametrize("clip", [True, False])
def test_between_small_and_ordinary_calls(dev, count, size, clip):
    from xsimgs_amd import optim

    sizes = [(size,)] * count
    before = _state(sizes, [TYPES[i % 3] for i in range(count)], [TYPES[(i + 1) % 3] for i in range(count)], 31, dev)
    p, g, m, v = ([x.to(dev) for x in xs] for xs in before)
    norm = _norm64([_f64(x) for x in before[1]], 2.0)
    total, each = optim.grad_norm(g, per_tensor=True)
    _close(total, norm, 2 * U)
    for i, x in enumerate(before[1]):
        _close(each[i], _norm64([_f64(x)], 2.0), 2 * U, i)
    step = torch.full((1,), 6, dtype=torch.int64, device=dev)
    got = optim.adam_step_(p, g, m, v, step, lr=1e-2, betas=BETAS, eps=EPS, max_norm=0.5 * norm if clip else None)
    assert (got is not None) == clip and int(step) == 7
    c = 0.5 * norm / (norm + 1e-6) if clip else 1.0
    _check_update((p, m, v), before, 7, [1e-2] * count, [0.0] * count, c)
    _close(optim.clip_grads_(g, 0.25 * norm), norm, 2 * U)
    c = 0.25 * norm / (norm + 1e-6)
    for x, old in zip(g, before[1]):
        off = (_f64(x) - c * _f64(old)).abs()
        assert bool((off <= (3 * U + 1.001 * HALF_ULP[x.dtype]) * c * _f64(old).abs() + 2 * SMALLEST[x.dtype]).all())


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("types", [(torch.float32, torch.float32), (torch.bfloat16, torch.float16)])
def test_update_of_more_than_the_caches_hold(dev, types, masked):
    """29 M elements of four arrays (over 256 MB) in a short-rowed and a long-rowed tensor, float64 on the GPU."""
    from xsimgs_amd import optim

    gen = torch.Generator(device=dev).manual_seed(2)
    n = 550_003
    shapes = [(n, 3), (n, 48), (n,)]

    def made(scale, dtype):
        return [(scale * torch.randn(s, generator=gen, device=dev)).to(dtype) for s in shapes]

    p, g, m = made(0.5, types[0]), made(1e-2, types[1]), made(1e-3, torch.float32)
    v = [x.square() for x in made(1e-2, torch.float32)]
    keep, masks = torch.ones(n, dtype=torch.bool, device=dev), None
    if masked:
        kept = _keep(n, 0.2, 4)
        keep, masks = torch.from_numpy(kept).to(dev), _pack(kept).to(dev)
        for x in g:
            x[~keep] = float("nan")
    before = [[x.clone() for x in xs] for xs in (p, g, m, v)]
    norm = math.sqrt(sum(float(x[keep].double().square().sum()) for x in g))
    step = torch.full((1,), 99, dtype=torch.int64, device=dev)
    got = optim.adam_step_(p, g, m, v, step, lr=1e-2, betas=BETAS, eps=EPS, max_norm=0.5 * norm, masks=masks)
    _close(got, norm, 2 * U)
    c = 0.5 * norm / (norm + 1e-6)
    for i in range(len(shapes)):
        p0, g0, m0, v0 = (xs[i][keep].double() for xs in before)
        p1, m1, v1 = _adam64(p0, g0, m0, v0, 100, 1e-2, 0.0, c)
        bounds = _adam_bounds(p0, g0, m0, v0, m1, v1, 100, 1e-2, c, types[0])
        for name, new, want, bound in zip("pmv", (p, m, v), (p1, m1, v1), bounds):
            off = (new[i][keep].double() - want).abs()
            assert bool((off <= bound).all()), (i, name, float((off / bound).max()))
        for new, old in ((p[i], before[0][i]), (m[i], before[2][i]), (v[i], before[3][i])):
            assert torch.equal(new[~keep], old[~keep])


@pytest.mark.parametrize("masked", [False, True])
def test_norm_and_clip_of_more_than_the_caches_hold(dev, masked):
    from xsimgs_amd import optim

    gen = torch.Generator(device=dev).manual_seed(5)
    n = 1_400_001
    g = [torch.randn(s, generator=gen, device=dev) for s in ((n, 3), (n, 48), (n,), (17,))]
    keep, masks = [torch.ones(x.shape[0], dtype=torch.bool, device=dev) for x in g], None
    if masked:
        kept = _keep(n, 0.2, 6)
        keep[:3] = [torch.from_numpy(kept).to(dev)] * 3
        masks = [_pack(kept).to(dev)] * 3 + [None]
        for x, k in zip(g, keep):
            x[~k] = float("inf")
    before = [x.clone() for x in g]
    each64 = [float(x[k].double().square().sum()) for x, k in zip(g, keep)]
    norm = math.sqrt(sum(each64))
    total, each = optim.grad_norm(g, masks=masks, per_tensor=True)
    _close(total, norm, 2 * U)
    for a, b in zip(each, each64):
        _close(a, math.sqrt(b), 2 * U)
    _close(optim.clip_grads_(g, 0.5 * norm, masks=masks), norm, 2 * U)
    c = 0.5 * norm / (norm + 1e-6)
    for x, old, k in zip(g, before, keep):
        off = (x[k].double() - c * old[k].double()).abs()
        assert bool((off <= 4 * U * c * old[k].double().abs()).all())
        assert torch.equal(x[~k], old[~k])


@pytest.mark.parametrize("count", [3, 200])
def test_captured_lists(dev, count):
    """A captured update of a short and of a long list, replayed on new gradients with other work between."""
    from xsimgs_amd import optim

    sizes = [(300 + i, 3) for i in range(count)]
    p, g, m, v = ([x.to(dev) for x in xs] for xs in _state(sizes, [torch.float32] * count, [torch.float32] * count, 5,
                                                             dev, fresh=True))
    step = torch.zeros(1, dtype=torch.int64, device=dev)
    eager = [[x.clone() for x in xs] for xs in (p, g, m, v)] + [step.clone()]
    fresh = [x.clone() for x in g]
    run = lambda p, g, m, v, step: optim.adam_step_(p, g, m, v, step, lr=1e-2, max_norm=0.1, skip_nonfinite=True)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run(*[[x.clone() for x in xs] for xs in (p, g, m, v)], step.clone())
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = run(p, g, m, v, step)
    for i in range(4):
        for x, y, f in zip(g, eager[1], fresh):
            x.copy_(f * (1 - 2 * i))
            y.copy_(f * (1 - 2 * i))
        if i == 2:   # a step that is left out, in the graph and beside it
            g[count // 2][0] = math.inf
            eager[1][count // 2][0] = math.inf
        graph.replay()
        torch.cuda.synchronize()
        want = run(*eager)
        optim.grad_norm([torch.randn(5000, device=dev) for _ in range(120)])
        torch.cuda.synchronize()
        assert torch.equal(norm, want), i
        for xs, ys in zip((p, m, v), (eager[0], eager[2], eager[3])):
            assert all(torch.equal(x, y) for x, y in zip(xs, ys)), i
        assert int(step) == int(eager[4]) == (i + 1 if i < 2 else i)


def test_results_are_the_same_bits_each_time(dev):
    from xsimgs_amd import optim

    g = torch.Generator(device=dev).manual_seed(1)
    for sizes in ([(40,), (3,)], [(90_000, 3), (90_000, 48)], [(1_500_000, 48)], [(200 + i, 3) for i in range(300)]):
        xs = [torch.randn(s, generator=g, device=dev) for s in sizes]
        first = [optim.grad_norm(xs, k, per_tensor=True) for k in (1.0, 2.0)]
        for _ in range(3):
            again = [optim.grad_norm(xs, k, per_tensor=True) for k in (1.0, 2.0)]
            assert all(torch.equal(a, b) for x, y in zip(first, again) for a, b in zip(x, y))
