"""The training step's operators and optimizer at the edges of what they take."""
import math

import pytest
import torch

from tests.test_gpu_optim import U, _check_update, _close, _f64, _norm64, _pack, _state

pytestmark = pytest.mark.gpu


# the kinds of call: one workgroup, terms in the update's own workgroups, a table, terms in a launch of their own
LISTS = {"small": [(7,)], "ordinary": [(300, 3)] * 30, "long": [(11, 3)] * 120, "many chunks": [(17_000_000,)]}


@pytest.mark.parametrize("kind", [1.0, 2.0])
@pytest.mark.parametrize("lists", LISTS)
def test_norm_that_float32_cannot_hold_skips_the_step(dev, lists, kind):
    """Finite gradients whose norm is above the largest float32: the caller gets inf, and nothing moves."""
    from xsimgs_amd import optim

    p, g, m, v = ([torch.full(s, x, device=dev) for s in LISTS[lists]] for x in (0.5, 0.0, 0.25, 0.125))
    g[0].view(-1)[:2] = 3e38
    g[-1].view(-1)[-2:] = -3e38
    assert math.isfinite(_norm64([_f64(x) for x in g], kind))
    step = torch.full((1,), 4, dtype=torch.int64, device=dev)
    for limit in (None, 1.0):
        norm = optim.adam_step_(p, g, m, v, step, lr=1e-2, max_norm=limit, norm_type=kind, skip_nonfinite=True)
        assert math.isinf(float(norm)) and int(step) == 4
        for xs, old in ((p, 0.5), (m, 0.25), (v, 0.125)):
            assert all(bool((x == old).all()) for x in xs)
    # the largest magnitude is a float32 and finite: this step is taken
    norm = optim.adam_step_(p, g, m, v, step, lr=1e-2, max_norm=1.0, norm_type=math.inf, skip_nonfinite=True)
    assert float(norm) == float(torch.tensor(3e38)) and int(step) == 5
    assert not bool((m[0] == 0.25).any())


def test_masks_of_another_size_are_refused(dev):
    """A mask with words to spare is another tensor's, or another dimension's; nothing is written."""
    from xsimgs_amd import optim

    n = 100
    whole = _pack(torch.arange(n).numpy() % 2 == 0).to(dev)
    sh = torch.ones(3, 4, n, device=dev)   # the layout whose rows are channels
    for x, mask in ((sh, whole), (torch.ones(96, 3, device=dev), whole), (torch.ones(97, 3, device=dev), whole[:3])):
        param = torch.nn.Parameter(x.clone())
        param.grad = x.clone()
        z = lambda: torch.zeros_like(x)
        for call in (lambda: optim.grad_norm([x], masks=mask), lambda: optim.clip_grads_([x], 0.1, masks=mask),
                     lambda: optim.adam_step_([x], [z()], [z()], [z()], torch.zeros(1, dtype=torch.int64, device=dev),
                                              lr=1.0, masks=[mask]),
                     lambda: optim.Adam([param], lr=1.0).step(masks={param: mask})):
            with pytest.raises(RuntimeError, match="size mismatch"):
                call()
        assert bool((x == 1).all()) and bool((param == 1).all())


@pytest.mark.parametrize("n", [5, 1003])
def test_sh_of_the_second_layout_by_rows(dev, n):
    """[3, K, N] coefficients under the Gaussians' mask, as 3 K tensors of N."""
    from xsimgs_amd import optim

    rows = 3 * 16
    keep = torch.rand(n, generator=torch.Generator().manual_seed(3)) < 0.4
    before = _state([(n,)] * rows, [torch.float32] * rows, [torch.float32] * rows, 90, dev)
    for x in before[1]:
        x[~keep] = float("nan")
    whole = [torch.stack(xs).view(3, 16, n).to(dev) for xs in before]
    p, g, m, v = (list(x.view(rows, n)) for x in whole)
    norm = _norm64([_f64(x)[keep] for x in before[1]], 2.0)
    step = torch.full((1,), 11, dtype=torch.int64, device=dev)
    got = optim.adam_step_(p, g, m, v, step, lr=1e-2, eps=1e-15, max_norm=0.5 * norm, masks=_pack(keep.numpy()).to(dev))
    _close(got, norm, 2 * U)
    _check_update((p, m, v), before, 12, [1e-2] * rows, [0.0] * rows, 0.5 * norm / (norm + 1e-6), [keep] * rows)
