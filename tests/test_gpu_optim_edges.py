"""The training step's operators and optimizer at the edges of what they take."""
import math

import pytest
import torch

from tests.test_gpu_optim import _f64, _norm64

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
