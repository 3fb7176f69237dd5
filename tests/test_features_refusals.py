"""What dropout and the feature norm refuse before anything runs: calls that would be answered wrongly in silence."""
import pytest
import torch

from xsimgs_amd import rendering


def test_what_drops_needs_a_seed():
    """Without one the same would be dropped in every step; where nothing is, none is needed."""
    from xsimgs_amd import frame

    x, a, o = torch.zeros(2, 3, 4), torch.zeros(4, 3), torch.zeros(4)
    st = frame.FrameState(None, torch.device("cpu"), torch.zeros(4, 3), a, torch.zeros(4, 4), o, None, a)
    for call in (lambda: rendering.group_norm_act(x, 1, drop=0.5), lambda: rendering.activate_gaussians(a, o, drop=0.5),
                 lambda: rendering.group_norm_act(x, 1, drop=0.5, seed=None), lambda: frame._drawn(st, 0.5, None)):
        with pytest.raises(ValueError, match="seed"):
            call()
    for call in (lambda: rendering.group_norm_act(x, 1), lambda: rendering.activate_gaussians(a, o),
                 lambda: frame._drawn(st, 0.0, None)):
        with pytest.raises(RuntimeError):      # past the seed: tensors on the CPU
            call()
