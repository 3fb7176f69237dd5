"""What dropout and the feature norm refuse before anything runs: calls that would be answered wrongly in silence."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from xsimgs_amd import rendering


CALLS = dict(dropout=lambda x: rendering.dropout(x, 0.5, 1),
             group_norm_act=lambda x: rendering.group_norm_act(x, 1),
             weight=lambda x: rendering.group_norm_act(torch.zeros(2, 3, 4), 1, x[0, 0]),
             bias=lambda x: rendering.group_norm_act(torch.zeros(2, 3, 4), 1, None, x[0, 0]),
             scales=lambda x: rendering.activate_gaussians(x[0, :, :3], torch.zeros(3), drop=0.5, seed=1)[0],
             logits=lambda x: rendering.activate_gaussians(torch.zeros(3, 3), x[0, :, 0], drop=0.5, seed=1)[1])


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_is_refused(name, requires_grad):
    """A tangent would be lost: the result would look like a constant."""
    with fwd.dual_level():
        x = fwd.make_dual(torch.randn(2, 3, 4), torch.randn(2, 3, 4))
        if requires_grad:
            x = x * torch.ones((), requires_grad=True)
        with pytest.raises(RuntimeError, match="forward-mode"):
            CALLS[name](x)

@pytest.mark.parametrize("name", [*CALLS, "drop_mask"])
@pytest.mark.parametrize("requires_grad", [False, True])
def test_tracing_is_refused(name, requires_grad):
    """A trace would record the result's allocation alone, and replay memory that nothing has written."""
    call = CALLS.get(name, lambda x: x.sum() + rendering.drop_mask(8, 0.5, 1, device="cpu").sum())
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(call, (torch.randn(2, 3, 4, requires_grad=requires_grad),), check_trace=False)

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
