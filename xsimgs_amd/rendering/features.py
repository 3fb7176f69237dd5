"""Group norm with an activation and dropout over rendered feature images, channels last as the compositor writes
them: what a network that decodes them starts each of its blocks with. An extension of this build."""
import torch

from .. import _C
from .drop import seed_arguments

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}


def group_norm_act(x: torch.Tensor, groups: int, weight=None, bias=None, *, act: str = "silu", eps: float = 1e-5,
                   mask=None, drop: float = 0.0, seed=None, stream: int = 0) -> torch.Tensor:
    """``drop(act((x - mean) / sqrt(variance + eps) * weight + bias))`` over each sample and each group of
    consecutive channels of ``x`` ``[batch, ..., channels]`` (float32, bfloat16 or float16 on the GPU; up to 4096
    channels, which ``groups`` divides; one camera's ``[H, W, ch]`` goes in as ``x[None]``). Sums are held in 32 and 64
    bits, the result is rounded once.

    ``weight``, ``bias``: one value per channel, float32 or of x's type, or None. ``act``: none, relu, silu or gelu (by
    the error function). ``mask``: ``[batch, ...]``, bool; pixels out of it are not read, do not count, and give 0 and
    no gradient (a sample without any gives zeros). ``drop``, ``seed``, ``stream``: the draws of ``dropout`` on the result; a
    ``seed`` is needed where ``drop`` is not 0, another for each step."""
    if act not in ACTIVATIONS:
        raise ValueError(f"act must be one of {', '.join(ACTIVATIONS)}, not {act!r}")
    seed, seed_at = seed_arguments(seed, drop, stream)
    return _C.group_norm_act(x, groups, weight, bias, ACTIVATIONS[act], eps, mask, drop, seed, seed_at, stream)


class FeatureNorm(torch.nn.Module):
    """``group_norm_act`` with its weight and bias, for ``frame.prepare(..., head=)`` and networks behind the
    compositor. Dropout acts in training mode only and takes the call's ``seed``; ``stream`` tells modules apart
    that share one (0 is the frame's Gaussians')."""

    def __init__(self, groups: int, channels: int, act: str = "silu", eps: float = 1e-5, drop: float = 0.0, *,
                 stream: int = 1, device=None, dtype=None):
        super().__init__()
        if act not in ACTIVATIONS or groups < 1 or channels % groups or not 0.0 <= drop <= 1.0:
            raise ValueError(f"FeatureNorm takes an activation ({', '.join(ACTIVATIONS)}), groups that divide the channels "
                             "and a drop probability in [0, 1]")
        self.groups, self.act, self.eps, self.drop, self.stream = groups, act, eps, drop, stream
        self.weight = torch.nn.Parameter(torch.ones(channels, device=device, dtype=dtype))
        self.bias = torch.nn.Parameter(torch.zeros(channels, device=device, dtype=dtype))

    def forward(self, x, mask=None, seed=None):
        drop = self.drop if self.training else 0.0
        if drop > 0.0 and seed is None:
            raise ValueError("a FeatureNorm that drops takes another seed in each training step")
        return group_norm_act(x, self.groups, self.weight, self.bias, act=self.act, eps=self.eps, mask=mask, drop=drop,
                              seed=seed, stream=self.stream)

    def extra_repr(self):
        return f"{self.groups}, {self.weight.numel()}, act={self.act}, eps={self.eps}, drop={self.drop}"
