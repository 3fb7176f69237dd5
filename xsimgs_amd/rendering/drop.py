"""Dropout whose draws come from a counter-based generator: a draw is a function of its number, the seed and the
stream, so the backward draws again and no mask is stored. An extension of this build.

``seed``: an int in [0, 2^63), another for each step; or an int64 tensor of one value on the GPU, which the kernels
read (a captured graph then draws anew on each replay if the value is changed in between; not between a forward
and its backward, which autograd refuses; as with any operator, a backward is captured while no eager graph of the same leaves
lives). ``stream``: a number in [0, 2^31), another for each place that
draws under one seed. Probabilities count in steps of 2^-32; what is kept is divided by the share that is kept."""
import torch

from .. import _C


def seed_arguments(seed, drop: float = 1.0, stream: int = 0):
    """(the number, the tensor or None). None is refused where something is dropped: a seed that is always the same drops
    the same places in every step."""
    if seed is None and not (0 < drop <= 1 and 0 <= stream < 1 << 31):
        return 0, None         # nothing is drawn, or the probability or the stream is refused behind this
    if isinstance(seed, torch.Tensor):
        return 0, seed
    if isinstance(seed, bool) or not isinstance(seed, int) or not 0 <= seed < 1 << 63:
        raise ValueError("seed must be an int in [0, 2^63) or an int64 tensor of one value, another for each step, "
                         f"not {seed!r}")
    return seed, None


def dropout(x: torch.Tensor, p: float, seed, *, stream: int = 0, shared: int = 0) -> torch.Tensor:
    """``x`` (float32, bfloat16 or float16 on the GPU) with elements zeroed with probability ``p`` and the others
    divided by the share kept; zeros whatever ``x`` holds there. ``shared``: so many trailing dimensions share one
    draw (1 drops whole rows of the last dimension; 2 a Gaussian's SH coefficients of ``[N, K, 3]``). A ``p`` of 0
    gives ``x`` itself."""
    if not 0 <= shared <= x.dim():
        raise ValueError(f"shared must lie in [0, {x.dim()}] for a tensor of {x.dim()} dimensions, not {shared}")
    row = 1
    for n in x.shape[x.dim() - shared:]:
        row *= n
    seed, seed_at = seed_arguments(seed)
    if p == 0:
        return x
    return _C.dropout(x, float(p), seed, seed_at, stream, max(row, 1))


def drop_mask(n: int, drop: float, seed, *, stream: int = 0, device=None) -> torch.Tensor:
    """Which of ``n`` Gaussians ``activate_gaussians(..., drop, seed, stream)`` keeps, as a packed mask (bit i % 32 of
    word i // 32), as ``ut_gs_tiling``'s ``packed_particle_mask`` and the optimizer's ``masks`` take it."""
    seed, seed_at = seed_arguments(seed)
    if device is None:
        device = seed_at.device if seed_at is not None else "cuda"
    return _C.drop_mask(n, float(drop), seed, seed_at, stream, torch.device(device))
