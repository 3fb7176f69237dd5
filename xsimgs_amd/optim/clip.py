"""The global norm of a list of tensors and clipping by it, each in a few launches whatever the number of
tensors, with nothing read back to the host. Tensors are float32, bfloat16 or float16 on one GPU, in any mix
of sizes (empty ones too) and strides; sums are held in 64 bits.

``masks``: None, one packed mask for every tensor, or a sequence with one (or None) per tensor. A packed mask
(``packed_visibility_mask``, ``packed_mask_from_instances``: bit i % 32 of word i // 32) covers the rows of
its tensor's first dimension and has the words that these need, no more (one word fits any 1 to 32 rows: below
that a mask of other rows cannot be told); rows whose bit is 0 are neither read nor written, whatever they
hold. (SH coefficients in the ``[3, K, N]`` layout go in as 3 K tensors, the rows of
their ``view(3 * K, N)``, each under the mask.)"""
import torch

from .. import _C


def listed_masks(masks, n: int) -> list:
    """One optional mask per tensor, or an empty list without any."""
    if masks is None:
        return []
    if isinstance(masks, torch.Tensor):
        return [masks] * n
    masks = list(masks)
    if len(masks) != n:
        raise ValueError(f"masks must hold one entry per tensor: {len(masks)} for {n}")
    return masks if any(m is not None for m in masks) else []


def grad_norm(tensors, norm_type: float = 2.0, *, masks=None, per_tensor: bool = False):
    """The norm (2, 1 or inf) over all elements of ``tensors`` as a float32 tensor of no dimensions; with
    ``per_tensor`` also each tensor's own, ``[len(tensors)]``. No elements: 0. NaNs make it NaN."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    total, each = _C.grad_norm(tensors, float(norm_type), listed_masks(masks, len(tensors)), bool(per_tensor))
    return (total, each) if per_tensor else total


def clip_grads_(tensors, max_norm: float, norm_type: float = 2.0, *, eps: float = 1e-6, masks=None) -> torch.Tensor:
    """Scales ``tensors`` in place by min(1, max_norm / (norm + eps)) and returns the norm before. Where the
    factor is 1 nothing is written; a norm that is not finite acts as in torch.nn.utils.clip_grad_norm_
    (NaN spreads, infinity zeros the finite values). A tensor that is not dense (or, under a mask, not contiguous)
    is worked on in a dense copy, which reads all of it; what changed is written back. No two tensors may share an element; strided ones may lie
    between each other's (should it take too long to tell, they are refused)."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    return _C.clip_grads_(tensors, float(max_norm), float(norm_type), float(eps), listed_masks(masks, len(tensors)))


def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False, *,
                    masks=None) -> torch.Tensor:
    """torch.nn.utils.clip_grad_norm_ over these kernels: clips the gradients of ``parameters`` (those that
    have one) and returns their norm before. ``masks`` as in the module's text, one per parameter.
    ``error_if_nonfinite`` reads the norm back before anything is scaled."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    masks = listed_masks(masks, len(parameters))
    kept = [i for i, p in enumerate(parameters) if p.grad is not None]
    grads = [parameters[i].grad for i in kept]
    masks = [masks[i] for i in kept] if masks else None
    if not grads:
        return torch.zeros((), device=parameters[0].device if parameters else None)
    if error_if_nonfinite and not bool(torch.isfinite(grad_norm(grads, norm_type, masks=masks))):
        raise RuntimeError(f"the norm of order {float(norm_type)} of the gradients is not finite, so they cannot be "
                           "clipped; pass error_if_nonfinite=False to scale them by it all the same")
    return clip_grads_(grads, max_norm, norm_type, masks=masks)
