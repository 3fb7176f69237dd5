"""What a training step does behind the frame's backward: the global gradient norm over many tensors,
clipping by it, and the Adam update under the renderer's packed visibility mask. Extensions of this
build (the reference's trainer is outside its rendering library)."""
from .adam import Adam, adam_step_
from .clip import clip_grad_norm_, clip_grads_, grad_norm

__all__ = ["Adam", "adam_step_", "clip_grad_norm_", "clip_grads_", "grad_norm"]
