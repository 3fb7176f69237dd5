"""Adam over many tensors in a few launches: decoupled weight decay, clipping by the global norm fused in (the
factor stays on the GPU and the gradients are not rewritten), and the renderer's packed visibility mask, under
which Gaussians out of view keep their parameters and moments. Moments are float32 whatever the parameter's
type; the step counter lives on the GPU, so a step can be captured in a graph and replayed (with the learning
rates it was captured with, and not a first step, which makes moments and counter)."""
import torch

from .. import _C
from .clip import listed_masks


def _rates(value):
    return value if isinstance(value, (int, float)) else list(value)


def _number(value, name) -> float:
    if isinstance(value, torch.Tensor) and value.device.type != "cpu":
        raise ValueError(f"{name} must be a number or a tensor on the CPU: one on {value.device} would be read back")
    return float(value)


def adam_step_(params, grads, exp_avgs, exp_avg_sqs, step, *, lr, betas=(0.9, 0.999), eps: float = 1e-8,
               weight_decay=0.0, max_norm: float | None = None, norm_type: float = 2.0,
               skip_nonfinite: bool = False, masks=None):
    """One update in place; with t = step + 1 and c = min(1, max_norm / (norm of all grads + 1e-6)) (1 without
    ``max_norm``):

        m += (1 - beta1) (c g - m);  v = beta2 v + (1 - beta2) (c g)^2
        p = p (1 - lr weight_decay) - lr / (1 - beta1^t) m / (sqrt(v) / sqrt(1 - beta2^t) + eps)

    ``step``: one int64 value on the GPU, which then holds t. ``lr`` and ``weight_decay``: a number, or one per
    tensor (not on the GPU: they would be read back). ``masks`` as in ``grad_norm`` (rows out of the mask do not change, and do not count in the norm).
    ``skip_nonfinite``: a norm that is not finite (as returned, in float32) leaves everything as it is, ``step``
    too. Returns the norm before clipping (with ``max_norm`` or ``skip_nonfinite``, else None). Parameters and
    gradients are float32, bfloat16 or float16; moments are float32 tensors of their parameter's sizes and strides."""
    params = list(params)
    return _C.adam_step_(params, list(grads), list(exp_avgs), list(exp_avg_sqs), step, _rates(lr),
                         _rates(weight_decay), float(betas[0]), float(betas[1]), float(eps),
                         None if max_norm is None else float(max_norm), float(norm_type), bool(skip_nonfinite),
                         listed_masks(masks, len(params)))


_OPTIONS = ("betas", "eps", "max_norm", "norm_type", "skip_nonfinite")   # of a whole optimizer


class Adam(torch.optim.Optimizer):
    """Adam over ``adam_step_``. Groups carry their own ``lr`` and ``weight_decay``; betas, eps, ``max_norm``,
    ``norm_type`` and ``skip_nonfinite`` hold for the whole optimizer, whose tensors are one list with one norm
    and one step counter: a parameter without a gradient sits a step out, and bias correction goes by the
    optimizer's count, not the parameter's as in torch.optim.Adam (one that joins late starts with corrections
    near 1, so its first step is up to (1 - beta1) / sqrt(1 - beta2) rates long; an optimizer of its own starts
    it as a new one). ``grad_norm`` is the last step's norm before clipping, or None."""

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-15, weight_decay: float = 0.0, *,
                 max_norm: float | None = None, norm_type: float = 2.0, skip_nonfinite: bool = False):
        if _number(lr, "lr") < 0.0 or eps < 0.0 or _number(weight_decay, "weight_decay") < 0.0 or not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError("lr, eps and weight_decay must not be negative, betas must lie in [0, 1)")
        super().__init__(params, dict(lr=lr, weight_decay=weight_decay))
        self.betas, self.eps = tuple(betas), eps
        self.max_norm, self.norm_type, self.skip_nonfinite = max_norm, norm_type, skip_nonfinite
        self.step_count = None   # int64 [1] on the parameters' GPU, from the first step on
        self.grad_norm = None

    def __getstate__(self):
        """What a copy or a pickle takes along: the base class knows its own attributes only."""
        return dict(super().__getstate__(), **{k: getattr(self, k) for k in (*_OPTIONS, "step_count", "grad_norm")})

    def add_param_group(self, param_group):
        if shared := set(_OPTIONS) & set(param_group):
            raise ValueError(f"{sorted(shared)} hold for the whole optimizer; a group may set lr and weight_decay")
        super().add_param_group(param_group)

    @torch.no_grad()
    def step(self, closure=None, *, masks=None):
        """``masks``: a dict from parameters to their packed masks, for those that have one."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        params, lr, decay = [], [], []
        for group in self.param_groups:
            rate, share = _number(group["lr"], "lr"), _number(group["weight_decay"], "weight_decay")
            for p in group["params"]:
                if p.grad is not None:
                    params.append(p)
                    lr.append(rate)
                    decay.append(share)
        self.grad_norm = None
        if not params:
            return loss
        for p in params:
            if not self.state[p]:
                self.state[p]["exp_avg"] = torch.zeros_like(p, dtype=torch.float32)
                self.state[p]["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.float32)
        if self.step_count is None:
            self.step_count = torch.zeros(1, dtype=torch.int64, device=params[0].device)
        self.grad_norm = adam_step_(params, [p.grad for p in params], [self.state[p]["exp_avg"] for p in params],
                                    [self.state[p]["exp_avg_sq"] for p in params], self.step_count, lr=lr,
                                    betas=self.betas, eps=self.eps, weight_decay=decay, max_norm=self.max_norm,
                                    norm_type=self.norm_type, skip_nonfinite=self.skip_nonfinite,
                                    masks=None if masks is None else [masks.get(p) for p in params])
        return loss

    def state_dict(self):
        """The base class's, with the step counter and the options that hold for the whole optimizer. The counter
        is the optimizer's own tensor, as the moments are: copy the dict to keep it over further steps."""
        return dict(super().state_dict(), step=self.step_count, options={k: getattr(self, k) for k in _OPTIONS})

    def load_state_dict(self, state_dict):
        """Options are taken over as the groups' rates are (a dict without any leaves those of this optimizer).
        The moments come back in float32 (the base class would give them their parameter's type). Another
        optimizer's dict is refused: torch.optim.Adam's, say, counts each parameter's steps and holds options
        that mean something else here. Its moments can come in a dict of this form, where all its counts agree."""
        moments = {"exp_avg", "exp_avg_sq"}
        states = [set(v) for v in state_dict["state"].values() if v]
        if "step" not in state_dict or any(s != moments for s in states) or (states and state_dict["step"] is None):
            raise ValueError("not a state dict of this optimizer: it has exp_avg and exp_avg_sq for each parameter and "
                             "one step counter (step) beside them")
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(ids, params):
            if any(v.shape != p.shape for v in state_dict["state"].get(i, {}).values()):
                raise ValueError(f"the moments of parameter {i} are not of its sizes {tuple(p.shape)}")
        super().load_state_dict({k: v for k, v in state_dict.items() if k not in ("step", "options")})
        for k, v in state_dict.get("options", {}).items():
            setattr(self, k, tuple(v) if k == "betas" else v)
        for i, p in zip(ids, params):
            for k, v in state_dict["state"].get(i, {}).items():
                self.state[p][k] = torch.empty_like(p, dtype=torch.float32).copy_(v)
        step = state_dict.get("step")
        self.step_count = None if step is None else step.detach().clone().to(params[0].device)
