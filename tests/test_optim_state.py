"""What ``optim.Adam`` keeps over copies, pickles and checkpoints, and what it refuses to take up. CPU only: the
native update is replaced by float64 arithmetic on the same arguments."""
import copy
import io
import pickle

import pytest
import torch

from xsimgs_amd import optim

OPTIONS = dict(betas=(0.8, 0.95), eps=1e-7, max_norm=0.5, norm_type=1.0, skip_nonfinite=True)


@pytest.fixture(autouse=True)
def calls(monkeypatch):
    """The arguments of each update, which is computed as adam_step_ documents it."""
    seen = []

    def update(params, grads, exp_avgs, exp_avg_sqs, step, *, lr, betas, eps, weight_decay, max_norm, norm_type,
               skip_nonfinite, masks):
        seen.append(dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, max_norm=max_norm, norm_type=norm_type,
                         skip_nonfinite=skip_nonfinite, masks=masks))
        norm = torch.linalg.vector_norm(torch.cat([g.double().reshape(-1) for g in grads]), norm_type)
        c = 1.0 if max_norm is None else min(1.0, max_norm / (float(norm) + 1e-6))
        step += 1
        t = int(step)
        for p, g, m, v, rate, decay in zip(params, grads, exp_avgs, exp_avg_sqs, lr, weight_decay):
            assert m.dtype == v.dtype == torch.float32
            g = c * g.double()
            m.copy_(betas[0] * m.double() + (1 - betas[0]) * g)
            v.copy_(betas[1] * v.double() + (1 - betas[1]) * g * g)
            root = (v.double() / (1 - betas[1] ** t)).sqrt() + eps
            p.copy_(p.double() * (1 - rate * decay) - rate / (1 - betas[0] ** t) * m.double() / root)
        return norm.float() if max_norm is not None or skip_nonfinite else None

    monkeypatch.setattr("xsimgs_amd.optim.adam.adam_step_", update)
    return seen


def _params():
    g = torch.Generator().manual_seed(5)
    return [torch.nn.Parameter(torch.randn(s, generator=g)) for s in ((6, 3), (4,))] + \
           [torch.nn.Parameter(torch.randn(7, generator=g).bfloat16())]


def _optimizer(ps, **options):
    return optim.Adam([dict(params=ps[:1], lr=1e-2, name="means"), dict(params=ps[1:], weight_decay=0.1)], lr=3e-3,
                      **options)


def _run(opt, ts):
    ps = [p for group in opt.param_groups for p in group["params"]]
    for t in ts:
        for i, p in enumerate(ps):
            p.grad = torch.randn(p.shape, generator=torch.Generator().manual_seed(10 * t + i)).to(p.dtype)
        opt.step()
    return [p.detach().clone() for p in ps]


@pytest.mark.parametrize("steps", [0, 2])
@pytest.mark.parametrize("how", ["copy", "pickle", "save"])
def test_copies_go_on_alike(calls, how, steps):
    opt = _optimizer(_params(), **OPTIONS)
    _run(opt, range(steps))
    if how == "copy":
        other = copy.deepcopy(opt)
    elif how == "pickle":
        other = pickle.loads(pickle.dumps(opt))
    else:
        torch.save(opt, file := io.BytesIO())
        file.seek(0)
        other = torch.load(file, weights_only=False)
    assert {k: getattr(other, k) for k in OPTIONS} == OPTIONS
    assert (other.step_count is None) == (steps == 0) and (steps == 0 or int(other.step_count) == steps)
    want = _run(opt, range(steps, steps + 2))
    assert steps == 0 or int(other.step_count) == steps   # its own counter, not the first one's
    got = _run(other, range(steps, steps + 2))
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and int(other.step_count) == int(opt.step_count) == steps + 2
    assert calls[-1] == calls[-3] and torch.equal(other.grad_norm, opt.grad_norm)


@pytest.mark.parametrize("through_file", [False, True])
def test_a_state_dict_brings_the_options(calls, through_file):
    """A resumed run goes on with what was saved, whatever the optimizer was built with."""
    opt = _optimizer(_params(), **OPTIONS)
    _run(opt, range(2))
    saved = opt.state_dict()
    if through_file:
        torch.save(saved, file := io.BytesIO())
        file.seek(0)
        saved = torch.load(file, weights_only=True)
    kept = copy.deepcopy(saved)
    other = _optimizer([torch.nn.Parameter(p.detach().clone()) for g in opt.param_groups for p in g["params"]],
                       betas=(0.5, 0.5), eps=1e-3)
    other.load_state_dict(saved)
    assert {k: getattr(other, k) for k in OPTIONS} == OPTIONS
    got = _run(other, [2, 3])
    for i, state in saved["state"].items():   # the other optimizer's steps write nothing of what was saved
        assert all(torch.equal(state[k], kept["state"][i][k]) for k in state)
    assert int(saved["step"]) == 2
    assert all(torch.equal(a, b) for a, b in zip(got, _run(opt, [2, 3]))) and calls[-1] == calls[-3]


def test_a_state_dict_without_options_leaves_them():
    opt = _optimizer(_params(), **OPTIONS)
    _run(opt, [0])
    other = _optimizer(_params(), betas=(0.5, 0.5), max_norm=2.0)
    other.load_state_dict({k: v for k, v in opt.state_dict().items() if k != "options"})
    assert other.betas == (0.5, 0.5) and other.max_norm == 2.0 and not other.skip_nonfinite and int(other.step_count) == 1


def test_a_state_dict_is_of_one_time():
    """Moments and counter in a dict belong together, also after further steps of its optimizer."""
    opt = _optimizer(_params())
    _run(opt, range(2))
    saved = opt.state_dict()
    now = _run(opt, [2])
    params = [torch.nn.Parameter(p.clone()) for p in now]
    other = _optimizer(params)
    other.load_state_dict(saved)
    assert int(other.step_count) == int(opt.step_count) == 3
    assert all(torch.equal(a, b) for a, b in zip(_run(other, [3]), _run(opt, [3])))


@pytest.mark.parametrize("steps", [0, 2])
@pytest.mark.parametrize("other", [torch.optim.Adam, torch.optim.AdamW, torch.optim.SGD])
def test_another_optimizers_state_dict_is_refused(other, steps):
    """Warm moments with a counter that starts again would be corrected as a first step's; nothing changes."""
    ps = _params()
    foreign = other([dict(params=ps[:1]), dict(params=ps[1:])], lr=0.1)
    _run(foreign, range(steps))
    opt = _optimizer(_params())
    _run(opt, [0])
    before = copy.deepcopy(opt.state_dict())
    with pytest.raises(ValueError, match="state dict of this optimizer"):
        opt.load_state_dict(foreign.state_dict())
    after = opt.state_dict()
    assert after["param_groups"] == before["param_groups"] and int(after["step"]) == 1
    for i, state in before["state"].items():
        assert state.keys() == after["state"][i].keys()
        assert all(torch.equal(state[k], after["state"][i][k]) for k in state)
    if other is torch.optim.Adam and steps:   # in this optimizer's form its moments and count go on
        theirs = foreign.state_dict()
        opt.load_state_dict(dict(before, step=torch.tensor([steps]), state={
            i: {k: v[k] for k in ("exp_avg", "exp_avg_sq")} for i, v in theirs["state"].items()}))
        assert int(opt.step_count) == steps
        first = opt.param_groups[0]["params"][0]
        assert torch.equal(opt.state[first]["exp_avg"], theirs["state"][0]["exp_avg"])


def test_a_state_dict_with_a_part_missing_is_refused():
    opt = _optimizer(_params())
    _run(opt, [0])
    whole = opt.state_dict()
    for part in (dict(whole, step=None), {k: v for k, v in whole.items() if k != "step"},
                 dict(whole, state={0: dict(exp_avg=torch.zeros(6, 3))})):
        with pytest.raises(ValueError, match="state dict of this optimizer"):
            _optimizer(_params()).load_state_dict(part)
    narrow = copy.deepcopy(whole)
    narrow["state"][0]["exp_avg"] = narrow["state"][0]["exp_avg"][:1]   # would fit by repetition
    with pytest.raises(ValueError, match="not of its sizes"):
        opt.load_state_dict(narrow)
    fresh = _optimizer(_params())
    fresh.load_state_dict(_optimizer(_params()).state_dict())   # before a first step there is none of it
    assert fresh.step_count is None and not fresh.state


@pytest.mark.parametrize("name", ["lr", "weight_decay"])
def test_rates_on_another_device_are_refused(calls, name):
    """Reading one back would wait for the GPU in every step. (A device without memory stands for the GPU.)"""
    far, near = torch.empty((), device="meta"), torch.tensor(0.25)
    ps = _params()
    with pytest.raises(ValueError, match=f"{name} must be a number"):
        optim.Adam(ps, **{name: far})
    opt = _optimizer(ps)
    opt.param_groups[1][name] = far
    with pytest.raises(ValueError, match=f"{name} must be a number"):
        _run(opt, [0])
    assert not calls and not opt.state
    opt.param_groups[1][name] = near
    _run(opt, [0])
    assert calls[0][name] == [opt.param_groups[0][name], 0.25, 0.25]
    opt = optim.Adam(ps, **{name: near})   # a tensor that its owner changes
    near.fill_(0.5)
    _run(opt, [0])
    assert calls[1][name] == [0.5] * 3
    x = torch.ones(4)
    from xsimgs_amd import _C
    for value in (far, [far]):
        args = dict(lr=1e-3, weight_decay=0.0, beta1=0.9, beta2=0.99, eps=1e-8, max_norm=None, norm_type=2.0,
                    skip_nonfinite=False, masks=[])
        with pytest.raises(ValueError, match=f"{name} must be a number"):
            _C.adam_step_([x], [x], [x], [x], torch.zeros(1, dtype=torch.int64), **dict(args, **{name: value}))
