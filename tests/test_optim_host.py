"""The training step's entry points refuse wrong arguments on the host, before any launch. CPU only: the
pointers here are placeholders that no call reaches."""
import ctypes as C
import math
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "xsimgs_amd", "libxsimgs_hip.so")
FAKE, WS = 1 << 20, C.c_void_p(1 << 20)


class Grad(C.Structure):  # xsg_grad_tensor, field for field
    _fields_ = [("data", C.c_void_p), ("numel", C.c_int64), ("mask", C.c_void_p), ("rows", C.c_int64),
                ("dtype", C.c_int)]


class AdamTensor(C.Structure):  # xsg_adam_tensor, field for field
    _fields_ = [("param", C.c_void_p), ("grad", C.c_void_p), ("exp_avg", C.c_void_p), ("exp_avg_sq", C.c_void_p),
                ("numel", C.c_int64), ("mask", C.c_void_p), ("rows", C.c_int64), ("lr", C.c_double),
                ("weight_decay", C.c_double), ("param_dtype", C.c_int), ("grad_dtype", C.c_int)]


class AdamOptions(C.Structure):  # xsg_adam_options, field for field
    _fields_ = [("beta1", C.c_double), ("beta2", C.c_double), ("eps", C.c_double), ("clip", C.c_int),
                ("skip_nonfinite", C.c_int), ("norm", C.c_int), ("max_norm", C.c_double)]


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(LIB):
        pytest.fail(f"{LIB} is not built: run __graft_entry__.build()")
    import torch  # noqa: F401  (loads torch's HIP runtime first, as the package does)
    lib = C.CDLL(LIB)
    lib.xsg_last_error.restype = C.c_char_p
    for name in ("xsg_grad_norm_workspace_bytes", "xsg_adam_step_workspace_bytes"):
        getattr(lib, name).restype = C.c_size_t
    lib.xsg_clip_grads.argtypes = [C.c_void_p, C.c_int, C.c_int, C.c_double, C.c_double, C.c_void_p, C.c_void_p,
                                   C.c_void_p]
    return lib


def _grads(*changes):
    out = (Grad * max(1, len(changes)))()
    for x, change in zip(out, changes):
        for k, v in dict(dict(data=FAKE, numel=12, mask=None, rows=0, dtype=0), **change).items():
            setattr(x, k, v)
    return out


WRONG = [  # one tensor's change, and what the message says
    (dict(numel=-1), b"negative size"),
    (dict(data=None), b"is null"),
    (dict(dtype=3), b"unknown type"),
    (dict(dtype=-1), b"unknown type"),
    (dict(mask=FAKE, rows=5), b"cannot have 5 rows"),
    (dict(mask=FAKE, rows=0), b"cannot have 0 rows"),
    (dict(mask=FAKE, rows=-3), b"rows under its mask"),
    (dict(mask=FAKE, rows=1, numel=(1 << 30) + 1), b"more than"),
    (dict(numel=1 << 62), b"too many elements"),
]


@pytest.mark.parametrize("change,text", WRONG)
def test_tensor_lists_are_checked(lib, change, text):
    ts = _grads({}, change)
    assert lib.xsg_grad_norm(ts, 2, 2, WS, None, WS, None) == -1
    assert text in lib.xsg_last_error()
    assert lib.xsg_clip_grads(ts, 2, 2, 1.0, 1e-6, WS, WS, None) == -1
    assert text in lib.xsg_last_error()


def test_norm_and_clip_arguments(lib):
    ts = _grads({})
    calls = [((ts, 1, 7, WS, None, WS, None), b"unknown norm"), ((ts, 1, 2, None, None, WS, None), b"null output"),
             ((ts, 1, 2, WS, None, None, None), b"null output"), ((ts, -1, 2, WS, None, WS, None), b"negative list"),
             ((None, 1, 2, WS, None, WS, None), b"null or negative"),
             ((ts, 1, 2, WS, None, C.c_void_p(FAKE + 8), None), b"aligned")]
    for args, text in calls:
        assert lib.xsg_grad_norm(*args) == -1
        assert text in lib.xsg_last_error(), text
    for limit, eps in ((-1.0, 0.0), (math.nan, 0.0), (1.0, -1e-9), (1.0, math.nan)):
        assert lib.xsg_clip_grads(ts, 1, 2, limit, eps, WS, WS, None) == -1
        assert b"must not be negative" in lib.xsg_last_error()


def test_adam_arguments(lib):
    def call(tensor=None, options=None, step=WS, workspace=WS):
        t = (AdamTensor * 1)()
        for k, v in dict(dict(param=FAKE, grad=FAKE, exp_avg=FAKE, exp_avg_sq=FAKE, numel=12, lr=1e-3),
                         **(tensor or {})).items():
            setattr(t[0], k, v)
        o = AdamOptions(0.9, 0.999, 1e-8, 1, 0, 2, 1.0)
        for k, v in (options or {}).items():
            setattr(o, k, v)
        assert lib.xsg_adam_step(t, 1, C.byref(o), step, None, workspace, None) == -1
        return lib.xsg_last_error()

    for k in ("param", "grad", "exp_avg", "exp_avg_sq"):
        assert b"null" in call({k: None})
    assert b"unknown type" in call(dict(param_dtype=9))
    assert b"unknown type" in call(dict(grad_dtype=9))
    assert b"rows under its mask" in call(dict(mask=FAKE, rows=7))
    assert b"negative size" in call(dict(numel=-4))
    for o in (dict(beta1=1.0), dict(beta2=-0.1), dict(beta1=math.nan)):
        assert b"betas" in call(options=o)
    assert b"eps" in call(options=dict(eps=-1.0))
    assert b"max_norm" in call(options=dict(max_norm=-1.0))
    assert b"max_norm" in call(options=dict(max_norm=math.nan))
    assert b"unknown norm" in call(options=dict(norm=5))
    assert b"step counter" in call(step=None)
    assert b"null workspace" in call(workspace=None)
    assert b"aligned" in call(workspace=C.c_void_p(FAKE + 128))
    assert lib.xsg_adam_step(None, 0, None, WS, None, WS, None) == -1


def test_workspace_queries(lib):
    one = lib.xsg_grad_norm_workspace_bytes(_grads({}), 1)
    many = lib.xsg_grad_norm_workspace_bytes(_grads(*[dict(numel=1 << 28)] * 9), 9)
    assert 0 < one < many < 1 << 20
    assert lib.xsg_grad_norm_workspace_bytes(_grads(dict(numel=-1)), 1) == 0
    o = AdamOptions(0.9, 0.999, 1e-8, 0, 0, 2, 0.0)
    t = (AdamTensor * 1)()
    assert lib.xsg_adam_step_workspace_bytes(t, 1, C.byref(o)) == 0
    o.clip = 1
    assert lib.xsg_adam_step_workspace_bytes(t, 1, C.byref(o)) > 0


def test_python_layer_refuses_cpu_tensors_and_lists():
    import torch

    from xsimgs_amd import optim

    x = torch.ones(4)
    for call in (lambda: optim.grad_norm([x]), lambda: optim.clip_grads_([x], 1.0),
                 lambda: optim.adam_step_([x], [x], [x], [x], torch.zeros(1, dtype=torch.int64), lr=1.0)):
        with pytest.raises(RuntimeError, match="GPU tensors"):
            call()
    with pytest.raises(ValueError, match="one entry per tensor"):
        optim.grad_norm([x, x], masks=[None])
    assert torch.equal(x, torch.ones(4))
