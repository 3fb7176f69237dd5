"""Dropout and the feature norm without a GPU: the generator's restatement against its published answers, and what
is refused before anything runs."""
import ctypes as C
import os

import numpy as np
import pytest
import torch

import xsimgs_amd
from tests import _draws
from xsimgs_amd import rendering

F = 0xFFFFFFFF


@pytest.mark.parametrize("counter, key, answer", [
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((F, F, F, F), (F, F), (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
     (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))])
def test_generator_answers(counter, key, answer):
    """The paper's known answers for ten rounds."""
    assert tuple(int(x) for x in _draws.philox(counter, key)) == answer


def test_draws_do_not_depend_on_where_a_run_starts():
    whole = _draws.draws(0, 100, 77, 3)
    for first in (1, 7, 8, 13):
        assert np.array_equal(_draws.draws(first, 40, 77, 3), whole[first:first + 40])
    assert not np.array_equal(_draws.draws(0, 100, 77, 2), whole) and not np.array_equal(_draws.draws(0, 100, 78, 3), whole)


@pytest.mark.parametrize("seed", [-1, 2 ** 63, 1.0, None, True, "1"])
def test_seeds_are_refused(seed):
    x = torch.zeros(4)
    for call in (lambda: rendering.dropout(x, 0.5, seed), lambda: rendering.drop_mask(4, 0.5, seed),
                 lambda: rendering.activate_gaussians(torch.zeros(4, 3), x, drop=0.5, seed=seed),
                 lambda: rendering.group_norm_act(torch.zeros(1, 4, 2), 1, drop=0.5, seed=seed)):
        with pytest.raises(ValueError, match="seed"):
            call()


def test_arguments_are_refused():
    x = torch.zeros(2, 3, 4)
    for shared in (-1, 4):
        with pytest.raises(ValueError, match="shared"):
            rendering.dropout(x, 0.5, 1, shared=shared)
    with pytest.raises(ValueError, match="act"):
        rendering.group_norm_act(x, 1, act="tanh")
    for kw in (dict(act="tanh"), dict(drop=1.5), dict(drop=-0.1)):
        with pytest.raises(ValueError, match="FeatureNorm"):
            rendering.FeatureNorm(2, 8, **kw)
    for groups in (0, 3):
        with pytest.raises(ValueError, match="FeatureNorm"):
            rendering.FeatureNorm(groups, 8)
    with pytest.raises(ValueError, match="another seed"):
        rendering.FeatureNorm(2, 4, drop=0.5)(x)
    for call in (lambda: rendering.dropout(x, 0.5, 1), lambda: rendering.group_norm_act(x, 2),
                 lambda: rendering.drop_mask(4, 0.5, 1, device="cpu"),
                 lambda: rendering.activate_gaussians(torch.zeros(4, 3), torch.zeros(4), drop=0.5, seed=1)):
        with pytest.raises(RuntimeError, match="GPU tensors"):
            call()


class Drop(C.Structure):       # xsg_drop_desc, field for field
    _fields_ = [("p", C.c_double), ("seed", C.c_uint64), ("seed_at", C.c_void_p), ("stream", C.c_uint32)]


class Norm(C.Structure):       # xsg_norm_desc, field for field
    _fields_ = [("dtype", C.c_int), ("batch", C.c_int64), ("pixels", C.c_int64), ("channels", C.c_int),
                ("groups", C.c_int), ("x", C.c_void_p), ("batch_stride", C.c_int64), ("pixel_stride", C.c_int64),
                ("weight", C.c_void_p), ("bias", C.c_void_p), ("weight_dtype", C.c_int), ("bias_dtype", C.c_int),
                ("mask", C.c_void_p), ("act", C.c_int), ("eps", C.c_double), ("drop", Drop)]


@pytest.fixture(scope="module")
def lib():
    lib = C.CDLL(xsimgs_amd.LIB_PATH)
    lib.xsg_last_error.restype = C.c_char_p
    lib.xsg_group_norm_act_workspace_bytes.restype = C.c_size_t
    return lib


P = C.c_void_p(1 << 20)   # a pointer that no refused call follows


def _norm(**kw):
    d = Norm(dtype=0, batch=2, pixels=5, channels=8, groups=2, x=P, batch_stride=40, pixel_stride=8, act=2, eps=1e-5)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw, says", [
    (dict(dtype=3), "unknown type"), (dict(dtype=-1), "unknown type"), (dict(batch=-1), "negative size"),
    (dict(pixels=-1), "negative size"), (dict(channels=0), "channels"), (dict(channels=4097, groups=1), "channels"),
    (dict(groups=0), "divide"), (dict(groups=3), "divide"), (dict(groups=-2), "divide"), (dict(act=4), "activation"), (dict(act=-1), "activation"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(weight=P, weight_dtype=1), "weight and bias"),
    (dict(bias=P, bias_dtype=2), "weight and bias"), (dict(x=None), "null"), (dict(pixel_stride=-8), "stride"),
    (dict(batch_stride=-8), "stride"), (dict(pixels=1 << 50), "too large"), (dict(pixel_stride=1 << 59), "too large"),
    (dict(batch_stride=1 << 60), "too large"), (dict(drop=Drop(p=1.5)), "probability"),
    (dict(drop=Drop(p=float("nan"))), "probability")])
def test_norm_refusals(lib, kw, says):
    d = _norm(**kw)
    assert lib.xsg_group_norm_act_workspace_bytes(C.byref(d), 0) == 0
    for call in (lambda: lib.xsg_group_norm_act_fwd(C.byref(d), P, P, P, None),
                 lambda: lib.xsg_group_norm_act_bwd(C.byref(d), P, P, P, P, P, P, None)):
        assert call() == -1
        assert says in lib.xsg_last_error().decode()


def test_norm_pointers_and_sizes(lib):
    d = _norm()
    odd = C.c_void_p((1 << 20) + 16)
    for call in (lambda: lib.xsg_group_norm_act_fwd(None, P, P, P, None), lambda: lib.xsg_group_norm_act_fwd(C.byref(d), None, P, P, None),
                 lambda: lib.xsg_group_norm_act_fwd(C.byref(d), P, None, P, None),
                 lambda: lib.xsg_group_norm_act_fwd(C.byref(d), P, P, odd, None),
                 lambda: lib.xsg_group_norm_act_fwd(C.byref(d), P, C.c_void_p((1 << 20) + 4), P, None),
                 lambda: lib.xsg_group_norm_act_bwd(C.byref(d), None, P, P, P, P, P, None),
                 lambda: lib.xsg_group_norm_act_bwd(C.byref(d), P, None, P, P, P, P, None),
                 lambda: lib.xsg_group_norm_act_bwd(C.byref(d), P, P, P, P, P, odd, None)):
        assert call() == -1
    # nothing to do: no error, no workspace, nothing launched
    for kw in (dict(batch=0), dict(pixels=0)):
        e = _norm(x=None, **kw)
        assert lib.xsg_group_norm_act_workspace_bytes(C.byref(e), 0) == 0
        assert lib.xsg_group_norm_act_fwd(C.byref(e), None, None, None, None) == 0
    assert lib.xsg_group_norm_act_bwd(C.byref(d), None, None, None, None, None, None, None) == 0
    many = _norm(batch=1 << 24, pixels=1, batch_stride=8)
    for call in (lambda: lib.xsg_group_norm_act_fwd(C.byref(many), P, P, P, None),
                 lambda: lib.xsg_group_norm_act_bwd(C.byref(many), P, P, P, P, P, P, None)):
        assert call() == -1 and "too many samples" in lib.xsg_last_error().decode()
    big = _norm(batch=6, pixels=2_073_600, channels=64, groups=8, batch_stride=64 * 2_073_600, pixel_stride=64)
    for backward in (0, 1):
        assert 0 < lib.xsg_group_norm_act_workspace_bytes(C.byref(big), backward) < 4 << 20


def test_dropout_refusals(lib):
    i64 = C.c_int64
    d, bad = Drop(p=0.5, seed=1), Drop(p=-0.5)
    for args in ((C.byref(bad), 0, i64(8), i64(1), P, P, None), (None, 0, i64(8), i64(1), P, P, None),
                 (C.byref(d), 3, i64(8), i64(1), P, P, None), (C.byref(d), 0, i64(-8), i64(1), P, P, None),
                 (C.byref(d), 0, i64(8), i64(0), P, P, None), (C.byref(d), 0, i64(8), i64(3), P, P, None),
                 (C.byref(d), 0, i64(8), i64(1), None, P, None), (C.byref(d), 0, i64(8), i64(1), P, None, None)):
        assert lib.xsg_dropout(*args) == -1
    assert lib.xsg_dropout(C.byref(d), 0, i64(0), i64(1), None, None, None) == 0
    assert lib.xsg_drop_mask(C.byref(bad), i64(8), P, None) == -1 and lib.xsg_drop_mask(None, i64(8), P, None) == -1
    assert lib.xsg_drop_mask(C.byref(d), i64(-1), P, None) == -1 and lib.xsg_drop_mask(C.byref(d), i64(8), None, None) == -1
    assert lib.xsg_drop_mask(C.byref(d), i64(0), None, None) == 0
    for f in (lib.xsg_activate_drop_fwd, lib.xsg_activate_drop_bwd):
        more = (P, P) if f is lib.xsg_activate_drop_bwd else ()
        assert f(C.byref(bad), i64(8), P, P, P, P, *more, None) == -1
        assert f(C.byref(d), i64(-1), P, P, P, P, *more, None) == -1
        assert f(C.byref(d), i64(8), P, None, P, P, *more, None) == -1
        assert f(C.byref(d), i64(0), None, None, None, None, *((None, None) if more else ()), None) == 0
