"""What clip_grads_ writes back of a strided tensor: what changed, and in rows of the mask only."""
import ctypes as C
import math
import os

import numpy as np
import pytest
import torch

from tests.test_gpu_optim import U, _close, _f64, _norm64, _pack, _values

LIB = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "xsimgs_amd", "libxsimgs_hip.so")


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(LIB):
        pytest.fail(f"{LIB} is not built: run __graft_entry__.build()")
    lib = C.CDLL(LIB)
    lib.xsg_last_error.restype = C.c_char_p
    lib.xsg_write_back.argtypes = [C.c_void_p, C.c_void_p, C.c_int64, C.c_int, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p,
                                   C.c_int64, C.c_void_p]
    return lib


def _call(lib, dst=1 << 20, src=1 << 20, numel=12, size=4, sizes=(3, 4), strides=(9, 2), mask=None, rows=0, stream=None,
          dims=None):
    ints = lambda xs: None if xs is None else (C.c_int64 * max(1, len(xs)))(*xs)
    return lib.xsg_write_back(dst, src, numel, size, len(sizes) if dims is None else dims, ints(sizes), ints(strides), mask,
                              rows, stream)


@pytest.mark.parametrize("change,text", [
    (dict(dst=None), b"null"), (dict(src=None), b"null"), (dict(numel=-1), b"-1 elements"), (dict(numel=13), b"do not make"),
    (dict(size=8), b"8 bytes"), (dict(size=1), b"1 bytes"), (dict(dims=17), b"17 dimensions"), (dict(dims=-1), b"dimensions"),
    (dict(sizes=(-3, -4)), b"do not make"), (dict(sizes=(1 << 40, 1 << 40)), b"do not make"),
    (dict(sizes=None, dims=2), b"without sizes"), (dict(mask=1 << 20, rows=5), b"cannot have 5 rows"),
    (dict(mask=1 << 20, rows=0), b"cannot have 0 rows"), (dict(numel=1 << 50), b"elements")])
def test_arguments_are_checked(lib, change, text):
    """On the host, before any launch: the pointers are placeholders that no call reaches."""
    assert _call(lib, **change) == -1
    assert text in lib.xsg_last_error()


def test_nothing_to_write(lib):
    assert _call(lib, numel=0, sizes=(5, 0, 7), strides=(1, 1, 1), dst=None, src=None) == 0
    assert _call(lib, numel=0, sizes=(1 << 40, 1 << 40, 0), strides=(1, 1, 1), dst=None, src=None) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("masked", [False, True])
def test_what_is_written(dev, lib, dtype, masked):
    """Against indexing on the CPU, where rows out of the mask and what lies between have values of their own."""
    gen = torch.Generator().manual_seed(4)
    for shape, view in (((70, 9), lambda b: b[:, 2:7]), ((9, 70), lambda b: b.t()[::2]), ((33, 5, 6), lambda b: b[:, 1::2, :5]),
                        ((1031,), lambda b: b[7::3]), ((3, 4, 5, 2), lambda b: b.permute(2, 0, 3, 1)[:4]),
                        ((700, 900), lambda b: b[1:, 1:].t())):
        base = torch.randn(shape, generator=gen).to(dtype)
        src = torch.randn(view(base).shape, generator=gen).to(dtype)
        src.view(-1)[0] = math.nan
        n = src.shape[0]
        kept = np.random.default_rng(n).random(n) < 0.4 if masked else np.ones(n, bool)
        want = base.clone()
        at = view(want)
        at[torch.from_numpy(kept)] = src[torch.from_numpy(kept)]
        on, dense, mask = base.to(dev), src.to(dev), _pack(kept).to(dev)
        t = view(on)
        rc = _call(lib, t.data_ptr(), dense.data_ptr(), t.numel(), t.element_size(), t.shape, t.stride(),
                   mask.data_ptr() if masked else None, n, torch.cuda.current_stream().cuda_stream)
        assert rc == 0, lib.xsg_last_error()
        bits = torch.int32 if dtype == torch.float32 else torch.int16
        assert torch.equal(on.cpu().view(bits), want.view(bits)), shape


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_clip_strided_under_a_mask(dev, dtype):
    """Columns and a transpose under masks: kept rows are scaled where they lie, the others keep their bits."""
    from xsimgs_amd import optim

    base = _values((120, 90), dtype, 4)
    cuts = [lambda b: b[:, 3:20], lambda b: b[:, 20::3].t(), lambda b: b[::2, 22]]
    kept = [np.random.default_rng(i).random(cut(base).shape[0]) < 0.5 for i, cut in enumerate(cuts)]
    for cut, k in zip(cuts, kept):
        cut(base)[torch.from_numpy(~k)] = math.nan
    on = base.to(dev)
    norm = _norm64([_f64(cut(base))[torch.from_numpy(k)] for cut, k in zip(cuts, kept)], 2.0)
    got = optim.clip_grads_([cut(on) for cut in cuts], 0.5 * norm, masks=[_pack(k).to(dev) for k in kept])
    _close(got, norm, 2 * U)
    c, want, scaled = 0.5 * norm / (norm + 1e-6), _f64(base), torch.zeros(base.shape, dtype=torch.bool)
    for cut, k in zip(cuts, kept):
        cut(want)[torch.from_numpy(k)] *= c
        cut(scaled)[torch.from_numpy(k)] = True
    new = on.cpu()
    off = (_f64(new) - want).abs()[scaled]
    assert bool((off <= (3 * U + 1.001 * torch.finfo(dtype).eps / 2) * want.abs()[scaled] + 2.0 ** -133).all())
    bits = torch.int32 if dtype == torch.float32 else torch.int16
    assert torch.equal(new.view(bits)[~scaled], base.view(bits)[~scaled])


@pytest.mark.gpu
def test_another_streams_rows_are_left_alone(dev):
    """Rows out of the mask are another stream's to write while a clip runs: a copy written back whole would undo
    it. A long tensor in the same call leaves time in between."""
    from xsimgs_amd import optim

    long, base = torch.ones(1_500_000_000, device=dev), torch.zeros(64, 6, device=dev)
    part = base[:, 1:4]
    part[::2] = 1.0
    masks = [None, _pack(np.arange(64) % 2 == 0).to(dev)]
    rows = part[1::2]
    side = torch.cuda.Stream()
    delay = torch.empty(1 << 26, device=dev)
    for turn in range(1, 6):
        torch.cuda.synchronize()
        optim.clip_grads_([long, part], 1e4, masks=masks)   # of 3.9e4
        with torch.cuda.stream(side):
            for _ in range(turn):
                delay.zero_()
            rows.fill_(float(turn))
        torch.cuda.synchronize()
        assert bool((rows == turn).all()), turn
        long.fill_(1.0)
