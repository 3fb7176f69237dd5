"""Group norm with an activation and dropout against its formula in 64 bits.

Tolerances, with U = 2^-24 (a rounding to float32), f the kept elements' factor and H the result's half step:

* the sums behind mean and variance go through at most 64 roundings each after another here (a thread's run, its
  workgroup, then 64 bits), each of U of what is summed: 64 U mean|x - mean| on the mean, 128 U relative on the
  deviation; the mean itself is rounded to float32: U |mean|. In units of the spread: dm = 64 U + 2 U |mean| rstd.
* xh is off by dm + (128 + 4) U |xh|, z = w xh + b by |w| of it and 4 U (|z| + |b|)
* an activation's slope is at most 1.13 and its curvature at most 0.8; the functions themselves are good to 8 U, and
  in the 16-bit types to (8 + 2 |z|) U (an exponent rounded before exp2): their own half step is far above
* gradients: dz is off by f |v_y| times (0.8 dz_z + (8 + 2 |z|) U), sums by 64 U of their terms' magnitudes and by
  their terms' errors; v_x carries these through its formula."""
import math

import pytest
import torch

from tests import _draws

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = list(HALF)
ACTS = ("none", "relu", "silu", "gelu")


def _randn(shape, seed, dev, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(dev)


def _act(z, act):
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if act == "gelu":
        phi = 0.5 * (1 + torch.erf(z / math.sqrt(2)))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return z, torch.ones_like(z)


def _formula(x, groups, w, b, act, eps, mask, drop, seed, stream, v_y=None):
    """{name: (value, bound on the error before the result's own rounding)} in 64 bits on the CPU."""
    shape, c = x.shape, x.shape[-1]
    n_b = shape[0]
    cg = c // groups
    keep = torch.ones(shape[:-1], dtype=torch.bool) if mask is None else mask.cpu().bool()
    keep = keep.reshape(n_b, -1, 1, 1)
    x = torch.where(keep, x.detach().cpu().double().reshape(n_b, -1, groups, cg), 0.0)
    w = torch.ones(c, dtype=torch.float64) if w is None else w.detach().cpu().double()
    b = torch.zeros(c, dtype=torch.float64) if b is None else b.detach().cpu().double()
    w, b = w.view(groups, cg), b.view(groups, cg)
    n = (keep.sum(1, keepdim=True) * cg).clamp(min=1)
    mean = x.sum((1, 3), keepdim=True) / n
    var = torch.where(keep, (x - mean) ** 2, 0.0).sum((1, 3), keepdim=True) / n
    rstd = torch.where(keep.any(1, keepdim=True), 1 / (var + eps).sqrt(), 0.0)
    xh = torch.where(keep, (x - mean) * rstd, 0.0)
    z = xh * w + b
    y, slope = _act(z, act)
    f = torch.ones_like(x)
    if drop:
        kept, factor = _draws.kept(x.numel(), drop, seed, stream)
        f = torch.as_tensor(kept).view(x.shape).double() * factor
    f = torch.where(keep, f, 0.0)
    dm = 64 * U + 2 * U * mean.abs() * rstd
    dxh = dm + 132 * U * xh.abs()
    dz_z = w.abs() * dxh + 4 * U * (z.abs() + b.abs())
    own = (8 + 2 * z.abs()) * U
    out = dict(y=((y * f).view(shape), (f * (1.13 * dz_z + own * y.abs())).view(shape)))
    if v_y is None:
        return out
    g = f * v_y.detach().cpu().double().reshape(x.shape)
    dz, e_dz = g * slope, g.abs() * (0.8 * dz_z + own * 1.13)
    if act == "relu":    # a kink: an error of z may pass it
        e_dz = e_dz + g.abs() * (z.abs() <= dz_z)

    def total(t, e, dims):
        return t.sum(dims, keepdim=True), (e + 64 * U * t.abs()).sum(dims, keepdim=True)

    tb, eb = total(dz, e_dz, (0, 1))
    tw, ew = total(dz * xh, e_dz * xh.abs() + dz.abs() * dxh, (0, 1))
    out["v_bias"], out["v_weight"] = (tb.view(c), eb.view(c)), (tw.view(c), ew.view(c))
    wdz, e_wdz = w * dz, w.abs() * (e_dz + 4 * U * dz.abs())
    m1, e1 = (t / n for t in total(wdz, e_wdz, (1, 3)))
    m2, e2 = (t / n for t in total(wdz * xh, e_wdz * xh.abs() + wdz.abs() * dxh, (1, 3)))
    dx = rstd * (wdz - m1 - xh * m2)
    e = rstd * (e_wdz + e1 + 8 * U * m1.abs() + xh.abs() * e2 + (dxh + 8 * U * xh.abs()) * m2.abs()) + 140 * U * dx.abs()
    out["v_x"] = (torch.where(keep, dx, 0.0).view(shape), torch.where(keep, e, 0.0).view(shape))
    return out


def _compare(name, got, want, error):
    half = HALF[got.dtype]
    bound = half * want.abs() + (1 + half) * error + (2.0 ** -25 if got.dtype == torch.float16 else 1e-38)
    off = (got.detach().cpu().double() - want).abs()
    worst = float((off / bound).max()) if off.numel() else 0.0
    assert got.shape == want.shape and bool((off <= bound).all()), f"{name}: {worst} of the bound"


def _run(x, groups, w=None, b=None, *, act="silu", eps=1e-5, mask=None, drop=0.0, seed=0, stream=0, v_y=None):
    """Forward alone, forward with a graph and backward, all checked; returns what came out."""
    from xsimgs_amd import rendering

    kw = dict(act=act, eps=eps, mask=mask, drop=drop, seed=seed, stream=stream)
    want = _formula(x, groups, w, b, act, eps, mask, drop, seed, stream, v_y)
    alone = rendering.group_norm_act(x.detach(), groups, None if w is None else w.detach(), None if b is None else b.detach(), **kw)
    assert alone.dtype == x.dtype and alone.is_contiguous()
    _compare("y", alone, *want["y"])
    if mask is not None:
        assert bool((alone[~mask.bool()] == 0).all())
    out = dict(y=alone)
    if v_y is None:
        return out
    leaves = {k: t.detach().requires_grad_() for k, t in (("v_x", x), ("v_weight", w), ("v_bias", b)) if t is not None}
    y = rendering.group_norm_act(leaves["v_x"], groups, leaves.get("v_weight"), leaves.get("v_bias"), **kw)
    assert torch.equal(y.detach(), alone)
    for k, g in zip(leaves, torch.autograd.grad(y, list(leaves.values()), v_y)):
        assert g.dtype == leaves[k].dtype
        _compare(k, g, *want[k])
        out[k] = g
    if mask is not None:
        assert bool((out["v_x"][~mask.bool()] == 0).all())
    return out


def _params(c, seed, dev, dtype=torch.float32):
    return (1 + 0.2 * _randn((c,), seed, dev)).to(dtype), (0.3 * _randn((c,), seed + 1, dev)).to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("channels, groups", [(1, 1), (2, 1), (2, 2), (3, 1), (3, 3), (4, 2), (5, 1), (5, 5), (6, 2), (7, 7),
                                              (8, 1), (8, 2), (9, 3), (12, 4), (16, 4), (17, 1), (24, 3), (32, 8), (33, 3),
                                              (48, 6), (64, 64), (65, 5), (96, 32), (129, 3), (256, 8), (257, 1), (320, 32),
                                              (512, 16), (513, 27), (640, 5)])
def test_channels_and_groups(dev, dtype, channels, groups):
    x = _randn((2, 9, 13, channels), channels, dev, dtype)
    w, b = _params(channels, 5, dev)
    _run(x, groups, w, b, v_y=_randn(x.shape, 7, dev, dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pixels", [1, 2, 3, 31, 64, 100, 255, 256, 257, 1000, 4099, 33_333])
@pytest.mark.parametrize("channels, groups", [(32, 8), (9, 3)])
def test_lengths(dev, dtype, pixels, channels, groups):
    x = _randn((1, pixels, channels), pixels, dev, dtype) + 0.5
    w, b = _params(channels, 5, dev)
    _run(x, groups, w, b, v_y=_randn(x.shape, 7, dev, dtype))


@pytest.mark.parametrize("channels, groups, dtype", [(2048, 32, torch.float32), (2052, 4, torch.float32), (4096, 64, torch.float32),
                                                     (4096, 4096, torch.bfloat16), (4095, 5, torch.float16), (3333, 11, torch.float32)])
def test_most_channels(dev, channels, groups, dtype):
    x = _randn((2, 37, channels), 3, dev, dtype)
    w, b = _params(channels, 5, dev)
    _run(x, groups, w, b, v_y=_randn(x.shape, 7, dev, dtype), drop=0.1, seed=3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("drop", [0.0, 0.3, 1.0])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("channels, groups", [(16, 4), (11, 1), (3, 3)])
def test_activations_drops_and_masks(dev, dtype, act, drop, masked, channels, groups):
    x = _randn((3, 5, 67, channels), 11, dev, dtype)
    w, b = _params(channels, 5, dev, dtype)
    mask = None
    if masked:
        mask = (torch.rand(x.shape[:-1], generator=torch.Generator().manual_seed(2)) < 0.6).to(dev)
        mask[1] = False                    # a sample without any pixel
        mask[2] = False
        mask[2, 3, 5] = True               # and one with a single one
        x[~mask] = float("nan")
        x[0, 0, 0] = float("inf")
        mask[0, 0, 0] = False
    out = _run(x, groups, w, b, act=act, mask=mask, drop=drop, seed=77, stream=3, v_y=_randn(x.shape, 7, dev, dtype))
    if drop == 1.0:
        assert all(bool((t == 0).all()) for t in out.values())


def test_large_values(dev):
    """An activation far out on both sides, with no NaN from an overflowing exponential."""
    x = _randn((1, 400, 8), 1, dev)
    for act in ACTS:
        w = torch.full((8,), 200.0, device=dev)
        _run(x, 2, w, torch.zeros(8, device=dev), act=act, v_y=_randn(x.shape, 7, dev))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_offsets_large_against_the_spread(dev, dtype):
    """A mean of 1000 spreads: the variance does not come from a difference of squares. (bfloat16 holds 100 spreads.)"""
    offset = 1000.0 if dtype == torch.float32 else 100.0
    x = (_randn((2, 3000, 16), 1, dev) + offset).to(dtype)
    w, b = _params(16, 5, dev)
    _run(x, 4, w, b, act="silu", v_y=_randn(x.shape, 7, dev, dtype))
    outlier = x.clone()
    outlier[:, 0] = 0                      # the first pixel is background
    _run(outlier, 4, w, b, act="silu")


def test_constant_groups(dev):
    x = torch.full((1, 50, 4), 3.25, device=dev)
    w, b = _params(4, 5, dev)
    _run(x, 2, w, b, act="none", v_y=_randn(x.shape, 7, dev))
    # a flat image far from zero is its bias, in every type
    from xsimgs_amd import rendering

    for dtype in TYPES:
        for pixels in (50, 40_000):
            flat = torch.full((1, pixels, 4), 1000.0, dtype=dtype, device=dev)
            assert torch.equal(rendering.group_norm_act(flat, 2, w, b, act="none"), b.to(dtype).expand(flat.shape))


@pytest.mark.parametrize("pixels", [30, 6000])
def test_samples_out_of_the_mask_without_eps(dev, pixels):
    x, (w, b) = _randn((3, pixels, 8), 1, dev), _params(8, 5, dev)
    mask = torch.ones(3, pixels, dtype=torch.bool, device=dev)
    mask[1] = False
    _run(x, 2, w, b, eps=0.0, mask=mask, v_y=_randn(x.shape, 7, dev))


@pytest.mark.parametrize("batch", [1, 7, 65, 1500])
def test_batches(dev, batch):
    x = _randn((batch, 6, 3, 8), 1, dev, torch.float16)
    w, b = _params(8, 5, dev)
    _run(x, 2, w, b, v_y=_randn(x.shape, 7, dev, torch.float16))
    _run(_randn((batch, 8), 1, dev), 2, w, b, v_y=_randn((batch, 8), 7, dev))     # no dimension of pixels


@pytest.mark.parametrize("dtype", TYPES)
def test_strides(dev, dtype):
    big = _randn((3, 20, 31, 37), 1, dev, dtype)
    flat = _randn((5000,), 2, dev, dtype)
    w, b = _params(32, 5, dev)
    views = [big[..., :32], big[..., 5:], big[:, 3:, 1:, 2:34], big[::2, :, :, 1:33], big[:, ::2, ::3, :32],
             big[:1].expand(4, 20, 31, 37)[..., 3:35], big.permute(0, 3, 1, 2)[:, :, :, :16].permute(0, 2, 1, 3)[..., :16],
             flat[1:1 + 32 * 9].view(1, 9, 32), flat[:32].expand(2, 7, 32)]
    for i, x in enumerate(views):
        c = x.shape[-1]
        _run(x, 4, w[:c], b[:c], v_y=_randn(x.shape, 7 + i, dev, dtype), drop=0.1, seed=9)
    # strided parameters, mask and gradient
    x = big[..., :32]
    wide = _randn((32, 2), 4, dev)
    mask = (torch.rand((3, 20, 62), generator=torch.Generator().manual_seed(2)) < 0.6).to(dev)[..., ::2]
    _run(x, 4, wide[:, 0], wide[:, 1], mask=mask, v_y=_randn((3, 31, 20, 32), 3, dev, dtype).transpose(1, 2))
    _run(x, 4, w, b, mask=mask.to(torch.uint8) * 3, v_y=_randn(x.shape, 3, dev, dtype))
    _run(x, 4, w, b, v_y=_randn((32,), 3, dev, dtype).expand(x.shape))


@pytest.mark.parametrize("weight, bias", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_without_parameters(dev, weight, bias, dtype):
    x = _randn((2, 77, 24), 1, dev, dtype)
    w, b = _params(24, 5, dev, dtype)
    _run(x, 3, w if weight else None, b if bias else None, v_y=_randn(x.shape, 7, dev, dtype))


def test_gradients_of_some(dev):
    """Each leaf's gradient is the same whichever others are asked for."""
    from xsimgs_amd import rendering

    x, (w, b), g = _randn((2, 500, 24), 1, dev), _params(24, 5, dev), _randn((2, 500, 24), 3, dev)
    whole = _run(x, 3, w, b, v_y=g)
    for some in range(1, 8):
        leaves = [t.detach().requires_grad_(bool(some >> i & 1)) for i, t in enumerate((x, w, b))]
        y = rendering.group_norm_act(leaves[0], 3, *leaves[1:])
        asked = [(k, t) for k, t in zip(("v_x", "v_weight", "v_bias"), leaves) if t.requires_grad]
        for (k, _), got in zip(asked, torch.autograd.grad(y, [t for _, t in asked], g)):
            assert torch.equal(got, whole[k])


def test_gradients_against_differences(dev):
    """Central differences of the formula in 64 bits, along random directions: h^2 terms are below 1e-7 here."""
    x, (w, b), g = _randn((1, 40, 6), 1, dev), _params(6, 5, dev), _randn((1, 40, 6), 3, dev)
    for act in ("none", "silu", "gelu"):
        out = _run(x, 2, w, b, act=act, drop=0.2, seed=5, v_y=g)
        h = 1e-4
        for k, i in (("v_x", 0), ("v_weight", 1), ("v_bias", 2)):
            at = [x.double().cpu(), w.double().cpu(), b.double().cpu()]
            d = torch.randn(at[i].shape, generator=torch.Generator().manual_seed(8), dtype=torch.float64)
            f = []
            for sign in (1, -1):
                moved = list(at)
                moved[i] = at[i] + sign * h * d
                y, _ = _formula(moved[0], 2, moved[1], moved[2], act, 1e-5, None, 0.2, 5, 0)["y"]
                f.append(float((y * g.double().cpu()).sum()))
            slope, got = (f[0] - f[1]) / (2 * h), float((out[k].double().cpu() * d).sum())
            assert abs(slope - got) <= 2e-5 * float(out[k].double().cpu().abs().mul(d.abs()).sum()), (act, k)


def test_dropout_behind_is_dropout(dev):
    """The fused dropout is rendering.dropout of the result under the same seed and stream."""
    from xsimgs_amd import rendering

    for c in (64, 32, 11, 3):
        for dtype in TYPES:
            x = _randn((2, 1301, c), 1, dev, dtype).requires_grad_()
            y = rendering.group_norm_act(x.detach(), 1, act="silu")
            # the last two: a threshold below 2^16, and one that a value's own 32 bits equal but for one
            u = _draws.draws(0, y.numel(), 6, 4)
            for p in (0.3, 0.999, 1e-5, (int(u[9 * c + 1]) + 1) / 2 ** 32):
                kept = rendering.dropout(torch.ones_like(y), p, 6, stream=4).ne(0)
                assert torch.equal(kept.cpu().view(-1), torch.as_tensor(_draws.kept(y.numel(), p, 6, 4)[0]))
                dropped = rendering.group_norm_act(x, 1, act="silu", drop=p, seed=6, stream=4)
                assert torch.equal(dropped != 0, kept & (y != 0))
                # with everything else out, v_b is the sum of the kept elements' factors and slopes
                b = torch.zeros(c, device=dev, requires_grad=True)
                z = rendering.group_norm_act(x, 1, None, b, act="none", drop=p, seed=6, stream=4)
                g, = torch.autograd.grad(z, b, torch.ones_like(z))
                want = kept.view(-1, c).double().sum(0) * _draws.kept(1, p, 6)[1]
                assert bool(((g.double() - want).abs() <= 128 * U * want).all())


def test_the_same_bits_each_time(dev):
    from xsimgs_amd import rendering

    x, (w, b), g = _randn((2, 200, 301, 48), 1, dev), _params(48, 5, dev), _randn((2, 200, 301, 48), 3, dev)
    leaves = [t.requires_grad_() for t in (x, w, b)]

    def once():
        y = rendering.group_norm_act(x, 6, w, b, drop=0.1, seed=2)
        return [y.detach(), *torch.autograd.grad(y, leaves, g)]

    first = once()
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, once()))


def test_offsets_past_32_bits(dev):
    """Two samples more than 2^32 elements apart, and pixels as far apart."""
    buf = torch.empty(2 ** 32 + 10_000, dtype=torch.bfloat16, device=dev)
    x = buf.as_strided((2, 50, 16), (2 ** 32, 16, 1))
    x.copy_(_randn((2, 50, 16), 1, dev, torch.bfloat16))
    w, b = _params(16, 5, dev)
    _run(x, 2, w, b, v_y=_randn(x.shape, 7, dev, torch.bfloat16))
    x = buf.as_strided((1, 3, 16), (0, 2 ** 31, 1))
    x.copy_(_randn((1, 3, 16), 1, dev, torch.bfloat16))
    _run(x, 2, w, b, v_y=_randn(x.shape, 7, dev, torch.bfloat16))


def test_a_long_image(dev):
    """More than 2^31 elements in one sample: its halves are alike, so its statistics are those of a half."""
    from xsimgs_amd import rendering

    half = torch.randn((1, 2 ** 25 + 1, 32), device=dev, dtype=torch.bfloat16)
    w, b = _params(32, 5, dev)
    y = rendering.group_norm_act(half, 8, w, b, drop=0.0)
    twice = rendering.group_norm_act(torch.cat([half, half], 1), 8, w, b)
    n = half.shape[1]
    # the statistics differ in their sums' order alone: a step of bfloat16 at most, where a rounding tips
    for part in (twice[:, :n], twice[:, n:]):
        off = (part.float() - y.float()).abs()
        assert bool((off <= 2.0 ** -7 * y.float().abs() + 1e-6).all()) and float((off > 0).float().mean()) < 0.01


def test_nothing(dev):
    from xsimgs_amd import rendering

    for shape in ((0, 5, 8), (3, 0, 8), (0, 8)):
        x, (w, b) = torch.zeros(shape, device=dev, requires_grad=True), _params(8, 1, dev)
        w.requires_grad_(), b.requires_grad_()
        y = rendering.group_norm_act(x, 2, w, b, drop=0.5, seed=1)
        assert y.shape == shape
        for t, g in zip((x, w, b), torch.autograd.grad(y.sum(), [x, w, b])):
            assert g.shape == t.shape and bool((g == 0).all())


def test_values_that_are_not_finite(dev):
    """A NaN or infinity in the mask reaches its own group alone; dropped elements are 0 all the same."""
    from xsimgs_amd import rendering

    for bad in (float("nan"), float("inf")):
        x = _randn((2, 300, 8), 1, dev)
        x[1, 20, 5] = bad
        y = rendering.group_norm_act(x, 2, act="none")
        assert bool(torch.isnan(y[1, :, 4:]).all()) and not bool(torch.isnan(y[0]).any() | torch.isnan(y[1, :, :4]).any())
        y = rendering.group_norm_act(x, 2, act="none", drop=0.5, seed=1)
        kept = torch.as_tensor(_draws.kept(x.numel(), 0.5, 1)[0]).view(x.shape).to(dev)
        assert torch.equal(torch.isnan(y[1, :, 4:]), kept[1, :, 4:])


def test_refusals(dev):
    from xsimgs_amd import rendering

    x, (w, b) = _randn((2, 5, 8), 1, dev), _params(8, 1, dev)
    f = rendering.group_norm_act
    for call, says in ((lambda: f(x, 3), "divide"), (lambda: f(x, 0), "divide"), (lambda: f(x[0, 0], 2), "batch"),
                       (lambda: f(x.double(), 2), "float32, bfloat16 or float16"), (lambda: f(x, 2, w[:7], b), "per channel"),
                       (lambda: f(x, 2, w.half(), b), "x's type"), (lambda: f(x, 2, w.cpu(), b), "same device"),
                       (lambda: f(x, 2, w, b, mask=torch.ones(2, 5, 8, dtype=torch.bool, device=dev)), "sizes"),
                       (lambda: f(x, 2, w, b, mask=torch.ones(2, 5, device=dev)), "bool"),
                       (lambda: f(x, 2, w, b, mask=torch.ones(2, 5, dtype=torch.bool)), "same device"),
                       (lambda: f(x, 2, w, b, eps=-1.0), "eps"), (lambda: f(x, 2, drop=2.0), "probability"),
                       (lambda: f(x, 2, drop=0.5, stream=-1), "stream"), (lambda: f(torch.zeros(1, 2, 4097, device=dev), 1), "channels"),
                       (lambda: f(x, 2, drop=0.5, seed=torch.zeros(2, dtype=torch.int64, device=dev)), "one int64")):
        with pytest.raises(RuntimeError, match=says):
            call()
    # a gradient's gradient: the first comes, the second is refused, also beside other terms
    x.requires_grad_()
    for y in (f(x, 2, w, b), rendering.dropout(x, 0.5, 1)):
        g, = torch.autograd.grad((y * x).sum(), x, create_graph=True)
        for total in (g.sum(), (g * x).sum()):
            with pytest.raises(RuntimeError, match="differentiated once"):
                torch.autograd.grad(total, x, retain_graph=True)


def test_graphs_and_streams(dev):
    """Forward and backward captured and replayed on new values and seeds, with other work of the same call between the
    replays; then two graphs one after the other."""
    from xsimgs_amd import rendering

    shape = (2, 33, 47, 24)
    x, (w, b), g = _randn(shape, 1, dev).requires_grad_(), _params(24, 5, dev), _randn(shape, 3, dev)
    leaves = [x, w.requires_grad_(), b.requires_grad_()]
    seed = torch.full((1,), 7, dtype=torch.int64, device=dev)

    def both(s):
        y = rendering.group_norm_act(x, 3, w, b, drop=0.2, seed=s)
        return [y.detach(), *torch.autograd.grad(y, leaves, g)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = both(7)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(eager, both(seed)))
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(both(seed))
    for i, s in enumerate((7, 8, 9, 2 ** 50)):
        with torch.no_grad():
            x.copy_(_randn(shape, 20 + i, dev))
        seed.fill_(s)
        want = both(s)
        for graph in graphs:
            graph.replay()
        both(3)
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(p, q) for p, q in zip(out, want)), s


def test_module(dev):
    from xsimgs_amd import rendering

    m = rendering.FeatureNorm(4, 32, drop=0.25, stream=2, device=dev)
    x = _randn((2, 9, 9, 32), 1, dev)
    with torch.no_grad():
        m.weight.add_(_randn((32,), 2, dev))
    assert torch.equal(m(x, seed=5), rendering.group_norm_act(x, 4, m.weight, m.bias, drop=0.25, seed=5, stream=2))
    m(x, seed=5).sum().backward()
    assert m.weight.grad is not None and m.bias.grad is not None
    m.eval()
    assert torch.equal(m(x), rendering.group_norm_act(x, 4, m.weight, m.bias))
    assert "drop=0.25" in repr(m) and set(m.state_dict()) == {"weight", "bias"}
