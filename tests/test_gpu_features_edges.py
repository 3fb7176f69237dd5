"""The feature norm and dropout at the places where they once went wrong. Tolerances: those of test_gpu_features, whose
formula in 64 bits is used; what is exact is said where it is asserted."""
import pytest
import torch

from tests.test_gpu_features import TYPES, _params, _randn, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("channels, groups, pixels", [(16, 4, 3000), (8, 1, 5000), (40, 40, 25_000), (65, 5, 9000)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("where", ["first", "middle", "last", "all but the last"])
def test_offsets_under_a_mask(dev, dtype, channels, groups, pixels, where):
    """A mean of many spreads, and parts of the image (first of all its beginning) that the mask empties and that hold no
    numbers: an empty part has no mean, and the joint variance is no difference of what 32 bits hold. With 40 groups the
    parts are too many for the kernels that need them to join them."""
    offset, spread = dict(zip(TYPES, ((1000.0, 1.0), (1000.0, 8.0), (1000.0, 1.0))))[dtype]
    x = (_randn((2, pixels, channels), 1, dev) * spread + offset).to(dtype)
    part = min(pixels // 3, 1500)
    mask = torch.ones(2, pixels, dtype=torch.bool, device=dev)
    mask[:, {"first": slice(0, part), "middle": slice(part, 2 * part), "last": slice(pixels - part, None),
             "all but the last": slice(0, pixels - 100)}[where]] = False
    x[~mask] = float("nan")
    w, b = _params(channels, 5, dev)
    _run(x, groups, w, b, mask=mask, v_y=_randn(x.shape, 7, dev, dtype))


def test_a_beginning_far_from_the_rest(dev):
    """The only pixel of the first part that the mask leaves lies hundreds of deviations from the mean."""
    x = _randn((1, 100_000, 4), 1, dev)
    x[:, 0] = 1e4
    mask = torch.ones(1, 100_000, dtype=torch.bool, device=dev)
    mask[:, 1:2000] = False
    w, b = _params(4, 5, dev)
    _run(x, 1, w, b, act="gelu", mask=mask, v_y=_randn(x.shape, 7, dev))

@pytest.mark.parametrize("value", [0.1, -77.77, 1000.1, 3e5 + 0.3])
@pytest.mark.parametrize("channels, groups", [(4, 2), (9, 3), (64, 8), (1, 1), (130, 1)])
def test_flat_images(dev, value, channels, groups):
    """Each pixel of a flat image is its bias, whatever the value: its mean is the value itself, and (x - mean) is 0."""
    from xsimgs_amd import rendering

    w, b = _params(channels, 5, dev)
    for dtype in TYPES:
        for pixels in (50, 3001, 40_000):
            flat = torch.full((1, pixels, channels), value if dtype != torch.float16 else value / 10, dtype=dtype, device=dev)
            assert torch.equal(rendering.group_norm_act(flat, groups, w, b, act="none"), b.to(dtype).expand(flat.shape))
            mask = torch.ones(1, pixels, dtype=torch.bool, device=dev)
            mask[:, :pixels // 4] = False
            mask[:, ::7] = False
            y = rendering.group_norm_act(flat, groups, w, b, act="none", mask=mask)
            assert torch.equal(y, torch.where(mask[..., None], b.to(dtype), 0.0).to(dtype))

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["relu", "silu", "gelu"])
@pytest.mark.parametrize("pixels", [30, 2500])
def test_biases_at_the_ends_of_float32(dev, dtype, act, pixels):
    """A channel that its bias switches off gives 0 and no gradient; one far on the other side is linear. At z = -88 and
    below each activation and its slope are less than 1e-36 in size."""
    from xsimgs_amd import rendering

    low = torch.tensor([torch.finfo(torch.float32).min, -1e30, -1e6, -200.0])
    high = torch.tensor([torch.finfo(torch.float32).max, 2.5e38, 1e30, 1e4])
    x, v_y = _randn((2, pixels, 12), 1, dev, dtype).requires_grad_(), _randn((2, pixels, 12), 7, dev, dtype)
    w = torch.ones(12, device=dev, requires_grad=True)
    b = torch.cat([low, high, torch.zeros(4)]).to(dev).requires_grad_()
    y = rendering.group_norm_act(x, 3, w, b, act=act)
    assert bool((y[..., :4].float().abs() <= 1e-30).all())
    z = rendering.group_norm_act(x, 3, w, b, act="none")       # the same values without an activation
    half = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    # the activation is z itself there: each is rounded once, after 8 units of float32
    far, want = y[..., 4:8].detach().double(), z[..., 4:8].detach().double()
    assert bool(((far == want) | ((far - want).abs() <= (2 * half + 2.0 ** -20) * want.abs())).all())
    v_x, v_w, v_b = torch.autograd.grad(y, [x, w, b], v_y)
    assert bool((v_x[..., :4] == 0).all()) and bool((v_w[:4].abs() <= 1e-30).all()) and bool((v_b[:4].abs() <= 1e-30).all())
    want = v_y[..., 4:8].double().sum((0, 1))
    assert bool(((v_b[4:8].double() - want).abs() <= 80 * 2.0 ** -24 * v_y[..., 4:8].double().abs().sum((0, 1))).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["relu", "silu", "gelu"])
@pytest.mark.parametrize("pixels", [30, 2500])
def test_an_infinite_bias(dev, dtype, act, pixels):
    """Activations of infinity are infinity."""
    from xsimgs_amd import rendering

    b = torch.full((8,), float("inf"), device=dev)
    y = rendering.group_norm_act(_randn((2, pixels, 8), 1, dev, dtype), 2, None, b, act=act)
    assert bool((y == float("inf")).all())

def test_a_frames_head_that_drops_needs_a_seed(dev):
    """Without one the same features would be dropped in every step; a head in evaluation needs none."""
    from tests.test_gpu_frame_drop import _image_grads, _scene
    from xsimgs_amd import frame, rendering

    for rig in (False, True):
        sc = _scene("rig" if rig else "cfg0", 8)
        st = frame.prepare(sc, dev, head=rendering.FeatureNorm(2, 8, drop=0.25))
        opt = frame.make_optimizer(st)
        before = [t.detach().clone() for t in (st.means, st.colors, st.head.weight)]
        grads = _image_grads(sc, 8, dev, rig)
        render = frame.render_rig if rig else frame.render_frame
        for call in (lambda: render(st), lambda: frame.train_frame(st, opt, grads, rig=rig),
                     lambda: frame.train_frame(st, opt, grads, rig=rig, drop=0.2)):
            with pytest.raises(ValueError, match="seed"):
                call()
        assert all(torch.equal(a, t.detach()) for a, t in zip(before, (st.means, st.colors, st.head.weight)))
        st.head.eval()
        frame.train_frame(st, opt, grads, rig=rig)
        assert not torch.equal(before[2], st.head.weight.detach())

def test_a_gradients_tangent_is_refused(dev):
    """A tangent of the incoming gradient alone (a dual parameter behind the operator) would be lost in the backward."""
    import torch.autograd.forward_ad as fwd

    from xsimgs_amd import rendering

    x = _randn((2, 20, 8), 1, dev).requires_grad_()
    a, o = _randn((20, 3), 2, dev).requires_grad_(), _randn((20,), 3, dev).requires_grad_()
    with fwd.dual_level():
        p = fwd.make_dual(torch.ones((), device=dev), torch.ones((), device=dev))
        for y, leaf in ((rendering.dropout(x, 0.5, 1), x), (rendering.group_norm_act(x, 2), x),
                        (rendering.activate_gaussians(a, o, drop=0.5, seed=1)[1], o),
                        (rendering.activate_gaussians(a, o, drop=0.5, seed=1)[0], a)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y.sum() * p, leaf)

def test_gradients_of_a_dropout_that_depend_on_nothing(dev):
    """Dropout is linear: its gradient depends on the incoming gradient alone, and where that is a constant so is it. A
    penalty on it beside other terms is differentiated as usual."""
    from xsimgs_amd import rendering

    x = _randn((50, 8), 1, dev).requires_grad_()
    g, = torch.autograd.grad(rendering.dropout(x, 0.5, 1).sum(), x, create_graph=True)
    assert not g.requires_grad
    again, = torch.autograd.grad((g * x).sum(), x)
    assert torch.equal(again, g)

def test_the_most_samples(dev):
    """2^23 - 1 samples forward and backward; one more is refused in both."""
    from xsimgs_amd import rendering

    n = 2 ** 23 - 1
    x, v_y = torch.randn((n, 2), device=dev), torch.randn((n, 2), device=dev)
    w, b = _params(2, 5, dev)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    y = rendering.group_norm_act(leaves[0], 1, *leaves[1:])
    v_x, v_w, v_b = torch.autograd.grad(y, leaves, v_y)
    for at in (slice(0, 500), slice(n // 2, n // 2 + 500), slice(n - 500, n)):
        some = _run(x[at], 1, w, b, v_y=v_y[at])
        assert torch.equal(y[at].detach(), some["y"]) and torch.equal(v_x[at], some["v_x"])
    xd = x.double()
    xh = (xd - xd.mean(1, keepdim=True)) / (xd.var(1, correction=0, keepdim=True) + 1e-5).sqrt()
    z = xh * w.double() + b.double()
    s = torch.sigmoid(z)
    dz = v_y.double() * s * (1 + z * (1 - s))
    # per term 132 U of xh (5e3 U where the spread is smaller than sqrt(eps): |mean| rstd) and 80 U of its own; sums in 64 bits
    for got, terms in ((v_b, dz), (v_w, dz * xh)):
        loose = (v_y.double().abs() * (1 + x.double().abs().amax(1, keepdim=True) * 320)).sum(0)
        assert bool(((got.double() - terms.sum(0)).abs() <= 400 * 2.0 ** -24 * loose).all())
    with pytest.raises(RuntimeError, match="too many samples"):
        rendering.group_norm_act(torch.zeros(n + 1, 2, device=dev), 1)


def test_more_groups_than_a_launch_has_workgroups(dev):
    """2049 samples of 4096 groups are more than 2^23: the launches that join their parts take several in turn. The samples
    repeat, so each gives what it gives in a call of 64."""
    from xsimgs_amd import rendering

    w, b = (t.to(torch.bfloat16) for t in _params(4096, 5, dev))
    for pixels in (3, 260):      # a forward in one launch, and in several
        one, g = _randn((1, pixels, 4096), 1, dev, torch.bfloat16), _randn((1, pixels, 4096), 2, dev, torch.bfloat16)
        want = _run(one, 4096, w, b, v_y=g)
        x = one.expand(2049, pixels, 4096).detach().requires_grad_()
        y = rendering.group_norm_act(x, 4096, w, b)
        v_x, = torch.autograd.grad(y, x, g.expand(x.shape))
        for got, name in ((y, "y"), (v_x, "v_x")):
            off = (got.detach().float() - want[name].float()).abs()
            assert bool((off <= 2.0 ** -7 * want[name].float().abs() + 1e-6).all())
            assert bool((got[1:] == got[:1]).all())
