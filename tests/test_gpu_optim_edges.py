"""The training step's operators and optimizer at the edges of what they take."""
import math
import random

import pytest
import torch

from tests.test_gpu_optim import U, _check_update, _close, _f64, _norm64, _pack, _state

pytestmark = pytest.mark.gpu


# the kinds of call: one workgroup, terms in the update's own workgroups, a table, terms in a launch of their own
LISTS = {"small": [(7,)], "ordinary": [(300, 3)] * 30, "long": [(11, 3)] * 120, "many chunks": [(17_000_000,)]}


@pytest.mark.parametrize("kind", [1.0, 2.0])
@pytest.mark.parametrize("lists", LISTS)
def test_norm_that_float32_cannot_hold_skips_the_step(dev, lists, kind):
    """Finite gradients whose norm is above the largest float32: the caller gets inf, and nothing moves."""
    from xsimgs_amd import optim

    p, g, m, v = ([torch.full(s, x, device=dev) for s in LISTS[lists]] for x in (0.5, 0.0, 0.25, 0.125))
    g[0].view(-1)[:2] = 3e38
    g[-1].view(-1)[-2:] = -3e38
    assert math.isfinite(_norm64([_f64(x) for x in g], kind))
    step = torch.full((1,), 4, dtype=torch.int64, device=dev)
    for limit in (None, 1.0):
        norm = optim.adam_step_(p, g, m, v, step, lr=1e-2, max_norm=limit, norm_type=kind, skip_nonfinite=True)
        assert math.isinf(float(norm)) and int(step) == 4
        for xs, old in ((p, 0.5), (m, 0.25), (v, 0.125)):
            assert all(bool((x == old).all()) for x in xs)
    # the largest magnitude is a float32 and finite: this step is taken
    norm = optim.adam_step_(p, g, m, v, step, lr=1e-2, max_norm=1.0, norm_type=math.inf, skip_nonfinite=True)
    assert float(norm) == float(torch.tensor(3e38)) and int(step) == 5
    assert not bool((m[0] == 0.25).any())


def test_masks_of_another_size_are_refused(dev):
    """A mask with words to spare is another tensor's, or another dimension's; nothing is written."""
    from xsimgs_amd import optim

    n = 100
    whole = _pack(torch.arange(n).numpy() % 2 == 0).to(dev)
    sh = torch.ones(3, 4, n, device=dev)   # the layout whose rows are channels
    for x, mask in ((sh, whole), (torch.ones(96, 3, device=dev), whole), (torch.ones(97, 3, device=dev), whole[:3])):
        param = torch.nn.Parameter(x.clone())
        param.grad = x.clone()
        z = lambda: torch.zeros_like(x)
        for call in (lambda: optim.grad_norm([x], masks=mask), lambda: optim.clip_grads_([x], 0.1, masks=mask),
                     lambda: optim.adam_step_([x], [z()], [z()], [z()], torch.zeros(1, dtype=torch.int64, device=dev),
                                              lr=1.0, masks=[mask]),
                     lambda: optim.Adam([param], lr=1.0).step(masks={param: mask})):
            with pytest.raises(RuntimeError, match="size mismatch"):
                call()
        assert bool((x == 1).all()) and bool((param == 1).all())


@pytest.mark.parametrize("n", [5, 1003])
def test_sh_of_the_second_layout_by_rows(dev, n):
    """[3, K, N] coefficients under the Gaussians' mask, as 3 K tensors of N."""
    from xsimgs_amd import optim

    rows = 3 * 16
    keep = torch.rand(n, generator=torch.Generator().manual_seed(3)) < 0.4
    before = _state([(n,)] * rows, [torch.float32] * rows, [torch.float32] * rows, 90, dev)
    for x in before[1]:
        x[~keep] = float("nan")
    whole = [torch.stack(xs).view(3, 16, n).to(dev) for xs in before]
    p, g, m, v = (list(x.view(rows, n)) for x in whole)
    norm = _norm64([_f64(x)[keep] for x in before[1]], 2.0)
    step = torch.full((1,), 11, dtype=torch.int64, device=dev)
    got = optim.adam_step_(p, g, m, v, step, lr=1e-2, eps=1e-15, max_norm=0.5 * norm, masks=_pack(keep.numpy()).to(dev))
    _close(got, norm, 2 * U)
    _check_update((p, m, v), before, 12, [1e-2] * rows, [0.0] * rows, 0.5 * norm / (norm + 1e-6), [keep] * rows)


def _scene(kind):
    from xsimgs_amd import synthetic

    if kind == "lidar":
        return synthetic.make_cfg3(seed=4, n=4000, width=128, n_beams=16)
    if kind == "camera":
        sc = synthetic.make_cfg0(seed=2, n=3000, width=96, height=64)
        sc.means[:500, 0] += 900.0   # beside the image
    else:
        sc = synthetic.make_cfg4(seed=4, n=6000, n_blobs=40)
        sc.cameras = synthetic.rig_cameras(80, 48, 63.0)[:3]   # a half of the circle
        sc.means[:500, 2] += 900.0   # above it
    return sc


@pytest.mark.parametrize("kind", ["camera", "rig", "lidar"])
def test_train_frame_updates_what_it_says(dev, kind):
    """Two steps of a frame, a rig and a lidar beside float64: the scene's parameters under their mask, and
    beside them parameters without dimensions and of the Gaussians' number, which no mask may hold back."""
    from xsimgs_amd import frame

    sc = _scene(kind)
    st = frame.prepare(sc, dev)
    gen = torch.Generator().manual_seed(1)
    cams = sc.cameras if kind == "rig" else sc.cameras[:1]
    shape = ((len(cams),) if kind == "rig" else ()) + (cams[0].height, cams[0].width)
    channels = 2 if kind == "lidar" else 3
    image = [(1e-3 * torch.randn(*s, generator=gen)).to(dev) for s in ((*shape, channels), shape, shape)]
    exposure, table = torch.nn.Parameter(torch.tensor(0.5, device=dev)), torch.nn.Parameter(torch.ones(sc.n, device=dev))
    opt = frame.make_optimizer(st, max_norm=1e-2)
    opt.add_param_group(dict(params=[exposure, table], lr=1e-2, name="others"))
    assert len(opt.param_groups) == 6
    params = [p for group in opt.param_groups for p in group["params"]]
    rates = [group["lr"] for group in opt.param_groups for _ in group["params"]]
    moments = [[torch.zeros(p.shape) for p in params] for _ in range(2)]
    own = [torch.tensor(3e-3), torch.randn(sc.n, generator=gen) * 1e-3]
    for t in (1, 2):
        old = [p.detach().cpu().clone() for p in params]
        exposure.grad, table.grad = (x.to(dev) for x in own)
        out = frame.train_frame(st, opt, image, rig=kind == "rig")
        grads = [out["grads"][group["name"]].cpu() for group in opt.param_groups[:5]] + own
        keep = torch.ones(sc.n, dtype=torch.bool)
        if kind != "lidar":
            seen = (out["radii"] > 0).all(-1).cpu()
            keep = seen.any(0) if kind == "rig" else seen
            assert 0 < int(keep.sum()) <= sc.n - 500
            assert not any(bool(g[~keep].any()) for g in grads[:5])
        norm = _norm64([_f64(g) for g in grads], 2.0)
        _close(out["grad_norm"], norm, 2 * U)
        now = [[p.detach() for p in params]] + [[opt.state[p][k] for p in params] for k in ("exp_avg", "exp_avg_sq")]
        everything = torch.ones(sc.n, dtype=torch.bool)
        keeps = [keep] * 5 + [torch.ones((), dtype=torch.bool), everything]
        _check_update(now, (old, grads, *moments), t, rates, [0.0] * 7, min(1.0, 1e-2 / (norm + 1e-6)), keeps)
        assert exposure.grad is None and table.grad is None and st.means.grad is not None
        assert float(exposure.detach()) != float(old[5]) and not bool((table.detach().cpu() == old[6]).any())
        moments = [[x.cpu().clone() for x in xs] for xs in now[1:]]


def test_train_frame_with_a_pose(dev):
    """A camera's position beside the scene: its gradient is this frame's alone, not a sum over the steps."""
    from xsimgs_amd import frame

    st = frame.prepare(_scene("camera"), dev)
    position = st.cams[0].pose.t.requires_grad_()
    gen = torch.Generator().manual_seed(1)
    image = [torch.randn(*s, generator=gen).to(dev) for s in ((64, 96, 3), (64, 96), (64, 96))]
    opt = frame.make_optimizer(st, rates=dict.fromkeys(frame.RATES, 0.0))
    opt.add_param_group(dict(params=[position], lr=0.0))
    frame.render_frame(st, backward=True, grads=image)
    once = position.grad.clone()
    assert bool(once.any())
    position.grad = None
    for t in (1, 2, 3):
        frame.train_frame(st, opt, image)
        # equal gradients: m is (1 - beta1^t) times them, but for the order of the frame's sums
        m = opt.state[position]["exp_avg"]
        assert bool(((m - (1 - 0.9 ** t) * once).abs() <= 1e-4 * once.abs().max()).all()), t


def test_rates_on_the_gpu_are_refused(dev):
    from xsimgs_amd import optim

    x = torch.ones(4, device=dev)
    far = torch.tensor([0.1], device=dev)
    for name in ("lr", "weight_decay"):
        with pytest.raises(ValueError, match=f"{name} must be a number"):
            optim.adam_step_([x], [x.clone()], [x.clone()], [x.clone()], torch.zeros(1, dtype=torch.int64, device=dev),
                             **dict(dict(lr=1e-3), **{name: far}))
        with pytest.raises(ValueError, match=f"{name} must be a number"):
            optim.Adam([torch.nn.Parameter(x)], **{name: far[0]})
    assert bool((x == 1).all())


def _places(t, base):
    """The bytes of base that t's elements lie in, each as often as it has an element there."""
    at = torch.zeros((), dtype=torch.int64)
    for size, stride in zip(t.shape, t.stride()):
        at = at.unsqueeze(-1) + torch.arange(size) * stride
    first = t.data_ptr() - base.data_ptr() + at.reshape(-1) * t.element_size()
    return (first.unsqueeze(-1) + torch.arange(t.element_size())).reshape(-1).tolist()


def test_strided_tensors_that_share_elements_are_refused(dev):
    from xsimgs_amd import optim

    base = torch.ones(40, 30, device=dev)
    flat = base.view(-1)
    for ts in ([base[:, :5], base[:, 4:9]], [base, base[:, 3]], [base[:, 3], base], [base[:, 3:9], base[7, :4]],
               [base[:, ::2].t(), base[5:6, 4]], [base[::2], base.t()[:, 2:3]], [flat[::6], flat[10::4]],
               [flat[1::2], flat.view(torch.int16).view(torch.float16)[3::400]]):
        with pytest.raises(RuntimeError, match="overlap"):
            optim.clip_grads_(ts, 1e-3)
    for t in (flat.as_strided((5, 7), (2, 3)), flat.as_strided((4, 3), (1, 1)), flat.as_strided((3, 3, 2), (10, 0, 1))):
        with pytest.raises(RuntimeError, match="share memory"):
            optim.clip_grads_([flat[1000:], t], 1e-3)
    assert bool((base == 1).all())
    # between each other's elements, in steps of other sizes and with elements of another type
    parts = [flat[::4], flat[2::4], base[:, 1:20:2][::2], base[:, 21::2][1::2],
             base[1::2, 1:20].view(torch.float16)[:, ::4].t()]
    assert optim.clip_grads_(parts, 1e9).isfinite()


def test_strided_tensors_any_way(dev):
    """Small views at random, of one buffer and two element sizes: refused exactly where elements are shared."""
    from xsimgs_amd import optim

    rng, told = random.Random(5), {True: 0, False: 0}
    for _ in range(300):
        base = torch.ones(64, device=dev)
        ts = []
        for _ in range(rng.randint(1, 3)):
            buffer = base if rng.random() < 0.7 else base.view(torch.float16)
            sizes = [rng.randint(1, 4) for _ in range(rng.randint(1, 3))]
            strides = [rng.randint(1, 12) for _ in sizes]
            reach = sum((n - 1) * s for n, s in zip(sizes, strides))
            if reach < buffer.numel():
                ts.append(buffer.as_strided(sizes, strides, rng.randrange(buffer.numel() - reach)))
        if not ts:
            continue
        places = [i for t in ts for i in _places(t, base)]
        shared = len(set(places)) < len(places)
        told[shared] += 1
        if shared:
            with pytest.raises(RuntimeError, match="overlap|share memory"):
                optim.clip_grads_(ts, 1e-3)
            assert bool((base == 1).all())
        else:
            optim.clip_grads_(ts, 1e9)
    assert min(told.values()) > 60, told


@pytest.mark.parametrize("clip", [False, True])
@pytest.mark.parametrize("lists", LISTS)
def test_rate_and_correction_are_rounded_once(dev, lists, clip):
    """Where everything else is exact in float32 (p = 0, m = g = v = 1, eps = 0, beta2 = 1/2 after many steps), a
    step is the corrected rate itself: lr / (1 - beta1^t), rounded to the nearest float32."""
    from xsimgs_amd import optim

    sizes = LISTS[lists]
    g, m, v = ([torch.ones(s, device=dev) for s in sizes] for _ in range(3))
    rng = random.Random(3)
    for _ in range(20 if lists != "many chunks" else 4):
        t, beta1 = rng.randint(60, 200), rng.choice([0.9, 0.95, 0.99])
        rates = [10 ** rng.uniform(-6, -1) for _ in sizes]
        p = [torch.zeros(s, device=dev) for s in sizes]
        step = torch.full((1,), t - 1, dtype=torch.int64, device=dev)
        optim.adam_step_(p, g, m, v, step, lr=rates, betas=(beta1, 0.5), eps=0.0, max_norm=1e9 if clip else None)
        assert all(bool((x == 1).all()) for xs in (m, v) for x in xs)
        for x, lr in zip(p, rates):
            want = torch.tensor(-lr / (1.0 - beta1 ** t), dtype=torch.float64).float()
            assert bool((x.cpu() == want).all()), (lr, beta1, t, float(x.view(-1)[0]), float(want))
