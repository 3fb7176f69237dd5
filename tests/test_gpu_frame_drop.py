"""Frames that drop Gaussians and frames with a feature head: the operators where the framework's own paths call them."""
import dataclasses

import pytest
import torch

from tests import _draws

pytestmark = pytest.mark.gpu


def _scene(kind="cfg0", channels=None, n=2500):
    from xsimgs_amd import synthetic

    if kind == "rig":
        sc = synthetic.make_cfg4(seed=1, n=20_000, n_blobs=60)
        sc = dataclasses.replace(sc, cameras=synthetic.rig_cameras(96, 64, 70.0, 3))
    elif kind == "lidar":
        sc = synthetic.make_cfg3(seed=1, n=20_000, width=128, n_beams=32)
    else:
        sc = synthetic.make_cfg0(seed=3, n=n, width=96, height=64)
    if channels is not None:
        g = torch.Generator().manual_seed(5)
        sc = dataclasses.replace(sc, sh_coeffs=None, colors=torch.rand(sc.n, channels, generator=g))
    return sc


def _image_grads(sc, channels, dev, rig=False, seed=9):
    g = torch.Generator().manual_seed(seed)
    cam = sc.cameras[0]
    lead = (len(sc.cameras),) if rig else ()
    shape = (*lead, cam.height, cam.width)
    return tuple((1e-3 * torch.randn(*shape, *last, generator=g)).to(dev) for last in ((channels,), (), ()))


@pytest.mark.parametrize("kind", ["cfg0", "lidar"])
def test_dropped_gaussians_are_not_there(dev, kind):
    """The frame is that of the scene without them, its opacities divided by the share kept."""
    from xsimgs_amd import frame, rendering

    sc = _scene(kind)
    st = frame.prepare(sc, dev)
    out = frame.render_frame(st, drop=0.3, seed=21)
    keep, factor = _draws.kept(sc.n, 0.3, 21)
    keep = torch.as_tensor(keep).to(dev)
    scales, opac = rendering.activate_gaussians(st.log_scales.detach(), st.opacity_logits.detach(), drop=0.3, seed=21)
    cam, spec = st.cams[0], sc.cameras[0]
    colors = out["colors"].detach()
    rgb, depth, alpha, _ = rendering.ut_gs_render(
        cam, st.means.detach()[keep], scales[keep], st.quats.detach()[keep], opac[keep], spec.width, spec.height,
        colors=colors[keep], tile_size_x=sc.tile_size[0], tile_size_y=sc.tile_size[1], use_phm=sc.use_phm)
    # the same pairs in the same order
    for got, want in ((out["rgb"], rgb), (out["depth"], depth), (out["alpha"], alpha)):
        assert torch.equal(got.detach(), want)
    assert bool((out["radii"][~keep] == 0).all()) and float(out["alpha"].detach().max()) > 0.1
    plain = frame.render_frame(st)
    assert plain["kept"] is None and not torch.equal(plain["rgb"], out["rgb"])
    assert torch.equal(frame.render_frame(st, drop=0.0, seed=21)["rgb"], plain["rgb"])


def test_rig_drops_the_same_gaussians(dev):
    from xsimgs_amd import frame

    sc = _scene("rig")
    st = frame.prepare(sc, dev, requires_grad=False)
    rig = frame.render_rig(st, drop=0.4, seed=5)
    for c in range(len(sc.cameras)):
        one = frame.render_frame(st, cam_index=c, drop=0.4, seed=5)
        assert torch.equal(one["radii"], rig["radii"][c])
        # the rig's colours are the unmasked evaluation's; the images agree as they do without a drop
        assert float((one["rgb"] - rig["rgb"][c]).abs().max()) <= 1e-4
    assert torch.equal(rig["kept"].view(torch.int32), one["kept"].view(torch.int32))


@pytest.mark.parametrize("kind", ["cfg0", "lidar", "rig"])
def test_training_leaves_dropped_gaussians_alone(dev, kind):
    from xsimgs_amd import frame

    sc = _scene(kind)
    st = frame.prepare(sc, dev)
    opt = frame.make_optimizer(st)
    rig = kind == "rig"
    channels = 2 if kind == "lidar" else 3
    names = [k for k in frame.RATES if getattr(st, k) is not None]
    for step in range(3):
        before = {k: getattr(st, k).detach().clone() for k in names}
        avg = {k: opt.state[getattr(st, k)]["exp_avg"].clone() for k in names} if step else {}
        out = frame.train_frame(st, opt, _image_grads(sc, channels, dev, rig, step), rig=rig, drop=0.3, seed=100 + step)
        keep = torch.as_tensor(_draws.kept(sc.n, 0.3, 100 + step)[0]).to(dev)
        for k in names:
            assert bool((out["grads"][k][~keep] == 0).all()), k
            assert torch.equal(getattr(st, k).detach()[~keep], before[k][~keep]), k
            if step:
                assert torch.equal(opt.state[getattr(st, k)]["exp_avg"][~keep], avg[k][~keep]), k
        assert not torch.equal(st.opacity_logits.detach()[keep], before["opacity_logits"][keep])


@pytest.mark.parametrize("rig", [False, True])
def test_a_head_over_the_features(dev, rig):
    """out["features"] is the head of the composited features; gradients reach the scene and the head as they do by
    hand; a training step moves both."""
    from xsimgs_amd import frame, rendering

    channels = 8
    sc = _scene("rig" if rig else "cfg0", channels)
    head = rendering.FeatureNorm(2, channels, drop=0.25)
    st = frame.prepare(sc, dev, head=head)
    assert head.weight.device.type == "cuda"
    render = frame.render_rig if rig else frame.render_frame
    grads = _image_grads(sc, channels, dev, rig)
    out = render(st, backward=True, grads=grads, seed=3)
    x = out["rgb"].detach().requires_grad_()
    y = rendering.group_norm_act(x if rig else x[None], 2, head.weight, head.bias, drop=0.25, seed=3, stream=1)
    assert torch.equal(y.view(out["features"].shape), out["features"])
    # the same image gradient without a head
    g_rgb, g_w, g_b = torch.autograd.grad(y, [x, head.weight, head.bias], grads[0].view(y.shape))
    assert torch.equal(head.weight.grad, g_w) and torch.equal(head.bias.grad, g_b)
    got = {k: v.clone() for k, v in out["grads"].items() if v is not None}
    frame.zero_grads(st)
    st.head = None
    plain = render(st, backward=True, grads=(g_rgb, *grads[1:]))
    assert "features" not in plain
    for k, g in got.items():
        # the compositor's backward adds atomically: equal up to the order of its sums
        assert float((g - plain["grads"][k]).abs().max()) <= 1e-4 * float(g.abs().max()) + 1e-12, k
    st.head = head
    head.weight.grad = head.bias.grad = None
    opt = frame.make_optimizer(st, rates=dict(head=1e-2))
    assert [g["lr"] for g in opt.param_groups if g["name"] == "head"] == [1e-2]
    old = head.weight.detach().clone(), st.colors.detach().clone()
    frame.train_frame(st, opt, grads, rig=rig, drop=0.2, seed=11)
    assert not torch.equal(head.weight.detach(), old[0]) and not torch.equal(st.colors.detach(), old[1])
    assert head.weight.grad is None
    # in evaluation nothing is drawn
    head.eval()
    with torch.no_grad():
        assert torch.equal(render(st)["features"], render(st, seed=77)["features"])


def test_a_head_that_drops_takes_the_steps_seed(dev):
    from xsimgs_amd import frame, rendering

    st = frame.prepare(_scene(channels=4), dev, head=rendering.FeatureNorm(1, 4, drop=0.5))
    a, b, c = (frame.render_frame(st, seed=s)["features"].detach() for s in (1, 1, 2))
    assert torch.equal(a, b) and not torch.equal(a, c)


def test_seed_on_the_gpu(dev):
    from xsimgs_amd import frame

    st = frame.prepare(_scene(), dev, requires_grad=False)
    seed = torch.full((1,), 8, dtype=torch.int64, device=dev)
    assert torch.equal(frame.render_frame(st, drop=0.5, seed=seed)["rgb"], frame.render_frame(st, drop=0.5, seed=8)["rgb"])


def test_operators_in_a_row(dev):
    """What a network does behind a frame: drop the features, norm, mix the channels, norm again; in one go and
    captured in a graph, against the same in 64 bits on the CPU."""
    from tests.test_gpu_features import U, _act
    from xsimgs_amd import rendering

    gen = torch.Generator().manual_seed(2)
    x, m, g = torch.randn(2, 20, 30, 16, generator=gen), 0.3 * torch.randn(16, 24, generator=gen), torch.randn(2, 20, 30, 24, generator=gen)
    leaves = [t.to(dev).requires_grad_() for t in (x, m)]
    v_y = g.to(dev)

    def run(x, m):
        a = rendering.dropout(x, 0.1, 4, stream=0)
        a = rendering.group_norm_act(a, 4, act="silu", drop=0.1, seed=4, stream=1)
        a = rendering.group_norm_act(a @ m, 8, act="gelu", drop=0.2, seed=4, stream=2)
        return a.detach(), torch.autograd.grad(a, [x, m], v_y)

    def norm(a, groups, act, p, stream):
        v = a.view(a.shape[0], -1, groups, a.shape[-1] // groups)
        var, mean = torch.var_mean(v, (1, 3), correction=0, keepdim=True)
        y = _act(((v - mean) / (var + 1e-5).sqrt()).view(a.shape), act)[0]
        keep, f = _draws.kept(a.numel(), p, 4, stream)
        return y * torch.as_tensor(keep).view(a.shape) * f

    wide = [t.double().requires_grad_() for t in (x, m)]
    keep, f = _draws.kept(x.numel(), 0.1, 4, 0)
    y = norm(norm(wide[0] * torch.as_tensor(keep).view(x.shape) * f, 4, "silu", 0.1, 1) @ wide[1], 8, "gelu", 0.2, 2)
    want = torch.autograd.grad(y, wide, g.double())
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        first = run(*leaves)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run(*leaves)
    for _ in range(3):
        graph.replay()
        run(*leaves)
        torch.cuda.synchronize()
        for a, (b, c) in zip((captured[0], *captured[1]), zip((first[0], *first[1]), (y, *want))):
            assert torch.equal(a, b)
            # two norms in a row, each within 400 roundings of what is largest in its sums
            assert float((b.detach().cpu().double() - c.detach()).abs().max()) <= 800 * U * float(c.detach().abs().max())
