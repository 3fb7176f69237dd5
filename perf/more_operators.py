"""Operators on either side of the compositor: group norm with an activation over rendered feature images
(channels last), and dropout from a counter-based generator, of a tensor's elements or rows and of a scene's
Gaussians.

A case is an operator on what this framework's users hold:

* ``norm``   ``group_norm_act`` on images ``[batch, height, width, channels]`` as the compositor writes them: ``train``
  forward and backward, else forward alone; ``view`` takes all channels but the last of a wider image (a strided
  view); ``valid`` is the share of pixels that hold something, given as a mask (a lidar's rays without a return hold
  NaN); ``drop`` adds dropout behind the activation
* ``drop``   ``dropout`` of a tensor, forward and backward; ``shared`` trailing dimensions share one draw
* ``gauss``  a training frame's activations with a share of the Gaussians dropped, forward and backward, and the
  packed mask of those kept, which the tiling takes

A value e of a draw with probability p is dropped where its 32 bits are below T = round(p 2^32). The upper 16 of
them are half e % 2 of word e % 8 / 2 (lower half first) of Philox4x32-10 (Salmon et al., "Parallel random numbers: as
easy as 1, 2, 3", 2011) with the seed's two words as key and the counter (two words of e / 8, stream, 0); the lower 16
are the same half and word under the counter (.., .., stream, 1). What is kept is divided by 1 - T / 2^32.

Plain form (``own`` false): elementary torch operations in 32 bits, rounded once.
"""
import math

import torch

own = False
DEV = "cuda"
EPS = 1e-5
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # a 16 x 16 patch of a 32-channel feature image around the viewer's cursor: the smallest call, latency
        dict(name="norm_patch", op="norm", batch=1, height=16, width=16, channels=32, groups=8, act="silu",
             type="float32"),
        # the viewer's feature image, half precision, forward alone
        dict(name="norm_view", op="norm", batch=1, height=600, width=800, channels=32, groups=8, act="silu",
             type="float16"),
        # training on a 1080p image of 64 features: forward and backward of the decoder's first norm
        dict(name="norm_1080p", op="norm", batch=1, height=1080, width=1920, channels=64, groups=8, act="silu",
             type="bfloat16", train=True),
        # a spinning lidar's range image, rays without a return masked, an odd number of features, with dropout
        dict(name="norm_lidar", op="norm", batch=1, height=128, width=2048, channels=65, groups=5, act="gelu",
             type="float32", valid=0.8, drop=0.1, train=True),
        # two cameras' widest features at an eighth of 1080p: 512 of 513 channels, the last holds something else
        dict(name="norm_wide", op="norm", batch=2, height=135, width=240, channels=512, groups=32, act="gelu",
             type="float32", view=True, train=True),
        # a decoder's block on a rig's features at a quarter: many groups, dropout, half precision
        dict(name="norm_block", op="norm", batch=6, height=225, width=400, channels=128, groups=32, act="silu",
             type="float16", drop=0.2, train=True),
        # a whole rig's 900p feature images, forward alone: the largest call
        dict(name="norm_rig", op="norm", batch=6, height=900, width=1600, channels=32, groups=4, act="silu",
             type="bfloat16"),
        # six cameras' appearance codes: latency
        dict(name="drop_codes", op="drop", shape="6 48", shared=0, drop=0.1, type="float32"),
        # the 1080p feature image in front of its decoder
        dict(name="drop_1080p", op="drop", shape="1080 1920 64", shared=0, drop=0.1, type="bfloat16"),
        # the SH coefficients of a million Gaussians, whole Gaussians at a time
        dict(name="drop_sh", op="drop", shape="1000000 16 3", shared=2, drop=0.25, type="float32"),
        # the viewer's small scene in training
        dict(name="gauss_view", op="gauss", n=10_000, drop=0.1),
        # a rig's scene, an odd number of Gaussians
        dict(name="gauss_rig", op="gauss", n=4_000_001, drop=0.2),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm", "norm", "drop", "drop", "gauss"])
    drop = rng.choice([round(rng.uniform(0.01, 0.6), 4), 0.5, 0.1])
    if op == "gauss":
        return dict(op=op, n=_log(rng, 1_000, 4_000_000), drop=drop)
    kind = rng.choice(list(TYPES))
    if op == "drop":
        n = _log(rng, 100, 130_000_000 if kind != "float32" else 60_000_000)
        inner = rng.choice([[], [3], [rng.randint(2, 70)], [rng.choice([1, 4, 9, 16]), 3]])
        return dict(op=op, shape=" ".join(map(str, [max(1, n // math.prod(inner)), *inner])), shared=rng.randint(0, len(inner)), drop=drop,
                    type=kind)
    channels = rng.choice([2, 3, 4, 8, 9, 16, 17, 32, 33, 64, 65, 128, 129, 256, 512, 513, rng.randint(2, 640)])
    groups = rng.choice([g for g in range(1, channels + 1) if channels % g == 0 and g <= 64])
    train = rng.random() < 0.6
    batch = rng.choice([1, 1, 2, 6, rng.randint(1, 12)])
    most = 250_000_000 if kind != "float32" else 120_000_000
    pixels = _log(rng, 40, max(80, most // (channels * batch * (2 if train else 1))))
    height = max(1, int(math.sqrt(pixels * rng.uniform(0.2, 1.0))))
    case = dict(op=op, batch=batch, height=height, width=max(1, min(pixels // height, 4096)), channels=channels,
                groups=groups, act=rng.choice(["silu", "silu", "gelu", "none"]), type=kind)
    if train:
        case["train"] = True
    if rng.random() < 0.25:
        case["view"] = True
    if rng.random() < 0.3:
        case["valid"] = round(rng.uniform(0.2, 0.95), 3)
    if rng.random() < 0.4:
        case["drop"] = drop
    return case


def _shape(case):
    return [int(n) for n in case["shape"].split()]


def _size(case):
    return 4 if case["type"] == "float32" else 2


def work(case):
    """Bytes: the inputs read once and the outputs written once (of pixels out of a mask, and of dropped rows,
    nothing is read); training reads x and the outputs' gradient and writes y and x's. Operations: about ten a value forward and
    sixteen backward for the norm with its activation, twenty for a draw of random bits."""
    if case["op"] == "gauss":
        n = case["n"]
        return {"bytes": n * (16 + 16 + 16 + 16) + n / 8, "flops": n * (4 * 12 + 20)}
    bits = 20 if case.get("drop") else 0
    if case["op"] == "drop":
        e = math.prod(_shape(case))
        draws = math.prod(_shape(case)[:len(_shape(case)) - case["shared"]])
        read = 1.0 - case["drop"] if case["shared"] else 1.0
        return {"bytes": 2 * e * _size(case) * (1 + read), "flops": 2 * (e + bits * draws)}
    pixels = case["batch"] * case["height"] * case["width"]
    e, read = pixels * case["channels"], case.get("valid", 1.0)
    mask = pixels if "valid" in case else 0
    times = 2 if case.get("train") else 1
    return {"bytes": times * (e * _size(case) * (1 + read) + mask) + (16 if case.get("train") else 8) * case["channels"],
            "flops": e * read * ((26 if case.get("train") else 10) + times * bits)}


# ---------------------------------------------------------------------------------------------- inputs
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _image(g, case, channels):
    """A feature image: per channel an offset and a spread of its own, smooth structure and noise on top; part
    of it background, which the compositor leaves at zero."""
    b, h, w = case["batch"], case["height"], case["width"]
    offset, spread = 0.5 * _randn(g, channels), torch.exp(0.5 * _randn(g, channels))
    across = torch.linspace(0.0, 6.0, w, device=DEV).view(1, 1, w, 1) + torch.linspace(0.0, 4.0, h, device=DEV).view(1, h, 1, 1)
    out = torch.empty(b, h, w, channels, dtype=TYPES[case["type"]], device=DEV)
    for i in range(b):
        x = _randn(g, 1, h, w, channels)
        x.add_(torch.sin(across + i)).mul_(spread).add_(offset)
        x.mul_(torch.rand(1, h, w, 1, generator=g, device=DEV) > 0.1)
        out[i] = x[0]
    return out


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    state = dict(case=case, seed=1 + 1_000_003 * int(seed), stream=int(seed) % 7)
    if case["op"] == "gauss":
        n = case["n"]
        state["inputs"] = [(-3.0 + 0.7 * _randn(g, n, 3)).requires_grad_(), (1.5 * _randn(g, n)).requires_grad_()]
        state["grads"] = [1e-3 * _randn(g, n, 3), 1e-3 * _randn(g, n)]
        return state
    kind = TYPES[case["type"]]
    if case["op"] == "drop":
        state["x"] = _randn(g, *_shape(case)).to(kind).requires_grad_()
        state["grad"] = (1e-2 * _randn(g, *_shape(case))).to(kind)
        return state
    c = case["channels"]
    x = _image(g, case, c + 1 if case.get("view") else c)
    if case.get("view"):
        x = x[..., :c]
    state["mask"] = None
    if "valid" in case:
        keep = torch.rand(x.shape[:-1], generator=g, device=DEV) < case["valid"]
        x.masked_fill_(~keep.unsqueeze(-1), math.nan)
        state["mask"] = keep
    train = bool(case.get("train"))
    state["x"] = x.detach().requires_grad_(train)
    state["weight"] = (1.0 + 0.2 * _randn(g, c)).requires_grad_(train)
    state["bias"] = (0.2 * _randn(g, c)).requires_grad_(train)
    if train:
        grad = torch.empty(x.shape, dtype=kind, device=DEV)
        for i in range(case["batch"]):
            grad[i] = 1e-2 * _randn(g, *x.shape[1:])
        state["grad"] = grad
    return state


# ------------------------------------------------------------------------------------------------- run
def run(state):
    op = state["case"]["op"]
    if op == "gauss":
        return (_own_gauss if own else _plain_gauss)(state)
    if op == "drop":
        return (_own_drop if own else _plain_drop)(state)
    return (_own_norm if own else _plain_norm)(state)


def _own_gauss(state):
    from xsimgs_amd import rendering

    case, inputs = state["case"], state["inputs"]
    draw_of = dict(drop=case["drop"], seed=state["seed"], stream=state["stream"])
    scales, opacities = rendering.activate_gaussians(*inputs, **draw_of)
    kept = rendering.drop_mask(case["n"], **draw_of, device=DEV)
    grads = torch.autograd.grad([scales, opacities], inputs, state["grads"])
    return dict(scales=scales.detach(), opacities=opacities.detach(), kept=kept.view(torch.int32), v_log_scales=grads[0],
                v_logits=grads[1])


def _own_drop(state):
    from xsimgs_amd import rendering

    case, x = state["case"], state["x"]
    y = rendering.dropout(x, case["drop"], state["seed"], stream=state["stream"], shared=case["shared"])
    return dict(y=y.detach(), v_x=torch.autograd.grad(y, x, state["grad"])[0])


def _own_norm(state):
    from xsimgs_amd import rendering

    case, x = state["case"], state["x"]
    leaves = [x, state["weight"], state["bias"]]
    y = rendering.group_norm_act(x, case["groups"], *leaves[1:], act=case["act"], eps=EPS, mask=state["mask"],
                                 drop=case.get("drop", 0.0), seed=state["seed"], stream=state["stream"])
    if not case.get("train"):
        return dict(y=y)
    grads = torch.autograd.grad(y, leaves, state["grad"])
    return dict(y=y.detach(), v_x=grads[0], v_weight=grads[1], v_bias=grads[2])


# ----------------------------------------------------------------------------------------- plain form
LOW = 0xFFFFFFFF


def _philox(c0, c1, c2, c3, seed):
    """Philox4x32-10 on int64 tensors of 32-bit words (the products' lower 64 bits are exact)."""
    k0, k1 = seed & LOW, (seed >> 32) & LOW
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & LOW) ^ c1 ^ k0, b & LOW, ((a >> 32) & LOW) ^ c3 ^ k1, a & LOW
        k0, k1 = (k0 + 0x9E3779B9) & LOW, (k1 + 0xBB67AE85) & LOW
    return torch.stack([c0, c1, c2, c3], 1)


def _kept(n, case, state):
    """Which of n draws are kept, and the factor of what is."""
    t = round(case["drop"] * 2.0 ** 32)
    block = torch.arange((n + 7) // 8, dtype=torch.int64, device=DEV)
    zero = torch.zeros_like(block)
    upper, lower = (_philox(block & LOW, block >> 32, zero + state["stream"], zero + i, state["seed"]) for i in (0, 1))
    half = torch.tensor([0, 16], device=DEV)
    bits = ((upper.unsqueeze(2) >> half) & 0xFFFF) << 16 | ((lower.unsqueeze(2) >> half) & 0xFFFF)
    return bits.view(-1)[:n] >= t, 1.0 / (1.0 - t / 2.0 ** 32)


def _plain_gauss(state):
    case = state["case"]
    kept, factor = _kept(case["n"], case, state)
    log_scales, logits = (x.detach() for x in state["inputs"])
    v_scales, v_opacities = state["grads"]
    scales, s = torch.exp(log_scales), 1.0 / (1.0 + torch.exp(-logits))
    bits = torch.zeros((case["n"] + 31) // 32 * 32, dtype=torch.int64, device=DEV)
    bits[:case["n"]] = kept
    words = (bits.view(-1, 32) << torch.arange(32, device=DEV)).sum(1)
    return dict(scales=scales, opacities=torch.where(kept, s * factor, 0.0), kept=words.to(torch.int32),
                v_log_scales=v_scales * scales, v_logits=torch.where(kept, v_opacities * factor * s * (1.0 - s), 0.0))


def _plain_drop(state):
    case, x = state["case"], state["x"].detach()
    lead = x.shape[:x.dim() - case["shared"]]
    kept, factor = _kept(math.prod(lead), case, state)
    kept = kept.view(*lead, *[1] * case["shared"])
    return {k: torch.where(kept, t.float() * factor, 0.0).to(t.dtype) for k, t in (("y", x), ("v_x", state["grad"]))}


def _act(z, act):
    """act(z) and its derivative."""
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return z * s, s * (1.0 + z * (1.0 - s))
    if act == "gelu":
        phi = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    return z, torch.ones_like(z)


def _plain_norm(state):
    case, x = state["case"], state["x"].detach()
    b, c, g = x.shape[0], case["channels"], case["groups"]
    pixels = x.shape[1] * x.shape[2]
    keep = torch.ones(b, pixels, 1, 1, dtype=torch.bool, device=DEV) if state["mask"] is None else state["mask"].view(b, pixels, 1, 1)
    n = torch.clamp(keep.sum(1, keepdim=True) * (c // g), min=1)
    grouped = torch.where(keep, x.reshape(b, pixels, g, c // g).float(), 0.0)

    def total(t, dims, keepdim=True):   # long sums in 64 bits
        return t.sum(dims, keepdim=keepdim, dtype=torch.float64)

    mean = (total(grouped, (1, 3)) / n).float()
    xh = torch.where(keep, grouped - mean, 0.0)
    rstd = (1.0 / torch.sqrt(total(xh.square(), (1, 3)) / n + EPS)).float()
    xh = xh * rstd
    weight, bias = (state[k].detach().view(g, c // g) for k in ("weight", "bias"))
    y, slope = _act(xh * weight + bias, case["act"])
    if case.get("drop"):
        kept, factor = _kept(x.numel(), case, state)
        scale = kept.view(y.shape) * factor
        y, slope = y * scale, slope * scale
    out = dict(y=torch.where(keep, y, 0.0).to(x.dtype).view(x.shape))
    if not case.get("train"):
        return out
    dz = torch.where(keep, state["grad"].view(b, pixels, g, c // g).float() * slope, 0.0)
    out["v_weight"], out["v_bias"] = (total(t, (0, 1), False).float().view(c) for t in (dz * xh, dz))
    dxh = dz * weight
    means = [(total(t, (1, 3)) / n).float() for t in (dxh, dxh * xh)]
    dx = rstd * (dxh - means[0] - xh * means[1])
    out["v_x"] = torch.where(keep, dx, 0.0).to(x.dtype).view(x.shape)
    return out


# --------------------------------------------------------------------------------------------- 64 bits
def _multiplied(x, m):
    """Upper and lower 32 bits of x m, by halves of 16 bits."""
    xl, xh, ml, mh = x & 0xFFFF, x >> 16, m & 0xFFFF, m >> 16
    low, mid1, mid2 = xl * ml, xh * ml, xl * mh
    mid = (low >> 16) + (mid1 & 0xFFFF) + (mid2 & 0xFFFF)
    return xh * mh + (mid1 >> 16) + (mid2 >> 16) + (mid >> 16), ((mid & 0xFFFF) << 16) | (low & 0xFFFF)


def _words(block, stream, last, seed):
    """The four output words of the numbered blocks, a round at a time in place."""
    w = [block % 2 ** 32, block // 2 ** 32, torch.full_like(block, stream), torch.full_like(block, last)]
    for r in range(10):
        key = [(seed % 2 ** 32 + r * 0x9E3779B9) % 2 ** 32, (seed // 2 ** 32 + r * 0xBB67AE85) % 2 ** 32]
        h0, l0 = _multiplied(w[0], 0xD2511F53)
        h2, l2 = _multiplied(w[2], 0xCD9E8D57)
        w = [h2 ^ w[1] ^ key[0], l2, h0 ^ w[3] ^ key[1], l0]
    return w


def _factors(n, drop, seed, stream):
    """float64 factors of n draws: 0 of what is dropped."""
    t = int(math.floor(drop * 2 ** 32 + 0.5))
    block = torch.arange(-(-n // 8), device=DEV)
    first, second = _words(block, stream, 0, seed), _words(block, stream, 1, seed)
    u = torch.empty(block.numel(), 8, dtype=torch.int64, device=DEV)
    for j in range(8):
        shift = 65536 if j % 2 else 1
        u[:, j] = (first[j // 2] // shift % 65536) * 65536 + second[j // 2] // shift % 65536
    return (u.view(-1)[:n] >= t).double() * (2.0 ** 32 / (2.0 ** 32 - t))


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "gauss":
        f = _factors(case["n"], case["drop"], s["seed"], s["stream"])
        a, o = (x.detach().double().requires_grad_() for x in s["inputs"])
        scales, opacities = a.exp(), torch.sigmoid(o) * f
        grads = torch.autograd.grad([scales, opacities], [a, o], [g.double() for g in s["grads"]])
        return dict(scales=scales.detach(), opacities=opacities.detach(), kept=None, v_log_scales=grads[0], v_logits=grads[1])
    if case["op"] == "drop":
        lead = _shape(case)[:len(_shape(case)) - case["shared"]]
        f = _factors(math.prod(lead), case["drop"], s["seed"], s["stream"]).view(*lead, *[1] * case["shared"])
        return dict(y=s["x"].detach().double() * f, v_x=s["grad"].double() * f)
    b, c, g = case["batch"], case["channels"], case["groups"]
    weight, bias = (s[k].detach().double().requires_grad_() for k in ("weight", "bias"))
    f = _factors(s["x"].numel(), case["drop"], s["seed"], s["stream"]).view(s["x"].shape) if case.get("drop") else None
    acts = dict(silu=torch.nn.functional.silu, gelu=torch.nn.functional.gelu, none=lambda z: z)
    ys, dxs, dws, dbs = [], [], [], []
    for i in range(b):
        # the pixels in the mask alone, as one sample of a list of pixels
        rows = slice(None) if s["mask"] is None else s["mask"][i].view(-1).nonzero().view(-1)
        flat = s["x"][i].detach().reshape(-1, c).double()
        x = flat[rows].clone().requires_grad_()
        y, dx = torch.zeros_like(flat), torch.zeros_like(flat)
        parts = x.view(-1, g, c // g)
        if x.numel():
            var, mean = torch.var_mean(parts, (0, 2), correction=0, keepdim=True)
            z = ((parts - mean) / (var + EPS).sqrt()).reshape(-1, c) * weight + bias
            out = acts[case["act"]](z)
            if f is not None:
                out = out * f[i].view(-1, c)[rows]
            y[rows] = out.detach()
            if case.get("train"):
                grads = torch.autograd.grad(out, [x, weight, bias], s["grad"][i].view(-1, c)[rows].double())
                dx[rows] = grads[0]
                dws.append(grads[1])
                dbs.append(grads[2])
        ys.append(y.view(s["x"].shape[1:]))
        dxs.append(dx.view(s["x"].shape[1:]))
    if not case.get("train"):
        return dict(y=torch.stack(ys))
    zero = torch.zeros(c, dtype=torch.float64, device=DEV)
    return dict(y=torch.stack(ys), v_x=torch.stack(dxs), v_weight=sum(dws, zero), v_bias=sum(dbs, zero))
