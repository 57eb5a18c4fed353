"""GPU: group norm with its activation (forward, backward, double backward), the gradient norm, the
clip and the clipped AdamW step against float64 formulas on the host.

Tolerances.  Group norm: ``_norm_ref.bound`` (256 fp32 roundings of the terms' magnitude and half a
step of the output type; derived there).  Norm of gradients: squares and their sum are float64, so
the result is off by its rounding to fp32 alone, 2^-24 (2^-23 asked).  Clipped values: the factor
and the product are each rounded to fp32 once (2 * 2^-24) and the value to its type."""
import math

import pytest
import torch

from tests._norm_ref import HALF, TINY, close, reference
from tests.test_norm_clip import SHAPES

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops():
    import gan_amd.ops as o
    return o


def make(shape, layout, act, dtype, seed, pdt=F32, scale=2.0, shift=0.5):
    g = torch.Generator().manual_seed(seed)
    C = shape[-1] if layout == "nhwc" else shape[0]
    r = lambda *s: torch.randn(*s, generator=g)   # noqa: E731
    slope = (0.25 + 0.1 * r(C)).to(pdt).to(DEV) if act == "prelu" else 0.2 if act == "leaky" else None
    t = dict(x=(r(*shape) * scale + shift).to(dtype), w=(1 + 0.3 * r(C)).to(pdt), b=(0.3 * r(C)).to(pdt),
             gy=r(*shape).to(dtype), v=r(*shape).to(dtype), cw=r(C).to(pdt), cb=r(C).to(pdt), cs=r(C).to(pdt))
    t = {k: u.to(DEV) for k, u in t.items()}
    t["w"][::3] *= -1
    return {**t, "slope": slope}


def same(a, b):
    """Equal bits, a NaN being equal to a NaN."""
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(), b.nan_to_num())


def run_all(ops, t, G, act, layout, eps=1e-5, params=True, cots=True):
    """Every output of the operator, its backward and its double backward."""
    x, gy = (t[k].detach().requires_grad_() for k in ("x", "gy"))
    w, b = ((t[k].detach().requires_grad_() for k in ("w", "b")) if params else (None, None))
    slope = t["slope"].detach().requires_grad_() if act == "prelu" else t["slope"]
    pars = [p for p in (w, b, slope if act == "prelu" else None) if p is not None]
    y = ops.group_norm_act(x, G, w, b, act=act, slope=slope, eps=eps, layout=layout)
    first = torch.autograd.grad(y, [x, *pars], gy.detach(), retain_graph=True)
    grads = torch.autograd.grad(y, [x, *pars], gy, create_graph=True)
    for a, c in zip(first, grads):
        assert same(a, c)
    cot = [t["v"]] + ([t["cw"], t["cb"]] if params else []) + ([t["cs"]] if act == "prelu" else [])
    if not cots:
        grads, cot = grads[:1], cot[:1]
    second = torch.autograd.grad(grads, [gy, x, *pars], cot, allow_unused=True)
    names = (["w", "b"] if params else []) + (["s"] if act == "prelu" else [])
    out = {"y": y, "gx": first[0], "g_gy": second[0], "g_x": second[1]}
    out.update({"g" + n: u for n, u in zip(names, first[1:])})
    out.update({"g_" + n: u for n, u in zip(names, second[2:])})
    with torch.no_grad():
        assert same(y, ops.group_norm_act(x, G, w, b, act=act, slope=slope, eps=eps, layout=layout))
    return out


def check_all(ops, t, G, act, layout, eps=1e-5, params=True, cots=True):
    got = run_all(ops, t, G, act, layout, eps, params, cots)
    ref = reference(t["x"], G, t["w"] if params else None, t["b"] if params else None, act, t["slope"], eps, layout,
                    t["gy"], t["v"], t["cw"] if params and cots else None, t["cb"] if params and cots else None,
                    t["cs"] if act == "prelu" and cots else None)
    for k, u in got.items():
        close(u, ref[k], k)


KINDS = [(F32, "silu"), (F32, "prelu"), (F32, "none"), (BF16, "leaky"), (BF16, "silu"), (F16, "prelu")]


@pytest.mark.parametrize("shape,G,layout", SHAPES)
@pytest.mark.parametrize("dtype,act", KINDS)
def test_group_norm(ops, shape, G, layout, dtype, act):
    check_all(ops, make(shape, layout, act, dtype, 3), G, act, layout)


@pytest.mark.parametrize("layout", ["nhwc", "cnhw"])
@pytest.mark.parametrize("act", ["silu", "prelu"])
def test_group_norm_without_parameters(ops, layout, act):
    shape = (3, 5, 4, 12) if layout == "nhwc" else (12, 3, 5, 4)
    check_all(ops, make(shape, layout, act, F32, 4), 4, act, layout, params=False)


@pytest.mark.parametrize("layout", ["nhwc", "cnhw"])
@pytest.mark.parametrize("act", ["silu", "leaky", "prelu"])
def test_group_norm_penalty_alone(ops, layout, act):
    """Only the data gradient is differentiated again (the gradient penalty)."""
    shape = (3, 40, 37, 12) if layout == "nhwc" else (12, 3, 40, 37)
    check_all(ops, make(shape, layout, act, F32, 5), 4, act, layout, cots=False)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_group_norm_parameters_of_the_data_type(ops, dtype):
    check_all(ops, make((4, 6, 6, 24), "nhwc", "prelu", dtype, 6, pdt=dtype), 3, "prelu", "nhwc")


@pytest.mark.parametrize("shape,G,layout", [((2, 16, 16, 12), 3, "nhwc"), ((1, 3000, 8), 2, "nhwc"),
                                            ((12, 2, 16, 16), 3, "cnhw"), ((4, 1, 40000), 2, "cnhw")])
def test_group_norm_far_mean(ops, shape, G, layout):
    """Values of spread 1 around 4096: the variance survives (sums in float64)."""
    check_all(ops, make(shape, layout, "silu", F32, 7, scale=1.0, shift=4096.0), G, "silu", layout)


@pytest.mark.parametrize("layout", ["nhwc", "cnhw"])
def test_group_norm_constant_group(ops, layout):
    """A group of one value repeated: variance 0, xh 0, y = act(b); gradients stay finite."""
    shape = (2, 4, 4, 8) if layout == "nhwc" else (8, 2, 4, 4)
    t = make(shape, layout, "silu", F32, 8)
    t["x"].fill_(3.25)
    check_all(ops, t, 2, "silu", layout)


@pytest.mark.parametrize("shape,G,layout", [((3, 5, 5, 8), 2, "nhwc"), ((100, 64, 8), 2, "nhwc"), ((1, 3000, 8), 2, "nhwc"),
                                            ((8, 3, 5, 5), 2, "cnhw"), ((4, 1, 40000), 2, "cnhw")])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_group_norm_nonfinite_stays_in_its_group(ops, shape, G, layout, value):
    t = make(shape, layout, "prelu", F32, 9)
    clean = run_all(ops, t, G, "prelu", layout)
    C = shape[-1] if layout == "nhwc" else shape[0]
    x = t["x"].clone()
    x.view(-1)[0] = value                                     # sample 0, channel 0
    got = run_all(ops, {**t, "x": x}, G, "prelu", layout)
    hit = torch.zeros(shape, dtype=torch.bool, device=DEV)
    if layout == "nhwc":
        hit[0, ..., :C // G] = True
    else:
        hit[:C // G, 0] = True
    for k in ("y", "gx", "g_gy", "g_x"):
        assert bool(torch.isnan(got[k][hit]).all()), k
        assert torch.equal(got[k][~hit], clean[k][~hit]), k
    for k in ("gw", "gs", "g_w"):
        assert torch.equal(got[k][C // G:], clean[k][C // G:]), k


@pytest.mark.parametrize("shape,layout", [((0, 4, 4, 8), "nhwc"), ((3, 0, 8), "nhwc"), ((8, 0, 4), "cnhw")])
def test_group_norm_empty(ops, shape, layout):
    t = make(shape, layout, "silu", F32, 10)
    x, w, b, gy = (t[k].detach().requires_grad_() for k in ("x", "w", "b", "gy"))
    y = ops.group_norm_act(x, 2, w, b, act="silu", layout=layout)
    assert y.shape == x.shape
    gx, gw = torch.autograd.grad(y, [x, w], gy, create_graph=True)
    assert gx.shape == x.shape and not gw.any()
    g = torch.autograd.grad(gx, [gy, x, w], t["v"], allow_unused=True)
    assert g[0].shape == x.shape and not g[2].any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape,G,layout", [((3, 7, 24), 3, "nhwc"), ((1, 3000, 16), 2, "nhwc"), ((12, 3, 37), 3, "cnhw"),
                                            ((4, 1, 40000), 2, "cnhw")])
def test_group_norm_alignment_and_order(ops, dtype, shape, G, layout):
    """Data one element off every alignment, and a map in another memory order: same results."""
    t = make(shape, layout, "silu", dtype, 11)
    want = run_all(ops, t, G, "silu", layout)

    def off(u):
        room = torch.empty(u.numel() + 1, dtype=u.dtype, device=DEV)
        room[1:] = u.reshape(-1)
        return room[1:].view(u.shape)

    got = run_all(ops, {**t, "x": off(t["x"]), "gy": off(t["gy"]), "v": off(t["v"])}, G, "silu", layout)
    turned = run_all(ops, {**t, "x": t["x"].transpose(0, 1).contiguous().transpose(0, 1)}, G, "silu", layout)
    for k in want:
        assert torch.equal(got[k], want[k]) and torch.equal(turned[k], want[k]), k


def test_group_norm_expanded_gradient_and_channels_last(ops):
    t = make((3, 8, 6, 6), "nhwc", "none", F32, 12)                          # an NCHW map here
    x = t["x"].to(memory_format=torch.channels_last).requires_grad_()
    w, b = torch.ones(8, device=DEV), torch.zeros(8, device=DEV)
    y = ops.group_norm_act(x.permute(0, 2, 3, 1), 4, w, b)
    ref = reference(x.detach().permute(0, 2, 3, 1), 4, w, b, "none", None, 1e-5, "nhwc",
                    torch.ones(3, 6, 6, 8))
    close(y, ref["y"], "y")
    y.sum().backward()                                                        # a gradient of stride 0
    close(x.grad.permute(0, 2, 3, 1).contiguous(), ref["gx"], "gx")


def test_group_norm_streams_and_repeats(ops):
    """Other streams, and the same bits every time."""
    for shape, G, layout in (((2, 33, 31, 100), 20, "nhwc"), ((12, 130, 33, 31), 4, "cnhw")):
        t = make(shape, layout, "prelu", F32, 13)
        want = run_all(ops, t, G, "prelu", layout)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = run_all(ops, t, G, "prelu", layout)
        torch.cuda.current_stream().wait_stream(s)
        for k in want:
            assert torch.equal(got[k], want[k]), k


def test_group_norm_many_samples(ops):
    """More samples than one block folds for the parameter gradients; tokens of one position."""
    check_all(ops, make((1300, 24), "nhwc", "prelu", F32, 14), 4, "prelu", "nhwc")
    check_all(ops, make((24, 1300), "cnhw", "silu", F32, 15), 4, "silu", "cnhw")


def test_group_norm_gradient_of_another_type(ops):
    """A float32 cotangent of a bf16 result is taken in the result's type."""
    t = make((3, 6, 5, 16), "nhwc", "silu", BF16, 23)
    x = t["x"].clone().requires_grad_()
    y = ops.group_norm_act(x, 4, t["w"], t["b"], act="silu")
    want = torch.autograd.grad(y, x, t["gy"], retain_graph=True)[0]
    assert torch.equal(torch.autograd.grad(y, x, t["gy"].float())[0], want)


def test_group_norm_one_sided_gradients(ops):
    """Some inputs without a gradient: the others' do not change."""
    t = make((3, 6, 5, 16), "nhwc", "prelu", F32, 16)
    full = run_all(ops, t, 4, "prelu", "nhwc")
    w = t["w"].clone().requires_grad_()
    y = ops.group_norm_act(t["x"], 4, w, t["b"], act="prelu", slope=t["slope"])
    assert torch.equal(torch.autograd.grad(y, w, t["gy"])[0], full["gw"])
    x = t["x"].clone().requires_grad_()
    y = ops.group_norm_act(x, 4, t["w"], t["b"], act="prelu", slope=t["slope"])
    assert torch.equal(torch.autograd.grad(y, x, t["gy"])[0], full["gx"])


class Block(torch.nn.Module):
    """A critic's block in channel rows: conv, group norm + activation, conv to one channel, mean."""

    def __init__(self, cin=3, c=8, act="prelu"):
        super().__init__()
        g = torch.Generator().manual_seed(5)
        par = lambda t: torch.nn.Parameter(t)   # noqa: E731
        self.w0, self.b0 = par(torch.randn(c, cin, 3, 3, generator=g) * 0.4), par(torch.randn(c, generator=g) * 0.1)
        self.gamma, self.beta = par(1 + 0.2 * torch.randn(c, generator=g)), par(0.2 * torch.randn(c, generator=g))
        self.slope = par(0.25 + 0.05 * torch.randn(c, generator=g))
        self.w1, self.b1 = par(torch.randn(1, c, 3, 3, generator=g) * 0.4), par(torch.zeros(1))
        self.act = act

    def forward(self, x, segments=1):
        from gan_amd import ops
        B, C, H, W = x.shape
        t = ops.conv2d(x.permute(1, 0, 2, 3), self.w0, self.b0, ops.conv_geo(B, C, H, W, self.w0.shape[0], 3, 1, 1), 1.0)
        t = ops.group_norm_act(t, 2, self.gamma, self.beta, act=self.act,
                               slope=self.slope if self.act == "prelu" else None, layout="cnhw")
        t = ops.conv2d(t, self.w1, self.b1, ops.conv_geo(B, self.w0.shape[0], H, W, 1, 3, 1, 1), 1.0)
        return t.reshape(B, H * W).mean(1, keepdim=True)

    def plain(self, x, p):
        F = torch.nn.functional
        t = F.conv2d(F.pad(x, (1,) * 4, mode="replicate"), p["w0"], p["b0"])
        B, C = t.shape[:2]
        t = t.reshape(B, 2, -1)
        t = (t - t.mean(2, keepdim=True)) / torch.sqrt(t.var(2, unbiased=False, keepdim=True) + 1e-5)
        t = t.reshape(B, C, *x.shape[2:]) * p["gamma"][:, None, None] + p["beta"][:, None, None]
        t = torch.where(t > 0, t, p["slope"][:, None, None] * t) if self.act == "prelu" else t * torch.sigmoid(t)
        return F.conv2d(F.pad(t, (1,) * 4, mode="replicate"), p["w1"], p["b1"]).reshape(B, -1).mean(1, keepdim=True)


class Toy(torch.nn.Module):
    """A generator for Block: one linear map of z to an image."""

    def __init__(self, z=4):
        super().__init__()
        self.w = torch.nn.Parameter(torch.randn(3 * 64, z, generator=torch.Generator().manual_seed(2)))

    def forward(self, z):
        from gan_amd import ops
        B = z.shape[0]
        t = ops.linear(z.reshape(B, -1).t().contiguous(), self.w, None, 0.5)
        return t.reshape(3, 8, 8, B).permute(3, 0, 1, 2).contiguous()


@pytest.mark.parametrize("act", ["silu", "prelu"])
def test_penalty_step_with_group_norm_and_clip(act):
    """A WGAN-GP critic step as a user runs it: a critic with group norm, the gradient penalty's
    double backward through the trainer, gradients in the flat buffer, the clipped AdamW step --
    against float64 torch.  Bar 1e-4 norm-relative: the convs' of tests/test_ops_gpu.py."""
    import gan_amd
    D = Block(act=act).to(DEV)
    before = {k: p.detach().double().cpu() for k, p in D.named_parameters()}
    rng = gan_amd.DeviceRNG(torch.device(DEV, 0), 11)
    tr = gan_amd.Train([], torch.device(DEV, 0), 1, 4, Toy().to(DEV), "g", D, "d", rng=rng, max_grad_norm=0.05)
    images = torch.randn(6, 3, 8, 8, generator=torch.Generator().manual_seed(9)).to(DEV)
    fake = tr.generate_fake(6)
    seen = {}
    penalty = tr.gradient_penalty

    def watched(real, fk, *a, **k):
        state = rng.state()
        eps = rng.rand((6,)).double().cpu().view(-1, 1, 1, 1)
        rng.set_state(state)
        seen["x"] = (1 - eps) * real.double().cpu() + eps * fk.detach().double().cpu()
        return penalty(real, fk, *a, **k)

    tr.gradient_penalty = watched
    real_loss, fake_loss, gp = tr.discriminator_backward(images, 6, gen_imgs=fake)
    p = {k: v.clone().requires_grad_() for k, v in before.items()}
    xh = seen["x"].requires_grad_()
    r = -D.plain(images.double().cpu(), p).mean()
    f = D.plain(fake.detach().double().cpu(), p).mean()
    (gx,) = torch.autograd.grad(D.plain(xh, p).sum(), xh, create_graph=True)
    pen = 10 * ((gx.reshape(6, -1).norm(dim=1) - 1) ** 2).mean()
    names = [k for k in p if not (act == "silu" and k == "slope")]
    want = dict(zip(names, torch.autograd.grad(r + f + pen, [p[k] for k in names], allow_unused=True)))
    pen = float(pen.detach())
    assert abs(float(gp.detach()) - pen) < 1e-4 * abs(pen)
    assert abs(float(real_loss.detach()) - float(r.detach())) < 1e-4
    assert abs(float(fake_loss.detach()) - float(f.detach())) < 1e-4
    got = {k: q.grad.double().cpu() for k, q in D.named_parameters() if k in want}
    flat = lambda d: torch.cat([torch.zeros(1) if u is None else u.reshape(-1) for u in d.values()])   # noqa: E731
    total = math.sqrt(sum(float(u.square().sum()) for u in want.values() if u is not None))
    for k in names:
        e = (got[k] - (0 if want[k] is None else want[k])).norm()
        assert float(e) < 1e-4 * max(total * 0.1, float(got[k].norm())), (k, float(e))
    # the clipped step from these gradients
    tr.optimizer_D.step()
    assert abs(float(tr.optimizer_D.grad_norm) - total) < 1e-4 * total
    q = {k: torch.nn.Parameter(v.clone()) for k, v in before.items() if k in want}
    opt = torch.optim.AdamW(q.values(), lr=0.0004, betas=(0.5, 0.999))
    for k in q:
        q[k].grad = got[k].clone()
    torch.nn.utils.clip_grad_norm_(q.values(), 0.05)
    opt.step()
    for k, u in D.named_parameters():
        if k in q:
            assert float((u.detach().double().cpu() - q[k].detach()).abs().max()) < 4e-4 * 1e-3 + 2.0 ** -22, k


@pytest.mark.parametrize("shape,G,layout,dtype", [((64, 64, 64, 24), 4, "nhwc", BF16), ((24, 64, 64, 64), 3, "cnhw", F32),
                                                  ((256, 64, 64, 24), 8, "nhwc", F16)])
def test_group_norm_large(ops, shape, G, layout, dtype):
    """Whole batches of full-size maps, up to and beyond the last-level cache: statistics and gradients
    by their sums (the tested quantities are linear or quadratic in the outputs)."""
    t = make(shape, layout, "leaky", dtype, 21)
    x, w, b = (t[k].detach().requires_grad_() for k in ("x", "w", "b"))
    y = ops.group_norm_act(x, G, w, b, act="leaky", slope=0.2, layout=layout)
    gx, gw, gb = torch.autograd.grad(y, [x, w, b], t["gy"])
    xd, gyd = t["x"].double(), t["gy"].double()
    if layout == "cnhw":
        xd, gyd, yd, gxd = (u.permute(1, 2, 3, 0) for u in (xd, gyd, y.double(), gx.double()))
    else:
        yd, gxd = y.double(), gx.double()
    B, C = xd.shape[0], xd.shape[-1]
    grp = lambda u: u.reshape(B, -1, G, C // G)   # noqa: E731
    d = grp(xd) - grp(xd).mean((1, 3), keepdim=True)
    r = 1 / torch.sqrt((d * d).mean((1, 3), keepdim=True) + 1e-5)
    wd, bd = (u.detach().double().reshape(1, 1, G, C // G) for u in (w, b))
    z = d * r * wd + bd
    a1 = torch.where(z > 0, 1.0, 0.2).double()
    half = HALF[dtype]
    err = (grp(yd) - z * a1).abs()
    assert bool((err <= (half + 2.0 ** -16) * ((z - bd).abs() + bd.abs()) + TINY[dtype]).all())
    u = grp(gyd) * a1 * wd
    xh = d * r
    m1, m2 = u.mean((1, 3), keepdim=True), (u * xh).mean((1, 3), keepdim=True)
    ref = r * (u - m1 - xh * m2)
    mag = r * (u.abs() + u.abs().mean((1, 3), keepdim=True) * (1 + xh.abs()))
    assert bool(((grp(gxd) - ref).abs() <= (half + 2.0 ** -16) * mag + TINY[dtype]).all())
    g = grp(gyd) * a1
    for got, want, size in ((gw, g * xh, g.abs() * xh.abs()), (gb, g, g.abs())):
        lim = 2.0 ** -16 * size.sum((0, 1)).reshape(C)
        assert bool(((got.double() - want.sum((0, 1)).reshape(C)).abs() <= lim).all())


MANY_CHUNKS = [((1, 200_000, 8), 2, "nhwc"), ((1, 90_001, 3), 3, "nhwc"), ((2, 1, 1_200_001), 1, "cnhw"),
               ((1, 1, 2_000_000), 1, "cnhw")]


@pytest.mark.parametrize("shape,G,layout", MANY_CHUNKS)
@pytest.mark.parametrize("dtype,act", [(F32, "prelu"), (BF16, "silu")])
def test_group_norm_many_chunks(ops, shape, G, layout, dtype, act):
    """One long sample over so many chunks that they are folded in two steps."""
    import ctypes
    from gan_amd import _lib
    B, C = (shape[0], shape[-1]) if layout == "nhwc" else (shape[1], shape[0])
    d = _lib.NormDesc(math.prod(shape) // (B * C), B, C, G, ("nhwc", "cnhw").index(layout), (F32, BF16).index(dtype), 0,
                      3 if act == "prelu" else 1, 0.0, 1e-5)
    for op in range(3):
        info = (ctypes.c_int * 11)()
        assert _lib.LIB.ganamd_group_norm_plan_info(d, op, info) == 0 and not info[0] and info[7] > 64
    check_all(ops, make(shape, layout, act, dtype, 24), G, act, layout)


@pytest.mark.parametrize("layout", ["nhwc", "cnhw"])
def test_group_norm_offsets_beyond_32_bits(ops, layout):
    """2.2e9 elements: the last sample alone gives the same, to its rounding."""
    B, H, C = 530, 64, 1024
    shape = (B, H, H, C) if layout == "nhwc" else (C, B, H, H)
    x = torch.empty(shape, dtype=BF16, device=DEV).normal_(0.5, 2.0)
    gy = torch.empty(shape, dtype=BF16, device=DEV).normal_()
    w, b = torch.full((C,), 1.25, device=DEV), torch.full((C,), -0.1, device=DEV)
    xl = x.requires_grad_()
    y = ops.group_norm_act(xl, 32, w, b, act="silu", layout=layout)
    (gx,) = torch.autograd.grad(y, xl, gy)
    last = (slice(-1, None),) if layout == "nhwc" else (slice(None), slice(-1, None))
    t = {k: u[last].detach().contiguous() for k, u in (("x", x), ("gy", gy))}
    ref = reference(t["x"], 32, w, b, "silu", None, 1e-5, layout, t["gy"])
    close(y[last].contiguous(), ref["y"], "y")
    close(gx[last].contiguous(), ref["gx"], "gx")


def test_group_norm_samples_beyond_16_bits(ops):
    for shape, layout in (((70_001, 8), "nhwc"), ((8, 70_001), "cnhw")):
        check_all(ops, make(shape, layout, "prelu", F32, 22), 2, "prelu", layout)


def test_two_streams_at_once(ops):
    """Norms and clips on two streams, issued in turn: neither disturbs the other."""
    ts = [make((6, 40, 40, 24), "nhwc", "prelu", F32, 30 + i) for i in range(2)]
    gs = [grads([5, 70_000, 300] * 60, [F32], 40 + i) for i in range(2)]
    want = [run_all(ops, t, 3, "prelu", "nhwc") for t in ts]
    outs = [[torch.empty_like(t) for t in g] for g in gs]
    norms = [ops.clip_grad_norm_(g, 0.01, out=o) for g, o in zip(gs, outs)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got, again, ns = [None] * 2, [[torch.empty_like(t) for t in g] for g in gs], [None] * 2
    torch.cuda.synchronize()
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = run_all_quiet(ops, ts[i])
                ns[i] = ops.clip_grad_norm_(gs[i], 0.01, out=again[i])
    torch.cuda.synchronize()
    for i in range(2):
        for a, k in zip(got[i], ("y", "gx", "gw")):
            assert torch.equal(a, want[i][k])
        assert torch.equal(ns[i], norms[i]) and all(torch.equal(a, b) for a, b in zip(again[i], outs[i]))


def run_all_quiet(ops, t):
    """Forward and backward without a look at the results in between."""
    x, w = (t[k].detach().requires_grad_() for k in ("x", "w"))
    y = ops.group_norm_act(x, 3, w, t["b"], act="prelu", slope=t["slope"])
    return [y, *torch.autograd.grad(y, [x, w], t["gy"])]


def test_clip_offsets_beyond_32_bits(ops):
    t = torch.empty(1_300_000_001, device=DEV).normal_()
    n = float(torch.linalg.vector_norm(t, dtype=torch.float64))
    tail = t[-1000:].clone()
    out = torch.empty_like(t)
    got = ops.clip_grad_norm_([t[:7], t[7:]], 0.5 * n, out=[out[:7], out[7:]])
    assert abs(float(got) - n) <= 2.0 ** -22 * n
    c = 0.5 * n / (n + 1e-6)
    assert bool(((out[-1000:].double() - tail.double() * c).abs() <= tail.double().abs() * 4 * 2.0 ** -24).all())


def test_group_norm_third_derivative_is_refused(ops):
    t = make((2, 4, 8), "nhwc", "silu", F32, 19)
    x, gy = (t[k].detach().requires_grad_() for k in ("x", "gy"))
    y = ops.group_norm_act(x, 2, t["w"], t["b"], act="silu")
    (gx,) = torch.autograd.grad(y, x, gy, create_graph=True)
    (g2,) = torch.autograd.grad(gx, x, t["v"], create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g2.sum().backward()


def test_group_norm_flat_gradients(ops):
    """Gradients of parameters in an optimizer's flat buffer are added there, and only when asked."""
    from gan_amd.optim import FusedAdamW
    D = Block().to(DEV)
    FusedAdamW(D)
    t = make((8, 3, 6, 6), "cnhw", "prelu", F32, 17)
    call = lambda x: ops.group_norm_act(x, 2, D.gamma, D.beta, act="prelu", slope=D.slope, layout="cnhw")   # noqa: E731
    x = t["x"].clone().requires_grad_()
    torch.autograd.grad(call(x), x, t["gy"])
    assert not D._flat.grad.any()
    free = [p.detach().clone().requires_grad_() for p in (D.gamma, D.beta, D.slope)]
    want = torch.autograd.grad(ops.group_norm_act(t["x"], 2, free[0], free[1], act="prelu", slope=free[2], layout="cnhw"),
                               free, t["gy"])
    for _ in range(2):
        call(x).backward(t["gy"])
    for p, g in zip((D.gamma, D.beta, D.slope), want):
        assert torch.equal(p.grad, g + g)
        assert p.grad.data_ptr() >= D._flat.grad.data_ptr()
    # asked for by autograd.grad, they are returned and the buffer stays as it is
    keep = D._flat.grad.clone()
    for p, g, u in zip((D.gamma, D.beta, D.slope), want, torch.autograd.grad(call(t["x"]), (D.gamma, D.beta, D.slope), t["gy"])):
        assert torch.equal(g, u)
    assert torch.equal(keep, D._flat.grad)
    # through the penalty: the second backward adds them to the buffer
    D._flat.grad.zero_()
    (gx,) = torch.autograd.grad(call(x), x, t["gy"], create_graph=True)
    assert not D._flat.grad.any()
    gx.backward(t["v"])
    y = ops.group_norm_act(x, 2, free[0], free[1], act="prelu", slope=free[2], layout="cnhw")
    (gx,) = torch.autograd.grad(y, x, t["gy"], create_graph=True)
    for p, g in zip((D.gamma, D.slope), torch.autograd.grad(gx, (free[0], free[2]), t["v"])):
        assert torch.equal(p.grad, g)


def test_group_norm_one_parameter_in_two_places(ops):
    """A parameter of a flat buffer that is weight and bias at once: the sum of both gradients arrives."""
    from gan_amd.optim import FusedAdamW
    D = Block().to(DEV)
    FusedAdamW(D)
    t = make((8, 3, 6, 6), "cnhw", "silu", F32, 18)
    free = [D.gamma.detach().clone().requires_grad_() for _ in range(2)]
    for order in (1, 2):
        D._flat.grad.zero_()
        got = []
        for w, b in ((D.gamma, D.gamma), free):
            x = t["x"].clone().requires_grad_()
            y = ops.group_norm_act(x, 2, w, b, act="silu", layout="cnhw")
            if order == 2:
                (gx,) = torch.autograd.grad(y, x, t["gy"], create_graph=True)
                y, up = gx, t["v"]
            else:
                up = t["gy"]
            if w is b:
                y.backward(up)
            else:
                got = torch.autograd.grad(y, free, up)
        assert torch.equal(D.gamma.grad, got[0] + got[1])
        assert D.gamma.grad.data_ptr() >= D._flat.grad.data_ptr()


def test_group_norm_backward_that_leaves_a_capture_is_refused(ops):
    """A captured backward into leaves that an eager graph of the default stream holds is refused before
    it runs; once that graph is gone, it is captured and replays."""
    from gan_amd._lib import HOST
    t = make((4, 8, 5, 5), "cnhw", "silu", F32, 19)
    x = t["x"].clone().requires_grad_()
    w, b = (t[k].detach().clone().requires_grad_() for k in "wb")
    call = lambda: ops.group_norm_act(x, 2, w, b, act="silu", layout="cnhw")   # noqa: E731
    want = torch.autograd.grad(call(), (x, w, b), t["gy"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = call()
        assert not HOST.crosses(y)
        del y
    eager = call()
    assert not HOST.crosses(eager)
    with torch.cuda.stream(side):
        y = call()
        assert HOST.crosses(y)
        for u, v in zip(torch.autograd.grad(y, (x, w, b), t["gy"]), want):      # no capture: no refusal
            assert torch.equal(u, v)
        del y
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = call()
        assert HOST.crosses(y)
        for again in (False, True):
            with pytest.raises(RuntimeError, match="capture"):
                torch.autograd.grad(y, (x, w, b), t["gy"], create_graph=again, retain_graph=True)
        kept = t["gy"] * 2
        del y
    del eager
    torch.cuda.synchronize()
    other = torch.cuda.CUDAGraph()
    with torch.cuda.graph(other):
        y = call()
        assert not HOST.crosses(y)
        got = torch.autograd.grad(y, (x, w, b), t["gy"])
        del y
    for _ in range(3):
        for g in got:
            g.fill_(float("nan"))
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        assert torch.equal(kept, t["gy"] * 2) and all(torch.equal(g, u) for g, u in zip(got, want))


def test_group_norm_graph(ops):
    """Forward, backward and double backward captured; replays with eager work between them."""
    for shape, G, layout in (((2, 9, 9, 12), 3, "nhwc"), ((1, 3000, 8), 2, "nhwc"), ((12, 2, 37), 3, "cnhw")):
        t = make(shape, layout, "prelu", F32, 18)
        warm = torch.cuda.Stream()
        warm.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(warm):
            run_all(ops, t, G, "prelu", layout)
        torch.cuda.current_stream().wait_stream(warm)
        torch.cuda.synchronize()

        def step():
            x, gy, w, b, s = (t[k].detach().requires_grad_() for k in ("x", "gy", "w", "b", "slope"))
            y = ops.group_norm_act(x, G, w, b, act="prelu", slope=s, layout=layout)
            g = torch.autograd.grad(y, [x, w, b, s], gy, create_graph=True)
            return [y, *g, *torch.autograd.grad(g[0], [gy, x, w, s], t["v"])]

        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        for i in range(3):
            t["x"].copy_(make(shape, layout, "prelu", F32, 20 + i)["x"])
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(outs, step()):
                assert torch.equal(a, b)


# ------------------------------------------------------------------ norm, clip, step

def grads(sizes, dtypes, seed, scale=1e-2):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * scale * 10 ** float(torch.randn((), generator=g))).to(dtypes[i % len(dtypes)]).to(DEV)
            for i, n in enumerate(sizes)]


def norm64(ts):
    return math.sqrt(sum(float(t.double().square().sum()) for t in ts))


LISTS = [([1], [F32]), ([7], [BF16]), ([0, 5, 0, 4097], [F32]), ([4096, 4095, 1, 8193], [F16, BF16, F32]),
         ([3] * 161, [F32]), (list(range(1, 500)), [F32, BF16]), ([1_000_003], [F32]), ([9_000_001, 17, 70_000], [BF16]),
         ([300_000] * 40, [F32, F16])]


@pytest.mark.parametrize("sizes,dtypes", LISTS)
@pytest.mark.parametrize("to", ["place", "same", "f32"])
def test_clip(ops, sizes, dtypes, to):
    ts = grads(sizes, dtypes, 1)
    n = norm64(ts)
    for t in ts:                                           # ragged starts: views one element in
        assert t.is_contiguous()
    assert abs(float(ops.grad_norm(ts)) - n) <= 2.0 ** -23 * n
    for most in (0.37 * n, 4 * n):
        c = min(1.0, most / (n + 1e-6))
        src = [t.clone() for t in ts]
        out = None if to == "place" else [torch.empty_like(t, dtype=t.dtype if to == "same" else F32) for t in ts]
        got = ops.clip_grad_norm_(src, most, out=out)
        assert got.dim() == 0 and got.dtype == F32 and abs(float(got) - n) <= 2.0 ** -23 * n
        for s, t, o in zip(src, ts, src if out is None else out):
            if out is not None:
                assert torch.equal(s, t)
            want = t.double() * c
            lim = want.abs() * (2 * 2.0 ** -24 * 1.01 + HALF[o.dtype]) + TINY[o.dtype]
            assert bool(((o.double() - want).abs() <= lim).all())
            if c == 1.0:
                assert torch.equal(o.double(), t.double())


def test_clip_views_of_a_buffer(ops):
    """Views that start anywhere in a buffer; what lies between them stays as it was."""
    for dt in (F32, BF16, F16):
        buf = torch.randn(50_000, device=DEV).to(dt)
        keep = buf.clone()
        spans = [(1, 2), (3, 700), (705, 4802), (4803, 4803), (9001, 49_999)]
        views = [buf[a:b] for a, b in spans]
        n = norm64(views)
        ops.clip_grad_norm_(views, 0.5 * n)
        mask = torch.zeros(50_000, dtype=torch.bool, device=DEV)
        for a, b in spans:
            mask[a:b] = True
        assert torch.equal(buf[~mask], keep[~mask])
        assert abs(norm64(views) - 0.5 * n) < 0.5 * n * (2.0 ** -9 if dt != F32 else 2.0 ** -20)


def test_clip_orders_and_infinity_norm(ops):
    base = torch.randn(6, 5, 4, 3, device=DEV)
    ts = [base.to(memory_format=torch.channels_last), torch.randn(31, 7, device=DEV).t(), torch.tensor(3.0, device=DEV)]
    want = max(float(t.abs().max()) for t in ts)
    assert float(ops.grad_norm(ts, float("inf"))) == want
    n = norm64(ts)
    ref = [t.double() * (1.0 / (n + 1e-6)) for t in ts]
    ops.clip_grad_norm_(ts, 1.0)
    for t, r in zip(ts, ref):
        assert bool(((t.double() - r).abs() <= r.abs() * 3 * 2.0 ** -24 * 1.01).all())
    ts = grads([5, 70_000], [F32], 3)
    m = max(float(t.abs().max()) for t in ts)
    ref = [t.double() * (0.5 * m / (m + 1e-6)) for t in ts]
    assert float(ops.clip_grad_norm_(ts, 0.5 * m, norm_type=float("inf"))) == m
    for t, r in zip(ts, ref):
        assert bool(((t.double() - r).abs() <= r.abs() * 3 * 2.0 ** -24 * 1.01).all())


def test_norm_range(ops):
    """Squares neither overflow nor vanish; zeros and nothing at all have norm 0."""
    big = torch.full((3, 1000), 1e25, device=DEV)
    small = torch.full((5000,), 1e-30, device=DEV)
    assert abs(float(ops.grad_norm([big])) / (1e25 * math.sqrt(3000)) - 1) < 2.0 ** -22
    assert abs(float(ops.grad_norm([small])) / (1e-30 * math.sqrt(5000)) - 1) < 2.0 ** -22
    assert float(ops.grad_norm([])) == 0 and float(ops.grad_norm([torch.zeros(0, device=DEV)])) == 0
    assert float(ops.clip_grad_norm_([], 1.0)) == 0
    z = torch.zeros(5, device=DEV)
    assert float(ops.clip_grad_norm_([z], 1.0)) == 0 and not z.any()
    t = torch.ones(4, device=DEV)
    ops.clip_grad_norm_([t], 0.0)
    assert not t.any()


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("kind", [2.0, float("inf")])
@pytest.mark.parametrize("n", [50, 5_000_000])
def test_clip_nonfinite(ops, value, kind, n):
    from gan_amd._lib import GanAmdError
    ts = grads([n, 9], [F32], 4)
    ts[0][n // 2] = value
    got = float(ops.grad_norm(ts, kind))
    assert got != got if value != value else got == value
    with pytest.raises(GanAmdError):
        ops.clip_grad_norm_([t.clone() for t in ts], 1.0, kind, error_if_nonfinite=True)
    ops.clip_grad_norm_(ts, 1.0, kind)
    if value != value:
        assert all(bool(torch.isnan(t).all()) for t in ts)
    else:                                                    # times 0: 0, and NaN at the infinity
        assert not ts[1].any() and bool(torch.isnan(ts[0][n // 2])) and int(torch.isnan(ts[0]).sum()) == 1


def test_clip_refuses_on_the_gpu(ops):
    from gan_amd._lib import GanAmdError
    t = torch.randn(8, 6, device=DEV)
    leaf = torch.randn(3, device=DEV, requires_grad=True)
    keep = t.clone()
    for f in (lambda: ops.clip_grad_norm_([t, t], 1.0), lambda: ops.clip_grad_norm_([t[:5], t[4:]], 1.0),
              lambda: ops.clip_grad_norm_([t[:, :3]], 1.0), lambda: ops.grad_norm([t[:, ::2]]),
              lambda: ops.clip_grad_norm_([t.expand(2, 8, 6)], 1.0), lambda: ops.clip_grad_norm_([leaf], 1.0),
              lambda: ops.clip_grad_norm_([t], 1.0, out=[]), lambda: ops.clip_grad_norm_([t], 1.0, out=[t[:4]]),
              lambda: ops.clip_grad_norm_([t], 1.0, out=[t.half()]), lambda: ops.grad_norm([t.double()]),
              lambda: ops.grad_norm([t, torch.zeros(2)]), lambda: ops.clip_grad_norm_([t.t()], 1.0, out=[torch.empty(6, 8, device=DEV)])):
        with pytest.raises(GanAmdError):
            f()
    assert torch.equal(t, keep)
    b = [torch.randn(8, device=DEV) for _ in range(4)]
    step = torch.zeros(1, dtype=torch.int32, device=DEV)
    with pytest.raises(GanAmdError):
        ops.clipped_adamw_(b[0], b[0], b[2], b[3], step, 1e-3, (0.9, 0.999), 1e-8, 0.0, 1.0)
    assert int(step) == 0


def adamw64(p, g, m, v, t, lr, betas, eps, wd, most):
    n = float(g.square().sum().sqrt())
    g = g * min(1.0, most / (n + 1e-6))
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    step = lr * (m / (1 - betas[0] ** t)) / ((v / (1 - betas[1] ** t)).sqrt() + eps)
    return p * (1 - lr * wd) - step, m, v, n, step


@pytest.mark.parametrize("n", [1, 3, 4, 4099, 65_537, 5_000_002])
@pytest.mark.parametrize("clipped", [True, False])
def test_clipped_adamw(ops, n, clipped):
    """Three steps against float64.  Every value is rounded fewer than 16 times a step."""
    g = torch.Generator().manual_seed(n)
    r = lambda: torch.randn(n, generator=g)   # noqa: E731
    p, m, v = r().to(DEV), (r() * 1e-2).to(DEV), (r() * 1e-2).square().to(DEV)
    step = torch.full((1,), 7, dtype=torch.int32, device=DEV)
    lr, betas, eps, wd = 4e-4, (0.5, 0.999), 1e-8, 0.01
    ref = [t.double() for t in (p, m, v)]
    for t in range(8, 11):
        gr = (r() * 2e-2).to(DEV)
        keep = gr.clone()
        full = float(gr.double().norm())
        most = (0.3 if clipped else 3.0) * full
        norm = ops.clipped_adamw_(p, gr, m, v, step, lr, betas, eps, wd, most)
        *ref, want, size = adamw64(*ref[:1], gr.double(), *ref[1:], t, lr, betas, eps, wd, most)
        assert int(step) == t and torch.equal(gr, keep) and abs(float(norm) - want) <= 2.0 ** -23 * want
        u = 16 * (t - 7) * 2.0 ** -24
        assert bool(((p.double() - ref[0]).abs() <= u * (ref[0].abs() + size.abs() + lr)).all())
        assert bool(((m.double() - ref[1]).abs() <= u * (ref[1].abs() + gr.double().abs() + 1e-2)).all())
        assert bool(((v.double() - ref[2]).abs() <= u * ref[2].abs() + 1e-30).all())


def test_clipped_adamw_agrees_with_the_plain_step(ops):
    """Under a limit that does not bind, the step is FusedAdamW's own; offset buffers too."""
    from gan_amd.optim import FusedAdamW
    a, b = (torch.nn.Linear(37, 29).to(DEV) for _ in range(2))
    b.load_state_dict(a.state_dict())
    oa, ob = FusedAdamW(a), FusedAdamW(b, max_grad_norm=1e9)
    for i in range(3):
        g = torch.randn(oa.flat.n_train, generator=torch.Generator().manual_seed(i)).to(DEV)
        oa.flat.grad.copy_(g)
        ob.flat.grad.copy_(g)
        oa.step()
        ob.step()
    assert abs(float(ob.grad_norm) - float(g.double().norm())) < 1e-5
    assert float((oa.flat.data - ob.flat.data).abs().max()) <= 4 * 2.0 ** -24
    room = [torch.randn(1002, device=DEV) for _ in range(4)]
    room[3].abs_()
    want = [t[1:].clone() for t in room]
    step = [torch.zeros(1, dtype=torch.int32, device=DEV) for _ in range(2)]
    k = (1e-3, (0.9, 0.999), 1e-8, 0.01, 2.0)
    ops.clipped_adamw_(*want, step[0], *k)
    edge = [t[:1].clone() for t in room]
    ops.clipped_adamw_(*[t[1:] for t in room], step[1], *k)
    for w, t, e in zip(want, room, edge):
        assert torch.equal(w, t[1:]) and torch.equal(t[:1], e)


def test_clip_and_step_graph(ops):
    """Captured clips and steps replay on new gradients; two graphs at once keep to their own scratch."""
    from gan_amd._lib import GanAmdError
    ts = grads([5, 70_000, 300], [F32, BF16], 5)
    outs = [torch.empty_like(t, dtype=F32) for t in ts]
    p, m, v, g = (torch.randn(30_001, device=DEV) for _ in range(4))
    v.abs_()
    step = torch.zeros(1, dtype=torch.int32, device=DEV)
    k = (1e-3, (0.9, 0.999), 1e-8, 0.01, 1.0)
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        ops.clip_grad_norm_(ts, 0.01, out=outs)
    torch.cuda.current_stream().wait_stream(warm)
    torch.cuda.synchronize()
    ga, gb = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(ga):
        with pytest.raises(GanAmdError):
            ops.clip_grad_norm_(ts, 0.01, out=outs, error_if_nonfinite=True)
        na = ops.clip_grad_norm_(ts, 0.01, out=outs)
    with torch.cuda.graph(gb):
        nb = ops.clipped_adamw_(p, g, m, v, step, *k)
    for i in range(3):
        for t, u in zip(ts, grads([5, 70_000, 300], [F32, BF16], 6 + i)):
            t.copy_(u)
        g.copy_(torch.randn(30_001, generator=torch.Generator().manual_seed(i)).to(DEV))
        state = [u.clone() for u in (p, m, v, step)]
        ga.replay()
        gb.replay()
        torch.cuda.synchronize()
        want = [torch.empty_like(o) for o in outs]
        assert torch.equal(ops.clip_grad_norm_(ts, 0.01, out=want), na)
        assert all(torch.equal(a, b) for a, b in zip(want, outs))
        n = ops.clipped_adamw_(state[0], g, state[1], state[2], state[3], *k)
        assert torch.equal(n, nb) and all(torch.equal(a, b) for a, b in zip(state, (p, m, v, step)))


def test_clip_counts_as_a_write(ops):
    """A tensor that autograd saved and the clip scaled is noticed."""
    t = torch.randn(50, device=DEV)
    w = torch.randn(50, device=DEV, requires_grad=True)
    y = (w * t).sum()
    ops.clip_grad_norm_([t], 0.1)
    with pytest.raises(RuntimeError, match="modified"):
        y.backward()


def test_clipped_adamw_counts_as_a_write(ops):
    """A convolution after a step on its weight uses the new weight, not the packed copy of the old."""
    w = torch.nn.Parameter(torch.randn(8, 8, 3, 3, generator=torch.Generator().manual_seed(1)).to(DEV))
    x = torch.randn(8, 2, 16, 16, generator=torch.Generator().manual_seed(2)).to(DEV)
    geo = ops.conv_geo(2, 8, 16, 16, 8, 3, 1, 1)
    conv = lambda w: ops.conv2d(x, w, None, geo, 1.0)   # noqa: E731
    old = conv(w).detach()
    step = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.clipped_adamw_(w.detach(), torch.ones_like(w), torch.zeros_like(w), torch.zeros_like(w), step, 0.1, (0.9, 0.99),
                       1e-8, 0.0, 1.0)
    new = conv(w).detach()
    assert not torch.equal(old, new)
    assert torch.equal(new, conv(torch.nn.Parameter(w.detach().clone())).detach())


def test_clipped_adamw_refuses_overlaps(ops):
    from gan_amd._lib import GanAmdError
    p, g, m, v = (torch.ones(64, device=DEV) for _ in range(4))
    step = torch.zeros(1, dtype=torch.int32, device=DEV)
    k = (1e-3, (0.9, 0.999), 1e-8, 0.01, 1.0)
    for bad in (dict(norm=p[3]), dict(norm=g[63:]), dict(norm=step.view(F32)), dict(step=v[5:6].view(torch.int32))):
        with pytest.raises(GanAmdError):
            ops.clipped_adamw_(p, g, m, v, bad.get("step", step), *k, norm=bad.get("norm"))
    assert int(step) == 0 and all(bool((t == 1).all()) for t in (p, g, m, v))


def test_optimizer_step_graph(ops):
    """FusedAdamW(max_grad_norm) captured and replayed; the norm is the replay's."""
    from gan_amd.optim import FusedAdamW
    a, b = (torch.nn.Linear(53, 31).to(DEV) for _ in range(2))
    b.load_state_dict(a.state_dict())
    oa, ob = FusedAdamW(a, max_grad_norm=0.5), FusedAdamW(b, max_grad_norm=0.5)
    g = [torch.randn(oa.flat.n_train, generator=torch.Generator().manual_seed(i)).to(DEV) for i in range(4)]
    for o in (oa, ob):                       # one eager step each, on a side stream
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            o.flat.grad.copy_(g[0])
            o.step()
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ob.step()
    for i in range(1, 4):
        oa.flat.grad.copy_(g[i])
        ob.flat.grad.copy_(g[i])
        oa.step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(oa.flat.data, ob.flat.data) and torch.equal(oa.grad_norm, ob.grad_norm)
        assert abs(float(ob.grad_norm) - float(g[i].double().norm())) <= 2.0 ** -23 * float(g[i].double().norm())
        assert int(ob.step_count) == i + 1


def test_clip_other_stream_and_repeats(ops):
    ts = grads([123_457, 9, 40_000], [F32, F16], 7)
    a, b = ([torch.empty_like(t) for t in ts] for _ in range(2))
    n = ops.clip_grad_norm_(ts, 0.02, out=a)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        k = ops.clip_grad_norm_(ts, 0.02, out=b)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(n, k) and all(torch.equal(x, y) for x, y in zip(a, b))


def test_forward_mode_is_refused_on_the_gpu(ops):
    import torch.autograd.forward_ad as fwad
    from gan_amd._lib import GanAmdError
    t = make((2, 4, 4, 8), "nhwc", "prelu", F32, 33)
    with fwad.dual_level():
        dual = lambda u: fwad.make_dual(u, torch.ones_like(u))   # noqa: E731
        for k in ("x", "w", "b", "slope"):
            a = {**t, k: dual(t[k])}
            with pytest.raises(GanAmdError, match="tangent"):
                ops.group_norm_act(a["x"], 2, a["w"], a["b"], act="prelu", slope=a["slope"])
        for f in (ops.grad_norm, lambda u: ops.clip_grad_norm_(u, 1.0)):
            with pytest.raises(GanAmdError, match="tangent"):
                f([t["x"], dual(t["gy"])])


def flat_case(ops, seed, act="prelu"):
    """A Block with its flat buffer, data, the call, and what one backward adds to the norm's parameters."""
    from gan_amd.optim import FusedAdamW
    D = Block(act=act).to(DEV)
    FusedAdamW(D)
    t = make((8, 3, 6, 6), "cnhw", act, F32, seed)
    pars = (D.gamma, D.beta, D.slope)
    call = lambda x: ops.group_norm_act(x, 2, D.gamma, D.beta, act=act, slope=D.slope, layout="cnhw")   # noqa: E731
    free = [p.detach().clone().requires_grad_() for p in pars]
    y = ops.group_norm_act(t["x"], 2, free[0], free[1], act=act, slope=free[2], layout="cnhw")
    want = torch.autograd.grad(y, free, t["gy"])
    torch.cuda.synchronize()
    return D, t, pars, call, want


def sleep():
    torch.cuda._sleep(20_000_000)       # about 10 ms: what does not wait for this stream is seen


def test_group_norm_flat_gradients_of_two_streams(ops):
    """One module on the default and on a side stream, one backward: both gradients arrive, and the
    caller's stream waits for them."""
    D, t, pars, call, want = flat_case(ops, 34)
    side = torch.cuda.Stream()
    for late in (0, 1):
        for first in (0, 1):                       # which stream makes the accumulators
            D._flat.grad.zero_()
            side.wait_stream(torch.cuda.current_stream())
            ys = [None, None]
            for i in (first, 1 - first):
                with torch.cuda.stream(side) if i else torch.cuda.stream(torch.cuda.current_stream()):
                    ys[i] = call(t["x"])
            with torch.cuda.stream(side) if late else torch.cuda.stream(torch.cuda.current_stream()):
                sleep()
            torch.autograd.backward(ys, [t["gy"], t["gy"]])
            got = [p.grad.clone() for p in pars]
            del ys
            for g, w in zip(got, want):
                assert torch.equal(g, w + w)
            assert all(p.grad.data_ptr() >= D._flat.grad.data_ptr() for p in pars)


@pytest.mark.parametrize("order", [1, 2])
def test_group_norm_flat_gradients_beside_a_living_graph(ops, order):
    """The parameters' accumulators are those of an eager graph of the default stream; the call runs on
    a side stream and x needs no gradient: the caller's stream still waits for the side stream's add."""
    D, t, pars, call, want = flat_case(ops, 35)
    older = call(t["x"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x = t["x"].clone().requires_grad_(order == 2)
        y, up = call(x), t["gy"]
        if order == 2:
            (y,), up = torch.autograd.grad(y, x, t["gy"], create_graph=True), t["v"]
        sleep()
    y.backward(up, inputs=list(pars))
    got = [p.grad.clone() for p in pars]
    torch.cuda.synchronize()
    del older, y
    if order == 2:
        x = t["x"].clone().requires_grad_()
        D._flat.grad.zero_()
        (gx,) = torch.autograd.grad(call(x), x, t["gy"], create_graph=True)
        gx.backward(t["v"], inputs=list(pars))
        want = [p.grad.clone() for p in pars]
    for g, w in zip(got, want):
        assert torch.equal(g, w)


def test_group_norm_flat_gradients_of_a_side_stream(ops):
    """All on one side stream: added by the kernel there, and the caller's stream waits for it."""
    D, t, pars, call, want = flat_case(ops, 36)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = call(t["x"])
        sleep()
    y.backward(t["gy"])
    for p, w in zip(pars, want):
        assert torch.equal(p.grad.clone(), w)


def test_group_norm_flat_gradients_captured(ops):
    """A captured backward adds to the flat buffer on every replay; beside a living eager graph of the
    default stream, whose accumulators no capture can reach, it is refused."""
    D, t, pars, call, want = flat_case(ops, 37)
    D._flat.grad.zero_()
    older = call(t["x"])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="capture"):
            call(t["x"]).backward(t["gy"])
    del older
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(t["x"]).backward(t["gy"])
    torch.cuda.synchronize()
    assert not D._flat.grad.any()
    total = [torch.zeros_like(w) for w in want]
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        total = [a + w for a, w in zip(total, want)]
        for p, a in zip(pars, total):
            assert torch.equal(p.grad, a)


def test_clipped_adamw_on_a_flat_buffer_counts_as_a_write(ops):
    """A convolution of a parameter in an optimizer's flat buffer, after the buffer itself was updated
    (by the op or by torch), uses the new weight; the optimizer's own step leaves its copies valid."""
    from gan_amd.optim import FusedAdamW
    D = Block().to(DEV)
    opt = FusedAdamW(D, max_grad_norm=1.0)
    f, n = opt.flat, opt.flat.n_train
    x = torch.randn(3, 2, 16, 16, generator=torch.Generator().manual_seed(2)).to(DEV)
    geo = ops.conv_geo(2, 3, 16, 16, 8, 3, 1, 1)
    conv = lambda w: ops.conv2d(x, w, None, geo, 1.0).detach()   # noqa: E731
    fresh = lambda: conv(torch.nn.Parameter(D.w0.detach().clone()))   # noqa: E731
    step, norm = torch.zeros(1, dtype=torch.int32, device=DEV), torch.zeros((), device=DEV)
    m, v = torch.zeros(n, device=DEV), torch.zeros(n, device=DEV)
    old = conv(D.w0)
    assert f.packs.entries
    for write in (lambda: ops.clipped_adamw_(f.data[:n], torch.ones(n, device=DEV), m, v, step, 0.1, (0.9, 0.99), 1e-8,
                                             0.0, 1.0, norm=norm), lambda: f.data.mul_(0.5)):
        write()
        assert not all(f.packs.valid(e) for e in f.packs.entries.values())
        new = conv(D.w0)
        assert not torch.equal(old, new) and torch.equal(new, fresh())
        assert torch.equal(conv(D.w0), new) and all(f.packs.valid(e) for e in f.packs.entries.values())
        old = new
    assert step._version and norm._version
    f.grad.fill_(0.01)
    opt.step()
    assert all(f.packs.valid(e) for e in f.packs.entries.values())
    assert not torch.equal(conv(D.w0), old) and torch.equal(conv(D.w0), fresh())


def test_optimizer_step_with_numbers_of_any_kind(ops):
    import numpy as np
    from gan_amd.optim import FusedAdamW
    got = []
    for num in (float, np.float32, torch.tensor):
        m = torch.nn.Linear(5, 3).to(DEV)
        with torch.no_grad():
            for p in m.parameters():
                p.fill_(0.5)
        o = FusedAdamW(m, lr=num(0.25), betas=(num(0.5), num(0.75)), eps=num(2.0 ** -20), weight_decay=num(0.125),
                       max_grad_norm=num(0.5))
        o.flat.grad.fill_(1.0)
        o.step()
        got.append(o.flat.data.clone())
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


@pytest.mark.parametrize("dtypes", [[F32], [BF16], [F16], [F32, BF16, F16]])
@pytest.mark.parametrize("to", ["place", "same", "f32"])
def test_clip_misaligned(ops, dtypes, to):
    """Gradients and outputs that start one, two and three elements into their buffers, each output
    elsewhere than its gradient; what surrounds the outputs stays."""
    sizes = [1, 2, 9, 255, 4096, 8191, 30_001]
    ts = grads(sizes, dtypes, 8)
    n = norm64(ts)
    c = 0.37 * n / (n + 1e-6)

    def off(t, k, dt=None):
        room = torch.full((t.numel() + 8,), 7.0, dtype=dt or t.dtype, device=DEV)
        view = room[k:k + t.numel()]
        if dt is None:
            view.copy_(t)
        return room, view

    src = [off(t, 1 + i % 3) for i, t in enumerate(ts)]
    dst = src if to == "place" else [off(t, 1 + (i + 1) % 3, t.dtype if to == "same" else F32) for i, t in enumerate(ts)]
    got = ops.clip_grad_norm_([v for _, v in src], 0.37 * n, out=None if to == "place" else [v for _, v in dst])
    assert abs(float(got) - n) <= 2.0 ** -23 * n
    for t, (room, o), (_, s) in zip(ts, dst, src):
        want = t.double() * c
        lim = want.abs() * (2 * 2.0 ** -24 * 1.01 + HALF[o.dtype]) + TINY[o.dtype]
        assert bool(((o.double() - want).abs() <= lim).all())
        at = o.storage_offset()
        assert bool((room[:at] == 7).all()) and bool((room[at + t.numel():] == 7).all())
        assert to == "place" or torch.equal(s, t)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_clip_permuted_in_place(ops, dtype):
    """Tensors of other memory orders, scaled in place and into outputs of their own strides."""
    g = torch.Generator().manual_seed(9)
    make_ = lambda *s: torch.randn(*s, generator=g).to(dtype).to(DEV)   # noqa: E731
    for out in (False, True):
        ts = [make_(6, 5, 4, 3).to(memory_format=torch.channels_last), make_(31, 7).t(), make_(9, 8, 7).permute(2, 0, 1),
              make_(33, 1, 5).transpose(0, 1)]
        ref = [t.double() for t in ts]
        n = norm64(ts)
        c = 0.5 * n / (n + 1e-6)
        dst = [torch.empty_like(t) for t in ts] if out else ts
        ops.clip_grad_norm_(ts, 0.5 * n, out=dst if out else None)
        for o, r, t in zip(dst, ref, ts):
            assert o.stride() == t.stride()
            lim = (r * c).abs() * (2 * 2.0 ** -24 * 1.01 + HALF[dtype]) + TINY[dtype]
            assert bool(((o.double() - r * c).abs() <= lim).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("value", [1e4, -3e5, 1e6, 1e8])
@pytest.mark.parametrize("shape,G,layout", [((2, 9, 9, 12), 2, "nhwc"), ((1, 3000, 8), 2, "nhwc"), ((2, 40, 37, 12), 3, "nhwc"),
                                            ((12, 2, 9, 9), 2, "cnhw"), ((4, 1, 40000), 2, "cnhw")])
def test_group_norm_large_constant_group(ops, shape, G, layout, dtype, value):
    """A group of one large value repeated has variance 0, not the rounding of its square."""
    t = make(shape, layout, "silu", dtype, 8)
    t["x"].fill_(value)
    check_all(ops, t, G, "silu", layout)


@pytest.mark.parametrize("shape,G,layout", [((2, 16, 16, 12), 3, "nhwc"), ((1, 3000, 8), 2, "nhwc"), ((2, 40, 37, 12), 3, "nhwc"),
                                            ((12, 2, 16, 16), 3, "cnhw"), ((4, 1, 40000), 2, "cnhw")])
def test_group_norm_very_far_mean(ops, shape, G, layout):
    """Values of spread 1 around 3e6, where fp32 steps by a quarter."""
    check_all(ops, make(shape, layout, "silu", F32, 7, scale=1.0, shift=3e6), G, "silu", layout)


@pytest.mark.parametrize("order", [1, 2])
def test_group_norm_flat_gradients_with_hooks(ops, order):
    """Gradient hooks of parameters in the flat buffer run, and what they return is what arrives there."""
    D, t, pars, call, want = flat_case(ops, 38)

    def back():
        D._flat.grad.zero_()
        x = t["x"].clone().requires_grad_()
        if order == 1:
            call(x).backward(t["gy"])
        else:
            (gx,) = torch.autograd.grad(call(x), x, t["gy"], create_graph=True)
            gx.backward(t["v"], inputs=list(pars))
        return [p.grad.clone() for p in pars]

    plain = back()
    if order == 1:
        assert all(torch.equal(a, b) for a, b in zip(plain, want))
    seen = []
    handles = [D.gamma.register_hook(lambda g: g * 2), D.slope.register_post_accumulate_grad_hook(lambda p: seen.append(p))]
    got = back()
    assert torch.equal(got[0], plain[0] * 2) and torch.equal(got[1], plain[1]) and torch.equal(got[2], plain[2])
    assert len(seen) == 1 and seen[0] is D.slope
    for h in handles:
        h.remove()
    assert all(torch.equal(a, b) for a, b in zip(back(), plain)) and len(seen) == 1


@pytest.mark.parametrize("shape,G,layout", [((3, 5, 5, 12), 3, "nhwc"), ((64, 40, 37, 12), 4, "nhwc"), ((1, 200_000, 8), 2, "nhwc"),
                                            ((2, 9, 4100), 4, "nhwc"), ((12, 3, 37), 3, "cnhw"), ((4, 1, 40_000), 2, "cnhw")])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_group_norm_forward_in_place_abi(ops, shape, G, layout, dtype):
    """The C entry point with y = x."""
    from gan_amd import _lib
    t = make(shape, layout, "silu", dtype, 39)
    want = ops.group_norm_act(t["x"], G, t["w"], t["b"], act="silu", layout=layout)
    B, C = (shape[0], shape[-1]) if layout == "nhwc" else (shape[1], shape[0])
    d = _lib.NormDesc(math.prod(shape) // (B * C), B, C, G, ("nhwc", "cnhw").index(layout), (F32, BF16).index(dtype), 0, 1, 0.0, 1e-5)
    n = _lib.c_size_t(0)
    assert _lib.LIB.ganamd_group_norm_workspace(d, 0, n) == 0
    ws = torch.empty(n.value // 4 + 1, device=DEV)
    stats = torch.empty(B, G, 2, dtype=torch.float64, device=DEV)
    x = t["x"].clone()
    assert _lib.LIB.ganamd_group_norm_fwd(d, x.data_ptr(), t["w"].data_ptr(), t["b"].data_ptr(), None, x.data_ptr(),
                                          stats.data_ptr(), ws.data_ptr(), ws.numel() * 4, _lib.stream()) == 0
    assert torch.equal(x, want)
