"""CPU: the formulas the group norm kernels are tested against (float64 autograd, differences), the
launch plans (every element owned once, every access in bounds), and the refusals of the
normalisation and clipping operators."""
import ctypes
import math

import pytest
import torch

from tests._norm_ref import reference

ACTS = ["none", "silu", "leaky", "prelu"]


def plain(x, G, w, b, act, slope, eps, layout):
    """Differentiable float64 group norm + activation."""
    if layout == "cnhw":
        C, B = x.shape[:2]
        xr = x.reshape(G, C // G, B, -1)
        shape = (G, C // G, 1, 1)
    else:
        B, C = x.shape[0], x.shape[-1]
        xr = x.reshape(B, -1, G, C // G)
        shape = (1, 1, G, C // G)
    d = xr - xr.mean((1, 3), keepdim=True)
    z = d / torch.sqrt((d * d).mean((1, 3), keepdim=True) + eps) * w.reshape(shape) + b.reshape(shape)
    if act == "silu":
        z = z * torch.sigmoid(z)
    elif act != "none":
        k = slope.reshape(shape) if act == "prelu" else slope
        z = torch.where(z > 0, z, k * z)
    return z.reshape(x.shape)


def case(shape, layout, act, seed):
    g = torch.Generator().manual_seed(seed)
    C = shape[-1] if layout == "nhwc" else shape[0]
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)   # noqa: E731
    slope = (0.25 + 0.1 * r(C)) if act == "prelu" else 0.2 if act == "leaky" else None
    return r(*shape) * 2 + 0.5, 1 + 0.3 * r(C), 0.3 * r(C), slope, r(*shape), r(*shape), r(C), r(C), r(C)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape,G,layout", [((2, 3, 2, 6), 3, "nhwc"), ((6, 2, 5), 2, "cnhw"), ((3, 4), 1, "nhwc")])
def test_formulas_match_autograd(shape, G, layout, act):
    x, w, b, slope, gy, v, cw, cb, cs = case(shape, layout, act, 1)
    leaves = [t.clone().requires_grad_() for t in (x, w, b, gy)]
    xl, wl, bl, gyl = leaves
    sl = slope.clone().requires_grad_() if act == "prelu" else slope
    y = plain(xl, G, wl, bl, act, sl, 1e-5, layout)
    pars = [xl, wl, bl] + ([sl] if act == "prelu" else [])
    grads = torch.autograd.grad(y, pars, gyl, create_graph=True)
    cots = [v, cw, cb] + ([cs] if act == "prelu" else [])
    second = torch.autograd.grad(grads, [gyl] + pars, cots, allow_unused=True)
    ref = reference(x, G, w, b, act, slope, 1e-5, layout, gy, v, cw, cb, cs if act == "prelu" else None)
    got = dict(zip(["y", "gx", "gw", "gb", "gs"], [y, *grads]))
    got.update(zip(["g_gy", "g_x", "g_w", "g_b", "g_s"], second))
    for name, t in got.items():
        t = torch.zeros_like(ref[name][0]) if t is None else t
        assert torch.allclose(t.reshape(ref[name][0].shape), ref[name][0], rtol=1e-10, atol=1e-10), name


@pytest.mark.parametrize("act", ["silu", "prelu"])
def test_formulas_match_differences(act):
    x, w, b, slope, gy, v, *_ = case((2, 3, 4), "nhwc", act, 2)
    ref = reference(x, 2, w, b, act, slope, 1e-5, "nhwc", gy, v)

    def value(x, w, b, gy, which):
        r = reference(x, 2, w, b, act, slope, 1e-5, "nhwc", gy)
        return float((r["y"][0] * gy).sum()) if which == 1 else float((r["gx"][0] * v).sum())

    h = 1e-6
    for which, names in ((1, ("gx", "gw", "gb")), (2, ("g_x", "g_w", "g_b"))):
        for name, t, arg in zip(names, (x, w, b), range(3)):
            for i in range(0, t.numel(), 5):
                e = torch.zeros(t.numel(), dtype=torch.float64)
                e[i] = h
                e = e.reshape(t.shape)
                args = [x, w, b]
                lo, hi = list(args), list(args)
                lo[arg], hi[arg] = t - e, t + e
                diff = (value(*hi, gy, which) - value(*lo, gy, which)) / (2 * h)
                assert abs(diff - float(ref[name][0].reshape(-1)[i])) < 1e-6, (name, i)


# ------------------------------------------------------------------ plans

def plan(shape, G, dtype, act, layout, op):
    from gan_amd import _lib
    B, C = (shape[0], shape[-1]) if layout == "nhwc" else (shape[1], shape[0])
    d = _lib.NormDesc(math.prod(shape) // (B * C), B, C, G, ("nhwc", "cnhw").index(layout),
                      (torch.float32, torch.bfloat16, torch.float16).index(dtype), 0, ACTS.index(act), 0.2, 1e-5)
    info, n = (ctypes.c_int * 11)(), _lib.c_size_t(0)
    assert _lib.LIB.ganamd_group_norm_plan_info(d, op, info) == 0
    assert _lib.LIB.ganamd_group_norm_workspace(d, op, n) == 0
    keys = ("resident", "V", "nt", "TX", "P", "CT", "nct", "S", "per", "SA", "perA")
    return dict(zip(keys, info)), n.value


SHAPES = [((1, 4, 4, 128), 8, "nhwc"), ((3, 5, 3), 1, "nhwc"), ((3, 7, 5), 5, "nhwc"), ((2, 9, 13), 13, "nhwc"),
          ((2, 4, 4, 1025), 5, "nhwc"), ((2, 3, 1025), 1025, "nhwc"), ((2, 3000, 8), 2, "nhwc"),
          ((1, 700, 100), 20, "nhwc"), ((2, 2, 4100), 4, "nhwc"), ((1, 1, 9000), 1, "nhwc"), ((5, 6), 3, "nhwc"),
          ((200, 33, 31, 12), 4, "nhwc"), ((1, 64, 64, 96), 32, "nhwc"), ((2, 6, 9), 9, "nhwc"),
          ((130, 16, 16, 36), 12, "nhwc"), ((1, 1, 1), 1, "nhwc"),
          ((6, 2, 5), 3, "cnhw"), ((8, 3), 2, "cnhw"), ((1025, 3, 4, 4), 1, "cnhw"), ((1025, 2, 4, 4), 1025, "cnhw"),
          ((16, 2, 1023), 4, "cnhw"), ((4, 1, 40000), 2, "cnhw"), ((48, 4, 64, 64), 8, "cnhw"), ((3, 2, 3), 3, "cnhw"),
          ((12, 130, 33, 31), 4, "cnhw"), ((600, 2, 2), 1, "cnhw"), ((1, 1, 1), 1, "cnhw"), ((7, 600, 64), 7, "cnhw")]


@pytest.mark.parametrize("shape,G,layout", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_plan_owns_every_element_once(shape, G, layout, dtype):
    """The kernels' index arithmetic, restated: loads lie inside the tensor, and the elements that
    count (not the moved-back front of a row's or plane's last vector) are each owned once."""
    B, C = (shape[0], shape[-1]) if layout == "nhwc" else (shape[1], shape[0])
    L = math.prod(shape) // (B * C)
    for op in range(3):
        for act in ("silu", "prelu"):
            p, _ = plan(shape, G, dtype, act, layout, op)
            V, P, CT = p["V"], p["P"], p["CT"]
            assert p["nt"] % 64 == 0 and p["nt"] <= 1024 and p["TX"] * P <= p["nt"]
            rows = layout == "nhwc"
            npos = L if rows else -(-L // V)
            if p["resident"]:
                assert CT % (C // G) == 0
                assert -(-npos // P) <= (8 if op == 2 or (op == 1 and not rows) else 16)
            else:
                for S, per in ((p["S"], p["per"]), (p["SA"], p["perA"])):
                    spans = [(s * per, min(npos, (s + 1) * per)) for s in range(S)]
                    assert spans[0][0] == 0 and spans[-1][1] == npos
                    assert all(a < b for a, b in spans) and all(x[1] == y[0] for x, y in zip(spans, spans[1:]))
            if not rows:
                assert P & (P - 1) == 0
            assert (p["nct"] - 1) * CT < C <= p["nct"] * CT
            # channels (rows) / positions (planes) owned by the vectors of a tile / plane
            own = []
            if rows:
                for t in range(p["nct"]):
                    c0, wid = t * CT, min(CT, C - t * CT)
                    for tx in range(p["TX"]):
                        cv = c0 + tx * V
                        if tx * V >= wid:
                            continue
                        ch = max(min(cv, c0 + wid - V), 0)
                        assert 0 <= ch and ch + V <= C and 0 <= cv - ch < V
                        assert ch + V <= c0 + wid          # nothing of the next tile is stored
                        own += range(cv, ch + V)
                assert own == list(range(C))
            else:
                for i in range(npos):
                    at = min(i * V, L - V)
                    assert 0 <= at and at + V <= L and 0 <= i * V - at < V
                    own += range(i * V, at + V)
                assert own == list(range(L))


# ------------------------------------------------------------------ refusals

def test_group_norm_refusals():
    from gan_amd import _lib, ops
    x = torch.zeros(2, 3, 3, 8)
    w = torch.ones(8)
    for kw in (dict(groups=3), dict(groups=0), dict(groups=-2), dict(groups=2.0), dict(act="gelu"),
               dict(layout="nchw"), dict(eps=0.0), dict(eps=float("nan")), dict(act="leaky"), dict(act="silu", slope=0.1),
               dict(act="none", slope=w), dict(act="prelu", slope=0.1), dict(weight=w.double()),
               dict(weight=w.half()), dict()):
        with pytest.raises(_lib.GanAmdError):
            ops.group_norm_act(x, **{**dict(groups=2, weight=w, bias=w), **kw})
    with pytest.raises(_lib.GanAmdError):
        ops.group_norm_act(x.double(), 2, w, w)
    with pytest.raises(_lib.GanAmdError):
        ops.group_norm_act(torch.zeros(8), 2, w, w)


def test_group_norm_abi_refusals():
    from gan_amd import _lib
    L = _lib.LIB
    n = _lib.c_size_t(0)
    good = dict(L=16, B=2, C=8, G=2, layout=0, dtype=0, param_dtype=0, act=1, slope=0.0, eps=1e-5)
    assert L.ganamd_group_norm_workspace(_lib.NormDesc(**good), 1, n) == 0 and n.value > 0
    need = n.value
    for bad in (dict(L=0), dict(B=0), dict(C=0), dict(G=0), dict(G=3), dict(layout=2), dict(dtype=3),
                dict(param_dtype=-1), dict(act=4), dict(eps=0.0), dict(eps=float("nan")), dict(L=1 << 31),
                dict(B=65535 * 512 + 1)):
        assert L.ganamd_group_norm_workspace(_lib.NormDesc(**{**good, **bad}), 0, n) == -1, bad
    d = _lib.NormDesc(**good)
    assert L.ganamd_group_norm_workspace(d, 3, n) == -1 and L.ganamd_group_norm_workspace(d, -1, n) == -1
    f = 0x1000                         # never dereferenced: every call below is refused on the host
    assert L.ganamd_group_norm_fwd(d, None, f, f, None, f, f, None, 0, None) == -1
    assert L.ganamd_group_norm_fwd(_lib.NormDesc(**{**good, "act": 3}), f, f, f, None, f, f, f, 1 << 20, None) == -1
    assert L.ganamd_group_norm_bwd(d, f, f, f, f, None, f, f, f, f, None, 0, f, need - 1, None) == -1
    assert L.ganamd_group_norm_bwd(d, f, f, f, f, None, f, f, f, f, f, 0, f, need, None) == -1
    assert L.ganamd_group_norm_bwd_bwd(d, None, *[None] * 3, f, f, f, f, None, f, f, f, f, f, None, 0, f, 1 << 30, None) == -1


def test_clip_refusals():
    from gan_amd import _lib, ops
    cpu = [torch.zeros(3)]
    for f in (lambda: ops.grad_norm(cpu), lambda: ops.clip_grad_norm_(cpu, 1.0), lambda: ops.grad_norm([None]),
              lambda: ops.grad_norm(cpu, 1.0), lambda: ops.grad_norm(cpu, 3), lambda: ops.clip_grad_norm_(cpu, -1.0),
              lambda: ops.clip_grad_norm_(cpu, float("nan")), lambda: ops.clip_grad_norm_(cpu, 1.0, norm_type=0)):
        with pytest.raises(_lib.GanAmdError):
            f()


def tensors(*rows):
    """An array of ganamd_tensor rows (p, out, n, dtype, out_dtype) and its address."""
    import array
    a = array.array("q", [v for p, out, n, d, o in rows for v in (p, out, n, d | o << 32)])
    return a, a.buffer_info()[0]


def test_clip_abi_refusals():
    from gan_amd import _lib
    L = _lib.LIB
    f, big = 0x100000, 1 << 40

    def clip(*rows, kind=0, most=1.0, norm=f, ws=f, size=big):
        keep, at = tensors(*rows)
        return L.ganamd_grad_clip(at, len(rows), kind, most, norm, ws, size, None)

    one = (0x1000, 0x1000, 16, 0, 0)
    assert clip((0x1000, 0x1000, -1, 0, 0)) == -1 and clip((0, 0, 4, 0, 0)) == -1
    assert clip((0x1000, 0, 4, 0, 0)) == -1 and clip((0x1000, 0x2000, 4, 3, 0)) == -1
    assert clip((0x1000, 0x2000, 4, 0, 1)) == -1 and clip((0x1000, 0x2000, 4, 2, 1)) == -1
    assert clip(one, kind=2) == -1 and clip(one, most=-1.0) == -1 and clip(one, most=float("nan")) == -1
    assert clip(one, norm=None) == -1 and clip(one, ws=None) == -1 and clip(one, size=15) == -1
    # shared memory: the same tensor twice, overlapping outputs, an output on another's input, on
    # part of its own input, in place in another type
    assert clip(one, one) == -1
    assert clip((0x1000, 0x1000, 16, 0, 0), (0x103c, 0x103c, 4, 0, 0)) == -1
    assert clip((0x1000, 0x2000, 16, 0, 0), (0x2010, 0x3000, 4, 0, 0)) == -1
    assert clip((0x2000, 0x1000, 16, 0, 0), (0x3000, 0x103f, 4, 1, 0)) == -1
    assert clip((0x1000, 0x1004, 16, 0, 0)) == -1 and clip((0x1000, 0x1000, 16, 1, 0)) == -1
    keep, at = tensors(one, (0, 0, 0, 0, 0))
    assert L.ganamd_grad_norm_workspace(at, 2) == 16
    assert L.ganamd_grad_norm(at, 2, 5, f, f, big, None) == -1 and L.ganamd_grad_norm(at, 2, 0, f, f, 8, None) == -1
    assert L.ganamd_grad_norm(None, 1, 0, f, f, big, None) == -1 and L.ganamd_grad_norm(at, -1, 0, f, f, big, None) == -1


def test_clipped_step_refusals():
    from gan_amd import _lib, ops
    L, f = _lib.LIB, 0x1000
    k = (1e-3, 0.9, 0.999, 1e-8, 0.0)
    assert L.ganamd_adamw_clip(f, f, f, f, 0, f, *k, 1.0, f, f, 1 << 20, None) == -1
    assert L.ganamd_adamw_clip(f, f, f, f, 8, f, *k, -1.0, f, f, 1 << 20, None) == -1
    assert L.ganamd_adamw_clip(f, f, f, f, 8, f, *k, 1.0, None, f, 1 << 20, None) == -1
    assert L.ganamd_adamw_clip(f, f, f, f, 8, f, *k, 1.0, f, f, 8, None) == -1
    t = [torch.zeros(8) for _ in range(4)]
    step = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(_lib.GanAmdError):
        ops.clipped_adamw_(*t, step, 1e-3, (0.9, 0.999), 1e-8, 0.0, 1.0)          # not on the GPU
    with pytest.raises(_lib.GanAmdError):
        ops.clipped_adamw_(t[0], torch.zeros(7), *t[2:], step, 1e-3, (0.9, 0.999), 1e-8, 0.0, 1.0)
    with pytest.raises(_lib.GanAmdError):
        ops.clipped_adamw_(*t, step, 1e-3, (0.9, 0.999), 1e-8, 0.0, -1.0)


def test_trainers_and_optimizer_take_max_grad_norm():
    import gan_amd
    from gan_amd.optim import FusedAdamW
    with pytest.raises(gan_amd._lib.GanAmdError):
        FusedAdamW(torch.nn.Linear(2, 2), max_grad_norm=-1.0)
    assert FusedAdamW(torch.nn.Linear(2, 2)).max_grad_norm is None
    assert FusedAdamW(torch.nn.Linear(2, 2), max_grad_norm=0.5).max_grad_norm == 0.5
    mk = lambda **kw: gan_amd.Train([], "cpu", 1, 4, torch.nn.Linear(2, 2), "g", torch.nn.Linear(2, 2), "d", **kw)  # noqa: E731
    with pytest.raises(ValueError):
        mk(rng=object(), max_grad_norm=-0.5)
    tr = mk(rng=object(), max_grad_norm=2.0)
    assert tr.optimizer_G.max_grad_norm == tr.optimizer_D.max_grad_norm == 2.0
    assert mk(rng=object()).optimizer_D.max_grad_norm is None


def test_forward_mode_is_refused():
    """A dual tensor's tangent is never dropped silently, whichever argument carries it."""
    import torch.autograd.forward_ad as fwad
    from gan_amd import _lib, ops
    x, w = torch.zeros(2, 3, 3, 8), torch.ones(8)
    step = torch.zeros(1, dtype=torch.int32)
    b = [torch.zeros(8) for _ in range(4)]
    with fwad.dual_level():
        dual = lambda t: fwad.make_dual(t, torch.ones_like(t))   # noqa: E731
        for f in (lambda: ops.group_norm_act(dual(x), 2, w, w), lambda: ops.group_norm_act(x, 2, dual(w), w),
                  lambda: ops.group_norm_act(x, 2, w, dual(w)), lambda: ops.grad_norm([dual(w)]),
                  lambda: ops.group_norm_act(x, 2, w, w, act="prelu", slope=dual(w)),
                  lambda: ops.clip_grad_norm_([dual(w)], 1.0),
                  lambda: ops.clipped_adamw_(b[0], dual(b[1]), *b[2:], step, 1e-3, (0.9, 0.999), 1e-8, 0.0, 1.0)):
            with torch.no_grad(), pytest.raises(_lib.GanAmdError, match="tangent"):
                f()
            with pytest.raises(_lib.GanAmdError, match="tangent"):
                f()


@pytest.mark.parametrize("L,C,G,layout,dtype", [(1, 1024, 32, 0, 0), (1, 1024, 32, 0, 1), (1, 96, 32, 0, 0), (1, 8, 2, 1, 0),
                                                (2048, 2048, 4, 0, 1), (40_000, 4, 2, 1, 0), (5, 1, 1, 0, 2)])
@pytest.mark.parametrize("op", [0, 1, 2])
def test_plan_refuses_what_no_launch_holds(L, C, G, layout, dtype, op):
    """The largest batch that is taken needs fewer than 2^32 threads in every launch over the maps; one
    sample more would not, unless the limit of 65535 * 512 samples comes first."""
    from gan_amd import _lib

    def threads(B):
        d = _lib.NormDesc(L, B, C, G, layout, dtype, 0, 1, 0.0, 1e-5)
        info, n = (ctypes.c_int * 11)(), _lib.c_size_t(0)
        rc = _lib.LIB.ganamd_group_norm_plan_info(d, op, info)
        assert rc == _lib.LIB.ganamd_group_norm_workspace(d, op, n)
        return None if rc else B * info[6] * max(info[7], info[9]) * info[2]

    lo, hi = 1, 65535 * 512 + 1
    assert threads(lo) and threads(hi) is None
    while hi - lo > 1:
        mid = (lo + hi) // 2
        if threads(mid) is None:
            hi = mid
        else:
            lo = mid
    assert threads(lo) < 1 << 32
    assert lo == 65535 * 512 or threads(lo) * hi // lo >= 1 << 32
    for B in (2_100_000, 4_200_000, 33_000_000):
        assert threads(B) is None or threads(B) < 1 << 32


def test_optimizer_numbers_of_any_kind(monkeypatch):
    """lr, betas, eps, weight decay and the norm's limit as numpy scalars or 0-dim tensors, as the step
    without a clip takes them: the native step is handed Python floats."""
    import numpy as np
    import gan_amd
    from gan_amd import optim
    seen = []
    monkeypatch.setattr(optim, "clipped_adamw_", lambda *a, **k: seen.append(a))
    one = lambda: torch.nn.Linear(2, 2)   # noqa: E731
    tr = gan_amd.Train([], "cpu", 1, 4, one(), "g", one(), "d", rng=object(), max_grad_norm=torch.tensor(2.0))
    for num in (np.float32, torch.tensor, np.float64, float):
        opts = [optim.FusedAdamW(one(), lr=num(0.5), betas=(num(0.25), num(0.75)), eps=num(2.0 ** -20),
                                 weight_decay=num(0.125), max_grad_norm=num(2.0)), tr.optimizer_D]
        opts[1].lr, opts[1].betas, opts[1].eps, opts[1].weight_decay = num(0.5), (num(0.25), num(0.75)), num(2.0 ** -20), num(0.125)
        for o in opts:
            assert type(o.max_grad_norm) is float
            o.step()
            lr, betas, eps, wd, most = seen.pop()[5:]
            got = (lr, *betas, eps, wd, most)
            assert got == (0.5, 0.25, 0.75, 2.0 ** -20, 0.125, 2.0) and all(type(v) is float for v in got)
            o.max_grad_norm = num(4.0)                   # set later
            o.step()
            assert seen.pop()[-1] == 4.0 and not seen
            o.max_grad_norm = 2.0
