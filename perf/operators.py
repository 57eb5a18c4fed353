"""Cases of the normalisation and clipping operators, for timing and for comparison with their plain forms.

``own`` False: elementary torch operations in 32 bits (64 where a sum is long or a value lies next
to an activation's kink).  ``own`` True: the calls a user makes of ``gan_amd``.

The operators: a group norm with its activation (forward; forward and backward of a training step;
the second derivative that a gradient penalty needs), the clipping of many gradient tensors by
their global norm, and the AdamW step of a flat parameter buffer under such a clip.
"""
import math
import random

import torch

own = False

EPS = 1e-5                                # group norm
LR, BETAS, ADAM_EPS, DECAY = 4e-4, (0.5, 0.999), 1e-8, 0.01
CLIP_EPS = 1e-6
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}


def listed():
    def norm(name, op, B, H, W, C, groups, dtype, act, layout="nhwc"):
        return dict(name=name, op=op, B=B, H=H, W=W, C=C, groups=groups, dtype=dtype, act=act, layout=layout)

    def clip(name, tensors, total, dtype, out):
        return dict(name=name, op="clip", tensors=tensors, total=total, dtype=dtype, out=out)

    return [
        # one image's smallest map on its way through a sampler: latency alone
        norm("norm one 4x4 map", "norm", 1, 4, 4, 128, 8, "float32", "silu"),
        # the last maps of the fake batch that a critic step draws without autograd
        norm("norm 64x64 maps", "norm", 64, 64, 64, 96, 32, "bfloat16", "silu"),
        # maps with the minibatch statistic as a channel of its own: rows of an odd length
        norm("norm 1025 channels", "norm", 64, 4, 4, 1025, 5, "float16", "prelu"),
        # a generator's training step at full size, the framework's own layout
        norm("train channel rows", "train", 64, 64, 64, 48, 8, "float32", "leaky", "cnhw"),
        # a ragged last batch of cropped images
        norm("train ragged", "train", 7, 33, 31, 100, 20, "float32", "prelu"),
        # the widest batch the benchmark runs its generator at
        norm("train 256 images", "train", 256, 64, 64, 96, 32, "bfloat16", "silu"),
        # a critic's maps under the gradient penalty, kinked and smooth activation
        norm("penalty channel rows", "penalty", 64, 32, 32, 128, 16, "float32", "leaky", "cnhw"),
        norm("penalty 64x64 maps", "penalty", 64, 64, 64, 64, 8, "float32", "silu"),
        # the gradients of a mapping network's layers
        clip("clip 24 tensors", 24, 530_000, "float32", "float32"),
        # a critic's gradients out of a bf16 backward, into the optimizer's fp32 buffer
        clip("clip 900 tensors", 900, 150_000_001, "bfloat16", "float32"),
        # the step of a style bank's slice, and of the whole generator
        dict(name="step 1M", op="step", n=1_050_001),
        dict(name="step 362M", op="step", n=362_300_000),
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "train", "train", "penalty", "penalty", "clip", "step"])
    if op == "step":
        return dict(op=op, n=_spread(rng, 1000, 360_000_000))
    if op == "clip":
        tensors = _spread(rng, 1, 2000)
        dtype = rng.choice(["float32", "bfloat16", "float16", "mixed"])
        return dict(op=op, tensors=tensors, total=max(tensors * 4, _spread(rng, 1000, 150_000_000)), dtype=dtype,
                    out=rng.choice(["float32", "same"]))
    most = {"norm": 100_000_000, "train": 100_000_000, "penalty": 16_000_000}[op]
    while True:
        B, C = _spread(rng, 1, 256), _spread(rng, 4, 1200)
        H = rng.choice([1, 2, 3, 4, 5, 7, 8, 13, 16, 25, 32, 33, 64])
        W = rng.choice([H, H, H + 1])
        groups = rng.choice([g for g in range(1, min(C, 64) + 1) if C % g == 0])
        # a group of a few values normalises to little but its rounding: no gradient is left to compare
        if B * H * W * C <= most and H * W * (C // groups) >= 32:
            return dict(op=op, B=B, H=H, W=W, C=C, groups=groups, dtype=rng.choice(sorted(DTYPES)),
                        act=rng.choice(["none", "silu", "leaky", "prelu"]), layout=rng.choice(["nhwc", "nhwc", "cnhw"]))


def _sizes(case):
    """Element counts of a model's parameter tensors: many small ones, a few that hold most."""
    r = random.Random(case["tensors"] * 7919 + case["total"])
    n, total = case["tensors"], case["total"]
    raw = [math.exp(r.gauss(0.0, 2.5)) for _ in range(n)]
    s = sum(raw)
    sizes = [1 + int((total - n) * v / s) for v in raw]
    sizes[0] += total - sum(sizes)
    return sizes


def _clip_types(case):
    n = case["tensors"]
    ins = [["float32", "bfloat16", "float16"][i % 3] for i in range(n)] if case["dtype"] == "mixed" else [case["dtype"]] * n
    return ins, (ins if case["out"] == "same" else ["float32"] * n)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if case["op"] == "step":
        n = case["n"]
        m = randn(n) * 1e-3
        return dict(case=case, p=randn(n), g=randn(n) * 2e-3, m=m, v=(randn(n) * 1e-3).square_().add_(1e-7),
                    step=torch.full((1,), 1000, dtype=torch.int32, device="cuda"), limit=0.25 * 2e-3 * math.sqrt(n))
    if case["op"] == "clip":
        sizes = _sizes(case)
        ins, outs = _clip_types(case)
        # one buffer per type, cut into the tensors, as a model's flat buffers are
        bufs, dst, grads, targets = {}, {}, [], []
        for t in sorted(set(ins)):
            k = sum(s for s, u in zip(sizes, ins) if u == t)
            bufs[t] = (randn(k) * torch.exp(randn(k) * 0.5) * 1e-3).to(DTYPES[t])
        for t in sorted(set(outs)):
            dst[t] = torch.zeros(sum(s for s, u in zip(sizes, outs) if u == t), dtype=DTYPES[t], device="cuda")
        at, to = dict.fromkeys(bufs, 0), dict.fromkeys(dst, 0)
        for s, t, u in zip(sizes, ins, outs):
            grads.append(bufs[t][at[t]:at[t] + s])
            targets.append(dst[u][to[u]:to[u] + s])
            at[t] += s
            to[u] += s
        return dict(case=case, grads=grads, targets=targets, bufs=bufs, dst=dst, limit=0.3e-3 * math.sqrt(case["total"]))
    B, H, W, C = (case[k] for k in "BHWC")
    dt = DTYPES[case["dtype"]]
    cn = case["layout"] == "cnhw"
    shape, per = ((C, B, H, W), (C, 1, 1, 1)) if cn else ((B, H, W, C), (C,))
    s = dict(case=case, x=(randn(*shape) * torch.exp(0.3 * randn(*per)) + randn(*per)).to(dt),
             w=1 + 0.3 * randn(C), b=0.3 * randn(C), slope=None)
    if case["act"] == "prelu":
        s["slope"] = 0.25 + 0.1 * randn(C)
    elif case["act"] == "leaky":
        s["slope"] = 0.2
    if case["op"] != "norm":
        s["gy"] = randn(*shape).to(dt)
    if case["op"] == "penalty":
        s["v"] = randn(*shape).to(dt)
    return s


# ------------------------------------------------------------------------------ the plain forms


def _plain_norm(s, x, w, b, slope):
    """y in 32 bits, from 32-bit x [B, L, C]-like views; differentiable as often as one likes."""
    case = s["case"]
    cn, G, C = case["layout"] == "cnhw", case["groups"], case["C"]
    B = case["B"]
    L = case["H"] * case["W"]
    if cn:
        xg, dims = x.reshape(G, C // G, B, L), (1, 3)
        shape = (G, C // G, 1, 1)
    else:
        xg, dims = x.reshape(B, L, G, C // G), (1, 3)
        shape = (1, 1, G, C // G)
    d = xg - xg.mean(dims, keepdim=True)
    r = torch.rsqrt((d * d).mean(dims, keepdim=True) + EPS)
    wv, bv = w.reshape(shape), b.reshape(shape)
    z = d * r * wv + bv
    act = case["act"]
    if act == "silu":
        z = z * (1 / (1 + torch.exp(-z)))
    elif act in ("leaky", "prelu"):
        with torch.no_grad():             # which side of the kink: in 64 bits
            x64 = xg.double()
            d64 = x64 - x64.mean(dims, keepdim=True)
            del x64
            pos = d64 * torch.rsqrt((d64 * d64).mean(dims, keepdim=True) + EPS) * wv + bv > 0
            del d64
        z = torch.where(pos, z, (slope.reshape(shape) if act == "prelu" else slope) * z)
    return z.reshape(x.shape)


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "step":
        g = s["g"]
        norm = torch.sqrt((g.double() * g.double()).sum())
        g = g * torch.clamp(s["limit"] / (norm + CLIP_EPS), max=1.0).float()
        s["step"] += 1
        t = s["step"].double()
        p, m, v = s["p"], s["m"], s["v"]
        p *= 1 - LR * DECAY
        m += (1 - BETAS[0]) * (g - m)
        v *= BETAS[1]
        v += (1 - BETAS[1]) * (g * g)
        size, root = (LR / (1 - BETAS[0] ** t)).float(), torch.sqrt(1 - BETAS[1] ** t).float()
        p -= size * (m / (torch.sqrt(v) / root + ADAM_EPS))
        return dict(p=p, m=m, v=v, step=s["step"], norm=norm.float())
    if op == "clip":
        ins, _ = _clip_types(case)
        flat = torch.cat([t.float() for t in s["grads"]])
        norm = torch.sqrt((flat.double() * flat.double()).sum())
        flat *= torch.clamp(s["limit"] / (norm + CLIP_EPS), max=1.0).float()
        torch._foreach_copy_(s["targets"], list(flat.split([t.numel() for t in s["grads"]])))
        return dict(norm=norm.float(), **s["dst"])
    dt = s["x"].dtype
    x = s["x"].float()
    if op == "norm":
        with torch.no_grad():
            return _plain_norm(s, x, s["w"], s["b"], s["slope"]).to(dt)
    leaves = [t.detach().requires_grad_() for t in (x, s["w"], s["b"]) + ((s["slope"],) if case["act"] == "prelu" else ())]
    slope = leaves[3] if case["act"] == "prelu" else s["slope"]
    y = _plain_norm(s, leaves[0], leaves[1], leaves[2], slope)
    if op == "train":
        got = torch.autograd.grad(y, leaves, s["gy"].float())
        return [y.detach().to(dt), got[0].to(dt), *got[1:]]
    gy = s["gy"].float().requires_grad_()
    (gx,) = torch.autograd.grad(y, leaves[0], gy, create_graph=True)
    # the bias moves the gradient of a kinked or absent activation nowhere
    smooth = case["act"] == "silu"
    wanted = [gy, *(leaves if smooth else [leaves[0], leaves[1], *leaves[3:]])]
    if case["act"] == "none":
        wanted = wanted[:3]
    got = torch.autograd.grad(gx, wanted, s["v"].float())
    return [gx.detach().to(dt), got[0].to(dt), got[1].to(dt), *got[2:]]


# ------------------------------------------------------------------------------ the framework's calls


def _own(s):
    from gan_amd import ops

    case = s["case"]
    op = case["op"]
    if op == "step":
        norm = ops.clipped_adamw_(s["p"], s["g"], s["m"], s["v"], s["step"], LR, BETAS, ADAM_EPS, DECAY, s["limit"])
        return dict(p=s["p"], m=s["m"], v=s["v"], step=s["step"], norm=norm)
    if op == "clip":
        norm = ops.clip_grad_norm_(s["grads"], s["limit"], out=s["targets"])
        return dict(norm=norm, **s["dst"])
    kw = dict(act=case["act"], slope=s["slope"], eps=EPS, layout=case["layout"])
    if op == "norm":
        with torch.no_grad():
            return ops.group_norm_act(s["x"], case["groups"], s["w"], s["b"], **kw)
    leaves = [t.detach().requires_grad_() for t in (s["x"], s["w"], s["b"])]
    if case["act"] == "prelu":
        leaves.append(s["slope"].detach().requires_grad_())
        kw["slope"] = leaves[3]
    y = ops.group_norm_act(leaves[0], case["groups"], leaves[1], leaves[2], **kw)
    if op == "train":
        return [y.detach(), *torch.autograd.grad(y, leaves, s["gy"])]
    gy = s["gy"].detach().requires_grad_()
    (gx,) = torch.autograd.grad(y, leaves[0], gy, create_graph=True)
    smooth = case["act"] == "silu"
    wanted = [gy, *(leaves if smooth else [leaves[0], leaves[1], *leaves[3:]])]
    return [gx.detach(), *torch.autograd.grad(gx, wanted, s["v"])]


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    op = case["op"]
    if op == "step":
        return {"bytes": 28 * case["n"], "flops": 18 * case["n"]}
    if op == "clip":
        ins, outs = _clip_types(case)
        sizes = _sizes(case)
        return {"bytes": sum(n * (SIZE[i] + SIZE[o]) for n, i, o in zip(sizes, ins, outs)), "flops": 3 * case["total"]}
    n = case["B"] * case["H"] * case["W"] * case["C"]
    # forward: x, y; training step: x, gy, y, gx; penalty: x, gy, v, gx, and the gradients of gy and x
    tensors, flops = {"norm": (2, 12), "train": (4, 36), "penalty": (6, 70)}[op]
    return {"bytes": tensors * SIZE[case["dtype"]] * n + 16 * case["C"], "flops": flops * n}


# ------------------------------------------------------------------------------ the definition in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "step":
        g = s["g"].double()
        norm = g.square().sum().sqrt()
        g *= min(1.0, s["limit"] / (float(norm) + CLIP_EPS))
        t = 1001
        m = BETAS[0] * s["m"].double() + (1 - BETAS[0]) * g
        v = BETAS[1] * s["v"].double() + (1 - BETAS[1]) * g.square_()
        del g
        p = s["p"].double() * (1 - LR * DECAY)
        p -= LR * (m / (1 - BETAS[0] ** t)) / ((v / (1 - BETAS[1] ** t)).sqrt_() + ADAM_EPS)
        return dict(p=p, m=m, v=v, step=None, norm=norm)
    if op == "clip":
        total = sum(float(b.double().square().sum()) for b in s["bufs"].values())
        c = min(1.0, s["limit"] / (math.sqrt(total) + CLIP_EPS))
        _, outs = _clip_types(case)
        got = {t: torch.cat([g.double() for g, u in zip(s["grads"], outs) if u == t]) * c for t in sorted(set(outs))}
        return dict(norm=torch.tensor(math.sqrt(total), dtype=torch.float64), **got)
    B, C, G, L = case["B"], case["C"], case["groups"], case["H"] * case["W"]
    cn = case["layout"] == "cnhw"

    def lay(t):                            # [B, L, G, C / G] in 64 bits
        t = t.double()
        return t.reshape(C, B, L).permute(1, 2, 0).reshape(B, L, G, C // G) if cn else t.reshape(B, L, G, C // G)

    def back(t):
        t = t.reshape(B, L, C)
        return t.permute(2, 0, 1).reshape(s["x"].shape) if cn else t.reshape(s["x"].shape)

    def over(t):                           # group means
        return t.mean((1, 3), keepdim=True)

    def channel(t):                        # per-channel sums
        return t.sum((0, 1)).reshape(C)

    x = lay(s["x"])
    w, b = s["w"].double().reshape(1, 1, G, C // G), s["b"].double().reshape(1, 1, G, C // G)
    x = x - over(x)
    r = (over(x.square()) + EPS).rsqrt()
    xh = x.mul_(r)
    z = xh * w + b
    act = case["act"]
    a2 = None
    if act == "none":
        y, a1 = z, torch.ones_like(z)
    elif act == "silu":
        sg = torch.sigmoid(z)
        y, a1, a2 = z * sg, sg * (1 + z * (1 - sg)), sg * (1 - sg) * (2 + z * (1 - 2 * sg))
    else:
        k = s["slope"].double().reshape(1, 1, G, C // G) if act == "prelu" else s["slope"]
        neg = z <= 0
        a1 = torch.where(neg, k, 1.0).expand_as(z) if act == "prelu" else torch.where(neg, float(k), 1.0).double()
        y = z * a1
    if op == "norm":
        return back(y)
    gy = lay(s["gy"])
    g = gy * a1
    u = g * w
    mu, mux = over(u), over(u * xh)
    gx = r * (u - mu - xh * mux)
    if op == "train":
        got = [back(y), back(gx), channel(g * xh), channel(g)]
        return got + ([channel(torch.where(neg, gy * z, 0.0))] if act == "prelu" else [])
    v = lay(s["v"])
    mvx = over(v * xh)
    q = r * (v - over(v) - xh * mvx)
    h = w * q
    e = -r * (v * mux + u * mvx)
    gw = channel(g * q)
    if a2 is not None:
        t = gy * a2 * h
        e += t * w
        gw = gw + channel(t * xh)
    g_x = r * (e - over(e) - xh * over(e * xh)) - r * xh * over(u * q)
    got = [back(gx), back(a1 * h), back(g_x), gw]
    if act == "silu":
        got.append(channel(t))
    if act == "prelu":
        got.append(channel(torch.where(neg, gy * h, 0.0)))
    return got
