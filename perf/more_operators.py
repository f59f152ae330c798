"""A gated feed-forward block, served and trained, and what stands between its backward pass and the optimizer: the norm of all gradients
and their clipping, in place or as AdamW reads them.

The block.  x [M, D], W_in [2 F, D] (the gate's rows, then the other projection's), W_out [N, F]:

    [g | u] = s (keep . x) W_in^T        h = act(g) u        y = s' (keep' . h) W_out^T

act is silu, gelu (with erf) or relu.  In training blocks of x and h are dropped, s = 1 / (1 - p); serving drops nothing.

Clipping.  norm = sqrt of the sum of all squares, or the largest magnitude; every gradient is multiplied by
min(1, max_norm / (norm + 1e-6)).
"""
import os
import random
import sys

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BETA1, BETA2, EPS, LR, DECAY = 0.9, 0.999, 1e-8, 1e-3, 0.01
SMALL = 1e-6  # beside the norm in the factor


def _package():
    at = os.path.join(os.getcwd(), "sparse-dropout_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import flash_dropout.functional as F

    return F


# ------------------------------------------------------------------------------------------------ cases
def _serve(m, d, f, n=None, act="silu", dtype="bf16"):
    return dict(kind="serve", m=m, d=d, f=f, n=n or d, act=act, dtype=dtype)


def _train(m, d, f, n=None, act="silu", dtype="bf16", bs=64, p=0.0):
    return dict(kind="train", m=m, d=d, f=f, n=n or d, act=act, dtype=dtype, bs=bs, p=p)


def _clip(dims, layers, dtype="bf16", norm="2", limit=1.0):
    """dims: features of one stack of layers, "784-1024-10"; every layer has its weights and a vector of as many elements as outputs.
    dtype "mixed": the weights in bf16, the vectors in fp32."""
    return dict(kind="clip", dims=dims, layers=layers, dtype=dtype, norm=norm, limit=limit)


def _step(dims, layers, dtype="fp32", norm="2", limit=1.0, step=10):
    return dict(kind="step", dims=dims, layers=layers, dtype=dtype, norm=norm, limit=limit, step=step)


def listed():
    return [
        # serving: one token, where what a call costs and the weights' bytes are all there is
        dict(_serve(1, 1024, 4096), name="serve 1 token"),
        # a few requests, a token each, through a block whose hidden width is 8/3 of its features and was not rounded up
        dict(_serve(24, 2048, 5461, act="gelu", dtype="fp16"), name="serve 24 tokens odd"),
        # a batch of 200 requests: too few rows to fill the chip, too many to only stream weights
        dict(_serve(200, 2048, 8192, dtype="fp16"), name="serve 200 tokens"),
        # a long prompt
        dict(_serve(8192, 2048, 8192), name="serve 8192 tokens"),
        # training: a small block on a small batch
        dict(_train(128, 256, 512, p=0.1, dtype="fp16"), name="train small"),
        # sizes nobody rounded, an activation of three, some blocks dropped
        dict(_train(3001, 1025, 777, 640, act="gelu", p=0.3), name="train odd"),
        # the block of 32 sequences of 128 tokens, nothing dropped
        dict(_train(4096, 1024, 4096, act="gelu", dtype="fp16"), name="train 4096 tokens"),
        # a large block, half of its blocks dropped
        dict(_train(8192, 2048, 8192, p=0.5), name="train 8192 tokens"),
        # the gradients of a small classifier, ten outputs
        dict(_clip("784-1024-1024-10", 1, "fp16"), name="clip classifier"),
        # those of five feed-forward blocks, vectors in 32 bits among them
        dict(_clip("2048-8192-2048", 5, "mixed"), name="clip blocks"),
        # the same two with their update: no gradient is wanted behind it
        dict(_step("784-1024-1024-10", 1, "fp32"), name="step classifier"),
        dict(_step("2048-8192-2048", 5, "bf16"), name="step blocks"),
    ]


# What the listed cases stand for.  No drawn case does more work of its kind than the largest listed one.
_MOST = {"serve": 8192 * 8192 * 3 * 2048, "train": 8192 * 8192 * 3 * 2048 / 2, "clip": 5 * 2 * 2048 * 8192, "step": 5 * 2 * 2048 * 8192}


def _size(rng, lo, hi, grain=1):
    """Spread over the logarithm of [lo, hi], a multiple of grain."""
    v = lo * (hi / lo) ** rng.random()
    return max(grain, int(v / grain + 0.5) * grain)


def draw(rng):
    kind = rng.choices(("serve", "train", "clip", "step"), (6, 6, 3, 3))[0]
    while True:
        grain = rng.choice((64, 64, 8, 1))
        if kind in ("serve", "train"):
            d, f = _size(rng, 64, 4096, grain), _size(rng, 64, 8192, grain)
            n = d if rng.random() < 0.7 else _size(rng, 64, 4096, grain)
            act, dtype = rng.choice(("silu", "silu", "gelu", "relu")), rng.choice(("fp16", "bf16"))
            if kind == "serve":
                c = _serve(_size(rng, 1, 8192), d, f, n, act, dtype)
                size = c["m"] * f * (2 * d + n)
            else:
                c = _train(_size(rng, 64, 16384, rng.choice((64, 1))), d, f, n, act, dtype, rng.choice((64, 64, 128, 32)),
                           rng.choice((0.0, 0.0, 0.1, 0.2, 0.3, 0.5, 0.75)))
                size = c["m"] * f * (2 * d + n) * (1 - c["p"])
        else:
            d = _size(rng, 64, 2048, grain)
            dims = f"{d}-{4 * d}-{d}" if rng.random() < 0.5 else f"{_size(rng, 128, 4096, grain)}-{d}-{_size(rng, 10, 1000)}"
            layers, norm, limit = rng.choice((1, 2, 3, 5)), rng.choice(("2", "2", "2", "inf")), rng.choice((0.01, 1.0, 1.0, 1e6))
            if kind == "clip":
                c = _clip(dims, layers, rng.choice(("fp16", "bf16", "fp32", "mixed")), norm, limit)
            else:
                c = _step(dims, layers, rng.choice(("fp16", "bf16", "fp32")), norm, limit, rng.choice((0, 1, 10, 1000)))
            size = layers * sum(i * o for i, o in _pairs(c))
        if size <= _MOST[kind]:
            return c


def _pairs(case):
    dims = [int(v) for v in case["dims"].split("-")]
    return list(zip(dims, dims[1:]))


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(dev).manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=gen, device=dev).mul_(std)

    if case["kind"] in ("serve", "train"):
        m, d, f, n, dt = case["m"], case["d"], case["f"], case["n"], _DTYPES[case["dtype"]]
        x = normal(m, d)
        x[:, torch.randint(d, (1 + d // 200,), generator=gen, device=dev)] *= 10  # a few features larger than the others
        s = dict(case=case, x=x.to(dt), w_in=normal(2 * f, d, std=d ** -0.5).to(dt), w_out=normal(n, f, std=f ** -0.5).to(dt))
        if case["kind"] == "train":
            for key in ("x", "w_in", "w_out"):
                s[key].requires_grad_()
            s["dy"] = normal(m, n, std=0.01).to(dt)
            s["masks"] = None
            if case["p"]:
                bs = case["bs"]
                s["masks"] = [torch.rand(-(-m // bs), -(-k // bs), generator=gen, device=dev) < case["p"] for k in (d, f)]
        return s
    host = random.Random(seed)
    s = dict(case=case, grads=[])
    shapes = [shape for i, o in _pairs(case) * case["layers"] for shape in ((o, i), (o,))]
    for shape in shapes:  # layers have gradients of different sizes
        dt = _DTYPES["fp32" if len(shape) == 1 else "bf16"] if case["dtype"] == "mixed" else _DTYPES[case["dtype"]]
        s["grads"].append(normal(*shape, std=0.02 * 10 ** -host.random()).to(dt))
    if case["kind"] == "step":
        dt = _DTYPES[case["dtype"]]
        s.update(step=torch.full((), case["step"], dtype=torch.int64, device=dev), params=[], first=[], second=[])
        for shape in shapes:
            s["params"].append(normal(*shape, std=shape[-1] ** -0.5).to(dt))
            first, second = normal(*shape, std=1e-4), normal(*shape, std=3e-4).square_()
            s["first"].append(first if case["step"] else first.zero_())
            s["second"].append(second if case["step"] else second.zero_())
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    return {"serve": _run_serve, "train": _run_train, "clip": _run_clip, "step": _run_step}[case["kind"]](state, case)


def _run_serve(s, case):
    if own:
        with torch.no_grad():
            return _package().gated_mlp(s["x"], s["w_in"], s["w_out"], case["act"])
    f = case["f"]
    a = s["x"].float() @ s["w_in"].float().t()
    h = _act(a[:, :f], case["act"])[0] * a[:, f:]
    return (h @ s["w_out"].float().t()).to(s["x"].dtype)


def _run_train(s, case):
    if own:
        F = _package()
        if case["p"]:
            y = F.hip_blockwise_dropout_gated_mlp(s["x"], s["w_in"], s["w_out"], case["bs"], case["p"], case["act"], masks=s["masks"])
        else:
            y = F.gated_mlp(s["x"], s["w_in"], s["w_out"], case["act"])
        return (y, *torch.autograd.grad(y, (s["x"], s["w_in"], s["w_out"]), s["dy"]))
    with torch.no_grad():
        m, d, f, dt = case["m"], case["d"], case["f"], s["x"].dtype
        x, w_in, w_out, dy = (s[key].float() for key in ("x", "w_in", "w_out", "dy"))
        kx, kh = (_keep(s["masks"][i], case, m, k) if case["p"] else 1.0 for i, k in enumerate((d, f)))
        xd = x * kx
        a = xd @ w_in.t()
        value, slope = _act(a[:, :f], case["act"])
        hd = value * a[:, f:] * kh
        y = hd @ w_out.t()
        dh = (dy @ w_out) * kh
        da = torch.cat((dh * a[:, f:] * slope, dh * value), 1)
        return y.to(dt), ((da @ w_in) * kx).to(dt), (da.t() @ xd).to(dt), (dy.t() @ hd).to(dt)


def _run_clip(s, case):
    if own:
        norm = _package().clip_grad_norm_(s["grads"], case["limit"], norm_type=float(case["norm"]))
    else:
        norm, by = _factor(s["grads"], case)
        for g in s["grads"]:
            g.copy_(g.float() * by)
    return {"norm": norm, "grads": s["grads"]}


def _run_step(s, case):
    out = {"params": s["params"], "first": s["first"], "second": s["second"]}
    if own:
        F = _package()
        out["norm"], by = F.grad_norm(s["grads"], norm_type=float(case["norm"]), max_norm=case["limit"])
        F.adamw_step(s["params"], s["grads"], s["first"], s["second"], s["step"], lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY,
                     grad_scale=by)
        return out
    out["norm"], by = _factor(s["grads"], case)
    s["step"] += 1
    t = s["step"].double()
    rate, root = (LR / (1 - BETA1 ** t)).float(), (1 / torch.sqrt(1 - BETA2 ** t)).float()
    for p, g, m, v in zip(s["params"], s["grads"], s["first"], s["second"]):
        g = g.float() * by
        m.copy_(m * BETA1 + g * (1 - BETA1))
        v.copy_(v * BETA2 + (g * g) * (1 - BETA2))
        p.copy_(p.float() * (1 - LR * DECAY) - rate * (m / (torch.sqrt(v) * root + EPS)))
    return out


# ------------------------------------------------------------------------------------------------ the plain form's parts
def _act(g, act):
    """The activation and its derivative."""
    if act == "relu":
        return g * (g > 0), (g > 0).float()
    if act == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    below = 0.5 * (1 + torch.erf(g * 2 ** -0.5))
    return g * below, below + g * torch.exp(-0.5 * g * g) * 0.3989422804014327


def _keep(mask, case, rows, cols):
    bs = case["bs"]
    return (~mask).repeat_interleave(bs, 0).repeat_interleave(bs, 1)[:rows, :cols].float() / (1 - case["p"])


def _factor(grads, case):
    """The norm, in 64 bits up to its end, and what gradients are multiplied by."""
    if case["norm"] == "inf":
        norm = torch.stack([g.abs().amax().double() for g in grads]).amax()
    else:
        norm = torch.stack([g.double().square().sum() for g in grads]).sum().sqrt()
    return norm.float(), (case["limit"] / (norm + SMALL)).clamp(max=1.0).float()


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "serve":
        gate, up = s["w_in"].double().split(case["f"])
        x = s["x"].double()
        return torch.mm(_exact_act(torch.mm(x, gate.t()), case["act"]) * torch.mm(x, up.t()), s["w_out"].double().t())
    if case["kind"] == "train":
        m, d, f, bs = case["m"], case["d"], case["f"], case["bs"]
        x, w_out, dy = s["x"].detach().double(), s["w_out"].detach().double(), s["dy"].double()
        gate, up = s["w_in"].detach().double().split(f)
        if case["p"]:
            ones = torch.ones(bs, bs, dtype=torch.float64, device=x.device)
            by_x, by_h = (torch.kron(1.0 - t.double(), ones)[:m, :k] / (1.0 - case["p"]) for t, k in zip(s["masks"], (d, f)))
        else:
            by_x, by_h = 1.0, 1.0
        xd = by_x * x
        u = torch.mm(xd, up.t())
        with torch.enable_grad():  # the activation's derivative by differentiation
            g = torch.mm(xd, gate.t()).requires_grad_()
            value = _exact_act(g, case["act"])
            slope, = torch.autograd.grad(value.sum(), g)
        value = value.detach()
        hd = by_h * (value * u)
        dh = by_h * torch.mm(dy, w_out)
        dg, du = dh * slope * u, dh * value
        return (torch.mm(hd, w_out.t()), by_x * (torch.mm(dg, gate) + torch.mm(du, up)), torch.cat((torch.mm(dg.t(), xd), torch.mm(du.t(), xd))),
                torch.mm(dy.t(), hd))
    flat = [g.double().flatten() for g in s["grads"]]
    norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(g, float(case["norm"])) for g in flat]), float(case["norm"]))
    by = min(1.0, case["limit"] / (float(norm) + 1e-6))
    if case["kind"] == "clip":
        return {"norm": norm, "grads": [g.double() * by for g in s["grads"]]}
    t = case["step"] + 1
    out = {"params": [], "first": [], "second": [], "norm": norm}
    for p, g, m, v in zip(s["params"], s["grads"], s["first"], s["second"]):
        p, g = p.double(), g.double() * by
        m = BETA1 * m.double() + (1.0 - BETA1) * g
        v = BETA2 * v.double() + (1.0 - BETA2) * g * g
        out["params"].append(p - LR * DECAY * p - LR * (m / (1.0 - BETA1 ** t)) / ((v / (1.0 - BETA2 ** t)).sqrt() + EPS))
        out["first"].append(m)
        out["second"].append(v)
    return out


def _exact_act(g, act):
    if act == "relu":
        return g.clamp_min(0.0)
    return g * torch.sigmoid(g) if act == "silu" else 0.5 * g * torch.special.erfc(-g / 2.0 ** 0.5)


# ------------------------------------------------------------------------------------------------ bounds
def work(case):
    """Dropped blocks are neither read nor multiplied, those of a gradient are written (zeros).  A clipped gradient is read and written once;
    in a step it is read."""
    size = 4.0 if case["dtype"] == "fp32" else 2.0
    if case["kind"] == "serve":
        m, d, f, n = (case[key] for key in "mdfn")
        return {"bytes": 2.0 * (m * d + 2 * f * d + n * f + m * n), "flops": 2.0 * m * f * (2 * d + n)}
    if case["kind"] == "train":
        m, d, f, n = (case[key] for key in "mdfn")
        keep = 1.0 - case["p"]
        return {"bytes": 2.0 * (m * d * keep + m * d + 2 * (2 * f * d + n * f) + 2 * m * n), "flops": 6.0 * m * f * (2 * d + n) * keep}
    weights, vectors = case["layers"] * sum(i * o for i, o in _pairs(case)), case["layers"] * sum(o for _, o in _pairs(case))
    n = weights + vectors
    if case["kind"] == "clip":
        return {"bytes": 2 * (size * weights + (4.0 if case["dtype"] == "mixed" else size) * vectors), "flops": 3.0 * n}
    # parameters read and written, gradients read, both averages read and written
    return {"bytes": (3 * size + 16.0) * n, "flops": 18.0 * n}
