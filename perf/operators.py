"""Training and serving linear layers in 8 bits: matrices held in 8-bit floating point with a scale for each block of 128, the
product of such matrices with weights that are kept, the block-dropout linear layer computed from them in both directions, and the
AdamW step over many tensors whose two averages are held in 32 or in 8 bits.

Formats.  A matrix in 8 bits is e4m3 (448 the largest) with a power of two for each block of 128 along a row, or of 128 x 128: the
least one with which the block's largest magnitude stays within 448, 1 for a block of zeros.  Columns behind the last are zeros up
to a multiple of 128.  AdamW's averages in 8 bits have a power of two for 128 consecutive elements; the first is e4m3, the second,
which has no sign, has five bits of exponent and three of mantissa (61440 the largest).  They are rounded stochastically, with bits
that are a function of the step and the element's place: an average that moves by a thousandth a step would stay where it is
under rounding to nearest.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BLOCK = 128
E4M3_MAX, E5M3_MAX = 448.0, 61440.0
BETA1, BETA2, EPS, LR, DECAY = 0.9, 0.999, 1e-8, 1e-3, 0.01


def _package():
    at = os.path.join(os.getcwd(), "sparse-dropout_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import flash_dropout.functional as F

    return F


# ------------------------------------------------------------------------------------------------ cases
def _quantize(rows, cols, block="row", dtype="bf16"):
    return dict(kind="quantize", rows=rows, cols=cols, block=block, dtype=dtype)


def _linear(m, k, n, dtype="bf16"):
    return dict(kind="linear", m=m, k=k, n=n, dtype=dtype)


def _train(m, k, n, dtype="fp16", bs=128, p=0.5):
    return dict(kind="train", m=m, k=k, n=n, dtype=dtype, bs=bs, p=p)


def _adamw(dims, layers, bits, dtype="fp32", step=10):
    """dims: features of one stack of layers, "784-1024-10"; every layer has its weights and a vector of as many elements as outputs."""
    return dict(kind="adamw", dims=dims, layers=layers, bits=bits, dtype=dtype, step=step)


def listed():
    return [
        # the activations of a few tokens, whose features end inside a block: what a call costs before the data does
        dict(_quantize(77, 1025), name="quantize 77 x 1025"),
        # the weights of a large square layer, as they are prepared once for serving or at every step in training
        dict(_quantize(8192, 8192, "square", "fp16"), name="quantize 8192 x 8192"),
        # serving: one token through the layer that leads a feed-forward block back to its width
        dict(_linear(1, 4096, 1024), name="linear 1 token"),
        # a batch of 200 requests, a token each, through a wide layer: too few rows to fill the chip, too many to only stream weights
        dict(_linear(200, 2048, 8192, "fp16"), name="linear 200 tokens"),
        # a long prompt through a large layer
        dict(_linear(8192, 8192, 8192), name="linear 8192 tokens"),
        # training: a small layer on a small batch
        dict(_train(128, 256, 256, p=0.1), name="train small"),
        # sizes nobody rounded: a batch as long as its data, features with one more appended, an odd number of outputs
        dict(_train(3001, 1025, 777, "bf16", p=0.3), name="train odd"),
        # the square layer that the package's headline step is about, half of its blocks dropped
        dict(_train(8192, 8192, 8192, p=0.5), name="train 8192"),
        # the update of a small classifier, ten outputs, averages in 32 bits
        dict(_adamw("784-1024-1024-10", 1, 32), name="adamw 32 bits classifier"),
        # the update of five feed-forward blocks in 16-bit parameters
        dict(_adamw("2048-8192-2048", 5, 32, "bf16"), name="adamw 32 bits blocks"),
        # averages in 8 bits: an odd classifier whose tensors end inside a block, and the same five feed-forward blocks
        dict(_adamw("777-1025-10", 1, 8), name="adamw 8 bits classifier"),
        dict(_adamw("2048-8192-2048", 5, 8), name="adamw 8 bits blocks"),
    ]


# What the listed cases stand for.  No drawn case does more work of its kind than the largest listed one.
_MOST = {"quantize": 8192 * 8192, "linear": 8192 ** 3, "train": 8192 ** 3 / 2, "adamw": 5 * 2 * 2048 * 8192}


def _size(rng, lo, hi, grain=1):
    """Spread over the logarithm of [lo, hi], a multiple of grain."""
    v = lo * (hi / lo) ** rng.random()
    return max(grain, int(v / grain + 0.5) * grain)


def draw(rng):
    kind = rng.choices(("quantize", "linear", "train", "adamw"), (2, 6, 6, 4))[0]
    while True:
        grain = rng.choice((64, 64, 8, 1))
        if kind == "quantize":
            c = _quantize(_size(rng, 1, 16384), _size(rng, 64, 8192, grain), rng.choice(("row", "square")), rng.choice(("fp16", "bf16", "fp32")))
            size = c["rows"] * c["cols"]
        elif kind == "linear":
            c = _linear(_size(rng, 1, 8192), _size(rng, 64, 8192, grain), _size(rng, 64, 8192, grain), rng.choice(("fp16", "bf16")))
            size = c["m"] * c["k"] * c["n"]
        elif kind == "train":
            c = _train(_size(rng, 64, 16384, rng.choice((64, 1))), _size(rng, 64, 8192, grain), _size(rng, 64, 8192, grain),
                       rng.choice(("fp16", "bf16")), rng.choice((128, 128, 128, 256, 384)), rng.choice((0.0, 0.1, 0.2, 0.3, 0.5, 0.75)))
            size = c["m"] * c["k"] * c["n"] * (1 - c["p"])
        else:
            d = _size(rng, 64, 2048, grain)
            dims = f"{d}-{4 * d}-{d}" if rng.random() < 0.5 else f"{_size(rng, 128, 4096, grain)}-{d}-{_size(rng, 10, 1000)}"
            c = _adamw(dims, rng.choice((1, 2, 3, 5)), rng.choice((8, 32)), rng.choice(("fp32", "fp32", "bf16", "fp16")), rng.choice((0, 1, 10, 1000, 100000)))
            size = c["layers"] * sum(i * o for i, o in _pairs(c))
        if size <= _MOST[kind]:
            return c


def _pairs(case):
    dims = [int(v) for v in case["dims"].split("-")]
    return list(zip(dims, dims[1:]))


def _blocks(n, bs=BLOCK):
    return -(-n // bs)


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev, dt = torch.device("cuda"), _DTYPES[case["dtype"]]
    gen = torch.Generator(dev).manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=gen, device=dev).mul_(std)

    def activations(m, k):
        """Normal, a few features twenty times as large as the others."""
        x = normal(m, k)
        x[:, torch.randint(k, (1 + k // 200,), generator=gen, device=dev)] *= 20
        return x.to(dt)

    if case["kind"] == "quantize":
        return dict(case=case, x=activations(case["rows"], case["cols"]))
    if case["kind"] == "linear":  # the weights are kept as they are served: codes and scales
        m, k, n = case["m"], case["k"], case["n"]
        data, scales = _quantize_square(normal(n, k, std=k ** -0.5).to(dt))
        return dict(case=case, x=activations(m, k), data=data, scales=scales)
    if case["kind"] == "train":
        m, k, n, bs = case["m"], case["k"], case["n"], case["bs"]
        return dict(case=case, x=activations(m, k).requires_grad_(), w=normal(n, k, std=k ** -0.5).to(dt).requires_grad_(),
                    dy=normal(m, n, std=0.01).to(dt),
                    mask=torch.rand(_blocks(m, bs), _blocks(k, bs), generator=gen, device=dev) < case["p"])
    s = dict(case=case, step=torch.full((), case["step"], dtype=torch.int64, device=dev), params=[], grads=[], first=[], second=[])
    for i, o in _pairs(case) * case["layers"]:
        for shape, std in (((o, i), i ** -0.5), ((o,), 1.0)):
            s["params"].append(normal(*shape, std=std).to(dt))
            s["grads"].append(normal(*shape, std=0.01).to(dt))
            first, second = normal(*shape, std=0.003), normal(*shape, std=0.01).square_()
            if case["step"] == 0:
                first, second = first.zero_(), second.zero_()
            if case["bits"] == 8:
                first, second = _encode(first, False, _half), _encode(second, True, _half)
            s["first"].append(first)
            s["second"].append(second)
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    return {"quantize": _run_quantize, "linear": _run_linear, "train": _run_train, "adamw": _run_adamw}[case["kind"]](state, case)


def _run_quantize(s, case):
    if own:
        data, scales = _package().fp8_quantize(s["x"], (1, 128) if case["block"] == "row" else (128, 128))
    else:
        data, scales = (_quantize_rows if case["block"] == "row" else _quantize_square)(s["x"])
    return {"data": data, "scales": scales}


def _run_linear(s, case):
    if own:
        return _package().fp8_linear(s["x"], s["data"], s["scales"])
    k = case["k"]
    w = _expand_square(s["data"], s["scales"])[:, :k]
    return (_expand_rows(*_quantize_rows(s["x"]))[:, :k] @ w.t()).to(s["x"].dtype)


def _run_train(s, case):
    if own:
        y = _package().hip_blockwise_dropout_matmul_fp8_mask(s["x"], s["mask"], case["bs"], case["p"], s["w"])
        return (y, *torch.autograd.grad(y, (s["x"], s["w"]), s["dy"]))
    with torch.no_grad():
        m, k, n, bs = case["m"], case["k"], case["n"], case["bs"]
        x, w, dy, dt = s["x"], _expand_square(*_quantize_square(s["w"]))[:, :k], s["dy"], s["x"].dtype
        keep = (~s["mask"]).repeat_interleave(bs, 0).repeat_interleave(bs, 1)[:m, :k].float() / (1 - case["p"])
        y = (_expand_rows(*_quantize_rows(x))[:, :k] * keep) @ w.t()
        dx = (_expand_rows(*_quantize_rows(dy))[:, :n] @ w) * keep
        # the weight gradient sums over the tokens: both of its operands have their blocks along the columns
        dw = _expand_rows(*_quantize_rows(dy.t()))[:, :m] @ (_expand_rows(*_quantize_rows(x.t()))[:, :m].t() * keep)
        return y.to(dt), dx.to(dt), dw.to(dt)


def _run_adamw(s, case):
    if own:
        F = _package()
        F.adamw_step(s["params"], s["grads"], s["first"], s["second"], s["step"], lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY)
        first, second = (s["first"], s["second"]) if case["bits"] == 32 else F.adamw_state_values(s["first"], s["second"])
        first, second = ([t.view(p.shape) for t, p in zip(ts, s["params"])] for ts in (first, second))
        return {"params": s["params"], "first": first, "second": second}
    s["step"] += 1
    t = s["step"].double()
    by, root = (LR / (1 - BETA1 ** t)).float(), (1 / torch.sqrt(1 - BETA2 ** t)).float()
    out = {"params": s["params"], "first": [], "second": []}
    for i, (p, g, first, second) in enumerate(zip(s["params"], s["grads"], s["first"], s["second"])):
        if case["bits"] == 32:
            g, m, v = g.float(), first, second
        else:  # in 64 bits: a value next to a border of its format goes to one side or the other
            g, m, v = g.double(), _decode(first, False, g.shape).double(), _decode(second, True, g.shape).double()
        m = m * BETA1 + g * (1 - BETA1)
        v = v * BETA2 + (g * g) * (1 - BETA2)
        p.copy_(p.float() * (1 - LR * DECAY) - by * (m.float() / (torch.sqrt(v.float()) * root + EPS)))
        if case["bits"] == 32:
            first.copy_(m), second.copy_(v)
        else:
            for kept, value, unsigned in ((first, m, False), (second, v, True)):
                codes, scales = _encode(value, unsigned, lambda n: _dither(n, s["step"], unsigned))
                kept[0].copy_(codes), kept[1].copy_(scales)
            m, v = _decode(first, False, g.shape), _decode(second, True, g.shape)
        out["first"].append(m)
        out["second"].append(v)
    return out


# ------------------------------------------------------------------------------------------------ the plain form's parts
def _exponent(most, limit):
    """The least e with most <= limit * 2^e, 0 where most is 0; limit: f * 2^a with f in [1/2, 1)."""
    f, a = math.frexp(limit)
    mantissa, e = torch.frexp(most)
    return torch.where(most > 0, e - a + (mantissa > f).int(), 0).clamp(-127, 127)


def _padded(x, rows):
    r, c = x.shape
    return torch.nn.functional.pad(x.float(), (0, -c % BLOCK, 0, -r % BLOCK if rows else 0))


def _power(e):
    return torch.ldexp(torch.ones((), device=e.device), e)


def _quantize_rows(x):
    x = _padded(x, False).view(x.shape[0], -1, BLOCK)
    e = _exponent(x.abs().amax(2), E4M3_MAX)
    return (x * _power(-e)[:, :, None]).to(torch.float8_e4m3fn).view(x.shape[0], -1), _power(e).to(torch.float8_e8m0fnu)


def _quantize_square(w):
    r = w.shape[0]
    w = _padded(w, True)
    w = w.view(w.shape[0] // BLOCK, BLOCK, w.shape[1] // BLOCK, BLOCK)
    e = _exponent(w.abs().amax((1, 3)), E4M3_MAX)
    q = (w * _power(-e)[:, None, :, None]).to(torch.float8_e4m3fn)
    return q.view(q.shape[0] * BLOCK, -1)[:r].contiguous(), _power(e).to(torch.float8_e8m0fnu)


def _expand_rows(data, scales):
    return (data.float().view(data.shape[0], -1, BLOCK) * scales.float()[:, :, None]).view(data.shape)


def _expand_square(data, scales):
    rows = scales.float().repeat_interleave(BLOCK, 0)[: data.shape[0]]
    return (data.float().view(data.shape[0], -1, BLOCK) * rows[:, :, None]).view(data.shape)


def _half(n):
    return 0.5


def _dither(n, step, low):
    """16 bits for each of n elements, over 2^16: those of M. O'Neill's permuted congruential generator (RXS-M-XS, 32 bits) one step behind
    the element's number plus the step's multiple of an odd constant; the high ones for the first average, the low ones for the second."""
    word = 0xFFFFFFFF
    s = (torch.arange(n, device=step.device) + step * 0x9E3779B1) & word
    s = (s * 747796405 + 2891336453) & word
    s = (((s >> ((s >> 28) + 4)) ^ s) * 277803737) & word
    s = (s >> 22) ^ s
    return ((s & 0xFFFF) if low else (s >> 16)).float() / 65536


def _encode(x, unsigned, dither):
    """(codes, scales), uint8: the values rounded down to the format's grid after `dither` of a grid step was added to their magnitude."""
    n = x.numel()
    limit, least, bias = (E5M3_MAX, -14, 15) if unsigned else (E4M3_MAX, -6, 7)
    x = torch.nn.functional.pad(x.reshape(-1), (0, -n % BLOCK)).view(-1, BLOCK)
    e = _exponent(x.abs().amax(1), limit)
    y = (x * torch.ldexp(torch.ones((), device=x.device, dtype=x.dtype), -e)[:, None]).view(-1)[:n]
    a = y.abs()
    at = (torch.frexp(a)[1] - 1).clamp_min(least)
    at = torch.where(a > 0, at, least)
    steps = torch.floor(torch.ldexp(a, 3 - at) + dither(n)).int()  # of 2^(at - 3): 8 and more of them for a normal number
    codes = steps + torch.where(at > least, (at + bias - 1) * 8, 0)
    if not unsigned:
        codes = codes + 128 * (y < 0).int()
    return codes.to(torch.uint8), (e + 127).to(torch.uint8)


def _decode(kept, unsigned, shape):
    codes, scales = kept[0].int(), kept[1].int()
    n = codes.numel()
    bias = 15 if unsigned else 7
    mag = codes if unsigned else codes & 127
    exponent, mantissa = mag >> 3, (mag & 7).float()
    value = torch.where(exponent > 0, torch.ldexp(mantissa + 8, exponent - bias - 3), torch.ldexp(mantissa, torch.full_like(exponent, 1 - bias - 3)))
    if not unsigned:
        value = torch.where(codes >= 128, -value, value)
    return torch.ldexp(value, (scales - 127).repeat_interleave(BLOCK)[:n]).view(shape)


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "quantize":
        side = 1 if case["block"] == "row" else BLOCK
        values, scales = _exact_blocks(s["x"].detach().double(), side)
        wide = torch.zeros(case["rows"], _blocks(case["cols"]) * BLOCK, dtype=torch.float64, device="cuda")
        by = scales.repeat_interleave(side, 0)[: case["rows"]].repeat_interleave(BLOCK, 1)
        wide[:, : case["cols"]] = values / by[:, : case["cols"]]
        return {"data": wide, "scales": scales}
    if case["kind"] == "linear":
        k, n = case["k"], case["n"]
        w = s["data"].double()[:, :k] * s["scales"].double().repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
        return _exact_blocks(s["x"].double(), 1)[0] @ w.t()
    if case["kind"] == "train":
        m, k, bs = case["m"], case["k"], case["bs"]
        x, dy, w = s["x"].detach().double(), s["dy"].double(), _exact_blocks(s["w"].detach().double(), BLOCK)[0]
        drop = torch.kron(s["mask"].double(), torch.ones(bs, bs, dtype=torch.float64, device="cuda"))[:m, :k]
        by = (1.0 - drop) / (1.0 - case["p"])
        y = (by * _exact_blocks(x, 1)[0]) @ w.t()
        dx = by * (_exact_blocks(dy, 1)[0] @ w)
        dw = _exact_blocks(dy.t(), 1)[0] @ (by * _exact_blocks(x.t(), 1)[0].t())
        return y, dx, dw
    t = case["step"] + 1
    out = {"params": [], "first": [], "second": []}
    for p, g, first, second in zip(s["params"], s["grads"], s["first"], s["second"]):
        p, g = p.double(), g.double()
        if case["bits"] == 8:
            first, second = _exact_state(first, False, p.shape), _exact_state(second, True, p.shape)
        m = BETA1 * first.double() + (1.0 - BETA1) * g
        v = BETA2 * second.double() + (1.0 - BETA2) * g * g
        out["params"].append(p - LR * DECAY * p - LR * (m / (1.0 - BETA1 ** t)) / ((v / (1.0 - BETA2 ** t)).sqrt() + EPS))
        if case["bits"] == 8:
            m, v = _exact_rounded(m, False, t), _exact_rounded(v, True, t)
        out["first"].append(m)
        out["second"].append(v)
    return out


def _exact_blocks(x, side):
    """The values that a matrix of 64-bit numbers has in 8 bits, and its scales: blocks of side x 128."""
    r, c = x.shape
    wide = torch.zeros(_blocks(r, side) * side, _blocks(c) * BLOCK, dtype=torch.float64, device=x.device)
    wide[:r, :c] = x
    tiles = wide.unfold(0, side, side).unfold(1, BLOCK, BLOCK)
    most = tiles.abs().amax((2, 3))
    scales = torch.exp2(torch.ceil(torch.log2(torch.where(most > 0, most, E4M3_MAX) / E4M3_MAX))).clamp(2.0 ** -127, 2.0 ** 127)
    # log2 near a whole number may have come out on its wrong side
    scales = torch.where(most > E4M3_MAX * scales, 2 * scales, scales)
    scales = torch.where((most <= E4M3_MAX * scales / 2) & (most > 0) & (scales > 2.0 ** -127), scales / 2, scales)
    y = wide / scales.repeat_interleave(side, 0).repeat_interleave(BLOCK, 1)
    grid = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    y = torch.round(y / grid) * grid  # (halves go to the even one)
    y = y * scales.repeat_interleave(side, 0).repeat_interleave(BLOCK, 1)
    return y[:r, :c], scales


def _table(unsigned):
    """The 256 values of a format."""
    bits, bias = (5, 15) if unsigned else (4, 7)
    half = [(j / 8 * 2.0 ** (1 - bias)) if i == 0 else (1 + j / 8) * 2.0 ** (i - bias) for i in range(1 << bits) for j in range(8)]
    return torch.tensor(half if unsigned else half + [-v for v in half], dtype=torch.float64, device="cuda")


def _exact_state(kept, unsigned, shape):
    codes, scales = kept
    return (_table(unsigned)[codes.long()] * torch.exp2(scales.double().repeat_interleave(BLOCK)[: codes.numel()] - 127)).view(shape)


def _exact_rounded(x, unsigned, t):
    """An average's values after it was put into 8 bits at step t."""
    limit, least = (E5M3_MAX, 2.0 ** -14) if unsigned else (E4M3_MAX, 2.0 ** -6)
    flat, n = x.reshape(-1), x.numel()
    wide = torch.zeros(_blocks(n) * BLOCK, dtype=torch.float64, device=x.device)
    wide[:n] = flat.abs()
    most = wide.view(-1, BLOCK).amax(1)
    scales = torch.exp2(torch.ceil(torch.log2(torch.where(most > 0, most, limit) / limit)))
    scales = torch.where(most > limit * scales, 2 * scales, scales)
    scales = torch.where((most <= limit * scales / 2) & (most > 0), scales / 2, scales).repeat_interleave(BLOCK)[:n]
    y = flat.abs() / scales
    grid = torch.exp2(torch.floor(torch.log2(y.clamp_min(least))) - 3)
    u = _dither(n, torch.tensor(t, device=x.device), unsigned).double()
    return (torch.floor(y / grid + u) * grid * scales * flat.sign()).view(x.shape)


# ------------------------------------------------------------------------------------------------ bounds
def work(case):
    """What is held in 8 bits is a byte and its share of a scale's; dropped blocks are not read, dropped blocks of a gradient are
    written (zeros)."""
    size = 4.0 if case["dtype"] == "fp32" else 2.0
    if case["kind"] == "quantize":
        r, c = case["rows"], case["cols"]
        return {"bytes": (size + 1) * r * c + (r if case["block"] == "row" else _blocks(r)) * _blocks(c), "flops": 2.0 * r * c}
    if case["kind"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        return {"bytes": 2.0 * m * k + n * k + _blocks(n) * _blocks(k) + 2.0 * m * n, "flops": 2.0 * m * k * n}
    if case["kind"] == "train":
        m, k, n, keep = case["m"], case["k"], case["n"], 1.0 - case["p"]
        return {"bytes": 2.0 * (m * k * keep + n * k + 2 * m * n + m * k + n * k), "flops": 6.0 * m * k * n * keep}
    n = case["layers"] * sum(i * o + o for i, o in _pairs(case))
    # parameters read and written, gradients read, both averages read and written; those in 8 bits are also returned as values
    each = 3 * size + (16.0 if case["bits"] == 32 else 4.0 * (1 + 1 / BLOCK) + 8.0)
    return {"bytes": each * n, "flops": 15.0 * n}
