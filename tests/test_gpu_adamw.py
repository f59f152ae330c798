"""The AdamW step on the GPU against its formulas in 64 bits.

Tolerances, relative to the terms' magnitudes: in 32 bits an average is two products and a sum, each off by half a step (2^-24), and its
factors are rounded: at most 4 * 2^-24 of either term.  The update lr' * m / (sqrt(v) * r + eps) has m and the root of v (v's
error counts half), three factors rounded to 32 bits, and six roundings, none by more than 2^-24 (2^-23 for the root and the quotient):
16 * 2^-24 of itself covers them.  The parameter is one product and a difference more and is rounded to its type.  Averages in 8 bits are
computed in 64 bits and put on their grid: equal values."""
import numpy as np
import pytest
import torch

from oracle import fp8_oracle as O

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import flash_dropout.functional as F
    from flash_dropout.hip import GEMM  # noqa: F401
    from flash_dropout.optim import AdamW

HYPER = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def np64(t):
    return t.detach().double().cpu().numpy()


def spread(n, seed, std=1.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(n, generator=gen) * std * 2.0 ** torch.randint(-10, 5, (n,), generator=gen)
    x[torch.rand(n, generator=gen) < 0.05] = 0
    return x


def codes_of(x, which, step=0):
    """An average's codes and scales, made from its values in 8 bits."""
    limit = O.FORMATS[which][0]
    values = O.rounded_state(np64(x), which, step).reshape(-1)
    wide = np.zeros(-(-values.size // 128) * 128)
    wide[: values.size] = np.abs(values)
    scales = O.least_power(wide.reshape(-1, 128).max(1), limit)
    table = O.state_table(which)
    order = np.argsort(np.where(np.isfinite(table), table, np.inf))[: np.isfinite(table).sum()]
    at = np.searchsorted(table[order], values / np.repeat(scales, 128)[: values.size])
    codes = order[np.minimum(at, len(order) - 1)]
    assert np.array_equal(table[codes] * np.repeat(scales, 128)[: values.size], values)
    return torch.from_numpy(codes.astype(np.uint8)).cuda(), torch.from_numpy((np.log2(scales) + 127).astype(np.uint8)).cuda()


def check_param(got, p, g, m, v, step, dtype, hyper=HYPER):
    lr, (b1, b2), eps, decay = (hyper[k] for k in ("lr", "betas", "eps", "weight_decay"))
    ref, _, _ = O.adamw(np64(p), np64(g), m, v, step, lr, b1, b2, eps, decay)
    # what the first average's error of 4 * 2^-24 of its terms moves the parameter by, and the update's own
    terms = b1 * np.abs(m) + (1 - b1) * np.abs(np64(g))
    root = np.sqrt((b2 * v + (1 - b2) * np64(g) ** 2) / (1 - b2 ** step)) + eps
    info = torch.finfo(dtype)
    with np.errstate(invalid="ignore", divide="ignore"):
        tol = 24 * 2.0 ** -24 * lr * terms / (1 - b1 ** step) / root + 3 * 2.0 ** -24 * np.abs(np64(p))
    tol += (info.eps / 2) * np.abs(ref) * (1 + info.eps) + info.smallest_normal * info.eps / 2 + 2.0 ** -149
    got = np64(got)
    # (a first average without a second is divided by eps alone; from half a step above the largest number on, a value rounds to infinity)
    over = np.isinf(got) & (np.sign(got) == np.sign(ref)) & (np.abs(ref) + tol >= info.max * (1 + info.eps / 4))
    assert (over | (np.abs(got - ref) <= tol)).all()


SIZES = [(1,), (127,), (128,), (129,), (1000,), (33, 65), (3, 7, 5, 5), (2048,), (2049,), (70000,)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("step", [0, 1, 1000])
def test_averages_in_32_bits(step, dtype):
    dt = DT[dtype]
    p = [spread(int(np.prod(s)), 10 + i).view(s).to(dt).cuda() for i, s in enumerate(SIZES)]
    g = [spread(int(np.prod(s)), 40 + i, 0.1).view(s).to(dt).cuda() for i, s in enumerate(SIZES)]
    m = [(spread(int(np.prod(s)), 70 + i, 0.1).view(s) * (step > 0)).cuda() for i, s in enumerate(SIZES)]
    v = [(spread(int(np.prod(s)), 90 + i, 0.1).view(s).square() * (step > 0)).cuda() for i, s in enumerate(SIZES)]
    before = [[t.clone() for t in ts] for ts in (p, g, m, v)]
    count = torch.tensor(step, device="cuda")
    F.adamw_step(p, g, m, v, count, **HYPER)
    assert count.item() == step + 1
    b1, b2 = HYPER["betas"]
    for i in range(len(SIZES)):
        p0, g0, m0, v0 = (b[i] for b in before)
        assert torch.equal(g[i], g0)
        rm, rv = b1 * np64(m0) + (1 - b1) * np64(g0), b2 * np64(v0) + (1 - b2) * np64(g0) ** 2
        assert (np.abs(np64(m[i]) - rm) <= 4 * 2.0 ** -24 * (b1 * np.abs(np64(m0)) + (1 - b1) * np.abs(np64(g0))) + 2.0 ** -149).all()
        assert (np.abs(np64(v[i]) - rv) <= 4 * 2.0 ** -24 * rv + 2.0 ** -149).all()
        check_param(p[i], p0, g0, np64(m0), np64(v0), step + 1, dt)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("step", [0, 3, 50000])
def test_averages_in_8_bits_are_those_of_the_definition(step, dtype):
    dt = DT[dtype]
    sizes = [int(np.prod(s)) for s in SIZES]
    p = [spread(n, 10 + i).to(dt).cuda() for i, n in enumerate(sizes)]
    g = [spread(n, 40 + i, 0.1).to(dt).cuda() for i, n in enumerate(sizes)]
    m = [codes_of(spread(n, 70 + i, 0.1) * (step > 0), "first") for i, n in enumerate(sizes)]
    v = [codes_of(spread(n, 90 + i, 0.1).square() * (step > 0), "second") for i, n in enumerate(sizes)]
    m0, v0 = ([np64(t) for t in ts] for ts in F.adamw_state_values(m, v))
    for (codes, scales), values, which in [(a, b, "first") for a, b in zip(m, m0)] + [(a, b, "second") for a, b in zip(v, v0)]:
        by = np.exp2(np64(scales) - 127).repeat(128)[: codes.numel()]
        assert np.array_equal(O.state_table(which)[codes.cpu().numpy()] * by, values)
    before = [t.clone() for t in p]
    count = torch.tensor(step, device="cuda")
    F.adamw_step(p, g, m, v, count, **HYPER)
    assert count.item() == step + 1
    m1, v1 = F.adamw_state_values(m, v)
    b1, b2 = HYPER["betas"]
    for i in range(len(sizes)):
        rm, rv = b1 * m0[i] + (1 - b1) * np64(g[i]), b2 * v0[i] + (1 - b2) * np64(g[i]) ** 2
        assert np.array_equal(np64(m1[i]), O.rounded_state(rm, "first", step + 1))
        assert np.array_equal(np64(v1[i]), O.rounded_state(rv, "second", step + 1))
        check_param(p[i], before[i], g[i], m0[i], v0[i], step + 1, dt)


def test_averages_in_8_bits_follow_slow_changes():
    """A gradient of twice the size that the second average stands for moves it, over many steps, to where 32 bits move it: each
    step is a hundredth of a code's distance."""
    n, beta2, steps = 128 * 64, 0.999, 400
    g = torch.full((n,), 2.0, device="cuda")
    p = torch.zeros(n, device="cuda")
    m, v = codes_of(torch.full((n,), 1.0), "first"), codes_of(torch.full((n,), 1.0), "second")
    count = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(steps):
        F.adamw_step([p], [g], [m], [v], count, lr=0.0, betas=(0.9, beta2), weight_decay=0.0)
    want = 4 - 3 * beta2 ** steps
    got = np64(F.adamw_state_values([m], [v])[1][0])
    # a rounding's variance is at most a quarter of a grid step (at most 1/4 here) squared, decayed: the mean over n elements of a
    # sum of `steps` such is off by 6 standard deviations with a probability below 1e-8
    assert abs(got.mean() - want) <= 6 * 0.125 * steps ** 0.5 / n ** 0.5


def test_what_is_not_finite_stays_with_its_element():
    n = 400
    p, g = spread(n, 1).cuda(), spread(n, 2).cuda()
    g[5], g[200], g[399] = float("nan"), float("inf"), float("-inf")
    m, v = codes_of(torch.zeros(n), "first"), codes_of(torch.zeros(n), "second")
    clean = torch.where(g.isfinite(), g, torch.zeros_like(g))
    pc, mc, vc = p.clone(), codes_of(torch.zeros(n), "first"), codes_of(torch.zeros(n), "second")
    F.adamw_step([p], [g], [m], [v], torch.zeros((), dtype=torch.int64, device="cuda"), **HYPER)
    F.adamw_step([pc], [clean], [mc], [vc], torch.zeros((), dtype=torch.int64, device="cuda"), **HYPER)
    (got,), (gotv,) = F.adamw_state_values([m], [v])
    (want,), (wantv,) = F.adamw_state_values([mc], [vc])
    fine = g.isfinite()
    for a, b in ((p, pc), (got, want), (gotv, wantv)):
        assert torch.equal(a[fine], b[fine])
    assert got[~fine].isnan().all() and gotv[5].isnan() and gotv[200].isinf() and gotv[399].isinf()


def test_many_tensors_of_mixed_types_and_a_step_without_any():
    kinds = [("fp32", "bf16", "fp16")[i % 3] for i in range(190)]
    sizes = [1 + 37 * i % 400 for i in range(190)]
    sizes[7] = 0
    p = [spread(n, i).to(DT[k]).cuda() for i, (n, k) in enumerate(zip(sizes, kinds))]
    g = [spread(n, 300 + i).to(DT[k]).cuda() for i, (n, k) in enumerate(zip(sizes, kinds))]
    m = [torch.zeros(n, device="cuda") for n in sizes]
    v = [torch.zeros(n, device="cuda") for n in sizes]
    before = [t.clone() for t in p]
    count = torch.zeros(1, dtype=torch.int64, device="cuda")
    versions = [t._version for t in (p[0], m[0], v[0], count)]
    F.adamw_step(p, g, m, v, count, **HYPER)
    assert count.item() == 1
    assert all(t._version > o for t, o in zip((p[0], m[0], v[0], count), versions))
    for i in range(190):
        check_param(p[i], before[i], g[i], np.zeros(sizes[i]), np.zeros(sizes[i]), 1, DT[kinds[i]])
    F.adamw_step([], [], [], [], count, **HYPER)
    assert count.item() == 2
    # a launch's table of tensors with elements, then only tensors without any
    some = lambda std: [torch.full((5,), std, device="cuda") for _ in range(56)] + [torch.zeros(0, device="cuda") for _ in range(3)]
    p, g, m, v = some(1.0), some(0.5), some(0.0), some(0.0)
    count.zero_()
    F.adamw_step(p, g, m, v, count, lr=0.25, weight_decay=0.0)
    assert count.item() == 1
    for t in p[:56]:  # one step of lr against a gradient of one sign
        assert ((t - 0.75).abs() <= 32 * 2.0 ** -24).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_memory_formats_and_unaligned_views(bits):
    w = spread(8 * 6 * 3 * 3, 5).view(8, 6, 3, 3).cuda().contiguous(memory_format=torch.channels_last)
    flat = spread(1001, 6).cuda()
    p = [w, flat[1:1000], spread(35 * 17, 7).view(35, 17).cuda().t()]
    g = [spread(t.numel(), 20 + i).view(t.shape).cuda() for i, t in enumerate(p)]  # (the first and last laid out otherwise)
    before = [t.clone() for t in p]
    if bits == 32:
        m, v = ([torch.zeros_like(t) for t in p] for _ in range(2))
    else:
        m, v = ([codes_of(torch.zeros(t.numel()), k) for t in p] for k in ("first", "second"))
    ends = flat[0].clone(), flat[1000].clone()
    F.adamw_step(p, g, m, v, torch.zeros((), dtype=torch.int64, device="cuda"), **HYPER)
    for a, b, c in zip(p, before, g):
        check_param(a, b, c, np.zeros(tuple(a.shape)), np.zeros(tuple(a.shape)), 1, torch.float32)
    assert torch.equal(flat[0], ends[0]) and torch.equal(flat[1000], ends[1])


def test_large_tensor():
    n = 128 * 50_000 + 3
    p, g = torch.zeros(n, device="cuda"), torch.randn(n, device="cuda")
    m, v = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    F.adamw_step([p], [g], [m], [v], torch.zeros((), dtype=torch.int64, device="cuda"), lr=1.0, weight_decay=0.0)
    want = -(g.double() / (g.double().abs() + 1e-8))  # (the corrected averages of one step are g and g^2)
    assert ((p.double() - want).abs() <= 24 * 2.0 ** -24).all()
    assert ((m.double() - 0.1 * g.double()).abs() <= 4 * 2.0 ** -24 * 0.1 * g.double().abs() + 2.0 ** -149).all()


def test_averages_in_8_bits_next_to_a_random_border():
    """0.9 m + 0.1 g is a multiple of the border's 2^-16 of a step, but for the last bits of 64, wherever 9 m + g is one of ten: either
    neighbour is right there, and the code is the one that the formula gives in torch, whose ldexp multiplies by pow(2, k)."""
    n = 128 * 4096
    gen = torch.Generator().manual_seed(3)
    m0 = torch.randint(8, 16, (n,), generator=gen).float() * torch.where(torch.rand(n, generator=gen) < 0.5, -1.0, 1.0)
    g = torch.randint(-200, 200, (n,), generator=gen).float()
    g = g + (-(9 * m0 + g)) % 5  # (9 m + g) / 10: a whole number of halves
    m0[::128], g[::128] = 15.0, 5.0
    m, v = codes_of(m0, "first"), codes_of(torch.zeros(n), "second")
    assert np.array_equal(np64(F.adamw_state_values([m], [v])[0][0]), np64(m0))
    F.adamw_step([torch.zeros(n, device="cuda")], [g.cuda()], [m], [v], torch.full((), 6, dtype=torch.int64, device="cuda"), betas=(0.9, 0.99))
    got, x = np64(F.adamw_state_values([m], [v])[0][0]), 0.9 * np64(m0) + (1 - 0.9) * np64(g)
    want = O.rounded_state(x, "first", 7)
    scales = np.repeat(np.exp2(np64(m[1]) - 127), 128)
    y = torch.from_numpy(np.abs(x)).cuda() * torch.ldexp(torch.ones(n, dtype=torch.float64, device="cuda"), 127 - m[1].int().repeat_interleave(128))
    at = (torch.frexp(y)[1] - 1).clamp_min(-6)
    in_torch = np64(torch.floor(torch.ldexp(y, 3 - at) + torch.from_numpy(O.dither(n, 7, "first")).cuda())) * np.exp2(np64(at) - 3) * scales
    grid = np.exp2(np.floor(np.log2(np.maximum(np.abs(x) / scales, 2.0 ** -6))) - 3)
    z = np.abs(x) / scales / grid + O.dither(n, 7, "first")
    border = np.abs(z - np.rint(z)) < 2.0 ** -40
    assert border.any() and not border.all()
    assert np.array_equal(got[~border], want[~border])
    assert np.array_equal(np.abs(got), in_torch)
    assert (np.abs(got - want) <= grid * scales).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_step_replays(bits):
    n = 5000
    p, g = spread(n, 1).cuda(), spread(n, 2).cuda()
    lr = torch.full((), 1e-2, device="cuda")

    def states():
        if bits == 32:
            return [torch.zeros(n, device="cuda")], [torch.zeros(n, device="cuda")]
        return [codes_of(torch.zeros(n), "first")], [codes_of(torch.zeros(n), "second")]

    pe, (me, ve), ce = p.clone(), states(), torch.zeros((), dtype=torch.int64, device="cuda")
    (m, v), c = states(), torch.zeros((), dtype=torch.int64, device="cuda")
    graph = torch.cuda.CUDAGraph()
    F.adamw_step([torch.zeros(4, device="cuda")], [torch.zeros(4, device="cuda")], [torch.zeros(4, device="cuda")], [torch.zeros(4, device="cuda")],
                 torch.zeros((), dtype=torch.int64, device="cuda"))
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        F.adamw_step([p], [g], m, v, c, lr=lr)
    assert c.item() == 0
    for i in range(3):
        g.copy_(spread(n, 50 + i))
        lr.fill_(1e-2 / (i + 1))
        graph.replay()
        F.adamw_step([pe], [g], me, ve, ce, lr=lr)
        assert torch.equal(p, pe) and c.item() == ce.item() == i + 1
        for a, b in zip(m + v, me + ve):
            assert all(torch.equal(x, y) for x, y in zip(a, b)) if bits == 8 else torch.equal(a, b)


# ---- the optimizer ------------------------------------------------------------------------------------------------------------
def model(seed=0):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Linear(300, 130), torch.nn.ReLU(), torch.nn.Linear(130, 10)).cuda()


def gradients(net, seed):
    for i, q in enumerate(net.parameters()):
        q.grad = spread(q.numel(), 100 * seed + i, 0.1).view(q.shape).to(q.dtype).cuda()


def test_the_optimizer_steps_like_torchs():
    a, b = model(), model()
    ours, torchs = AdamW(a.parameters(), lr=1e-2, weight_decay=0.1), torch.optim.AdamW(b.parameters(), lr=1e-2, weight_decay=0.1)
    for i in range(5):
        for net in (a, b):
            gradients(net, i)
        if i in (1, 3):  # one parameter sits a step out
            a[0].bias.grad = b[0].bias.grad = None
        ours.step()
        torchs.step()
    for x, y in zip(a.parameters(), b.parameters()):
        # five steps of about lr each, their relative errors (see above) of both sides
        assert (x - y).abs().max() <= 2 * 5 * (24 * 1e-2 * 4 + 3 * float(y.abs().max())) * 2.0 ** -24
    assert ours.state[a[0].bias]["step"].item() == 3 and ours.state[a[0].weight]["step"].item() == 5


@pytest.mark.parametrize("bits", [32, 8])
def test_a_saved_optimizer_goes_on_where_it_was(bits, tmp_path):
    a = model().bfloat16() if bits == 8 else model()
    opt = AdamW(a.parameters(), lr=1e-2, state_bits=bits)
    dt = next(a.parameters()).dtype
    for i in range(3):
        gradients(a, i)
        if i == 1:
            a[2].bias.grad = None
        opt.step()
    torch.save({"opt": opt.state_dict(), "net": a.state_dict()}, tmp_path / "s.pt")
    saved = torch.load(tmp_path / "s.pt", weights_only=True)
    b = model(1).to(dt)
    b.load_state_dict(saved["net"])
    again = AdamW(b.parameters(), lr=5.0, state_bits=bits)
    again.load_state_dict(saved["opt"])
    for i in range(3, 5):
        for net, o in ((a, opt), (b, again)):
            for j, q in enumerate(net.parameters()):
                q.grad = spread(q.numel(), 10 * i + j).view(q.shape).to(dt).cuda()
            o.step()
    for x, y in zip(a.parameters(), b.parameters()):
        assert torch.equal(x, y)
        assert opt.state[x]["step"].item() == again.state[y]["step"].item()
        for s, t in zip(opt.state_values(x), again.state_values(y)):
            assert torch.equal(s, t) and s.shape == x.shape
    assert opt.state[a[2].bias]["step"].item() == 4


def test_refusals():
    z = lambda *s, **k: torch.zeros(*s, device="cuda", **k)
    count = z((), dtype=torch.int64)
    ok = [z(130)], [z(130)], [z(130)], [z(130)]
    F.adamw_step(*ok, count)
    for bad in (([z(130)], [z(131)], [z(130)], [z(130)]), ([z(130)], [], [z(130)], [z(130)]), ([z(130)], [z(130)], [z(13, 10)], [z(130)]),
                ([z(260)[::2]], [z(130)], [z(130)], [z(130)]), ([z(130)], [z(130)], [z(130).half()], [z(130)]),
                ([ok[0][0]] * 2, ok[1] * 2, [z(130), z(130)], [z(130), z(130)]),
                ([z(130)], [z(130)], [(z(130, dtype=torch.uint8), z(1, dtype=torch.uint8))], [(z(130, dtype=torch.uint8), z(1, dtype=torch.uint8))]),
                ([z(130)], [z(130)], [(z(130, dtype=torch.uint8), z(2, dtype=torch.uint8))], [z(130)])):
        with pytest.raises(ValueError):
            F.adamw_step(*bad, count)
    for kind in (torch.float64, torch.int32):
        with pytest.raises(TypeError):
            F.adamw_step([z(130, dtype=kind)], [z(130, dtype=kind)], [z(130)], [z(130)], count)
    with pytest.raises(TypeError):
        F.adamw_step([z(130)], [z(130).half()], [z(130)], [z(130)], count)
    for step in (torch.zeros((), dtype=torch.int64), z(()), z(2, dtype=torch.int64)):
        with pytest.raises(ValueError):
            F.adamw_step(*ok, step)
    for kw in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1.0), dict(weight_decay=-1.0), dict(lr=float("nan")),
               dict(lr=z((), dtype=torch.float64))):
        with pytest.raises(ValueError):
            F.adamw_step(*ok, count, **kw)
    with pytest.raises(ValueError):
        F.adamw_state_values(ok[2], ok[3])
    with pytest.raises(ValueError):
        AdamW([z(3)], state_bits=16)
    assert count.item() == 1


def test_tensors_that_share_memory_are_refused():
    """Each written tensor is nobody else's, scales and parts of a buffer included; gradients may be shared, and neighbours touch."""
    z = lambda *s, **k: torch.zeros(*s, device="cuda", **k)
    count = z((), dtype=torch.int64)
    flat, grad, m, v = z(512), torch.ones(512, device="cuda"), z(512), z(512)
    F.adamw_step([flat[:256], flat[256:]], [grad[:256], grad[:256]], [m[:256], m[256:]], [v[:256], v[256:]], count)
    assert count.item() == 1 and flat.all()
    codes = lambda n=256: (z(n, dtype=torch.uint8), torch.full((-(-n // 128),), 127, dtype=torch.uint8, device="cuda"))
    a, b, c, d = codes(), codes(), codes(), codes()
    shared = (c[0], a[1])
    before = [t.clone() for t in (flat, m, v, *a, *b, *c, *d)]
    for bad in (([flat[:256], flat[128:384]], [grad[:256]] * 2, [m[:256], m[256:]], [v[:256], v[256:]]),
                ([flat[:256], flat[256:]], [grad[:256]] * 2, [m[:256], m[255:511]], [v[:256], v[256:]]),
                ([flat[:256]], [grad[:256]], [m[:256]], [m[128:384]]),
                ([flat[:256]], [grad[:256]], [flat[256:]], [flat[255:511]]),
                ([flat[:256], flat[256:]], [grad[:256], flat[:256]], [m[:256], m[256:]], [v[:256], v[256:]]),
                ([flat[:256]], [m[100:356]], [m[:256]], [v[:256]]),
                ([flat[:256], flat[256:]], [grad[:256]] * 2, [a, shared], [b, d]),
                ([flat[:256]], [grad[:256]], [a], [(b[0], a[1])])):
        with pytest.raises(ValueError, match="share memory"):
            F.adamw_step(*bad, count)
    assert count.item() == 1
    assert all(torch.equal(s, t) for s, t in zip(before, (flat, m, v, *a, *b, *c, *d)))
    F.adamw_step([flat[:256], flat[256:]], [grad[:256]] * 2, [a, c], [b, d], count)
    assert count.item() == 2 and all(t[0].any() for t in (a, b, c, d))
    own = torch.full((300,), 2.0, device="cuda")  # a parameter that is its own gradient
    F.adamw_step([own], [own], [z(300)], [z(300)], z((), dtype=torch.int64), lr=0.5, eps=0.0, weight_decay=0.0)
    assert ((own - 1.5).abs() <= 24 * 2.0 ** -24).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_averages_are_laid_out_like_their_parameters(bits):
    """Steps, values, a save and a load of a channels-last and a turned parameter equal those of contiguous ones with each element's own
    gradient; a parameter that is laid out anew keeps none of its averages' codes."""
    shape = (24, 5, 3, 3)
    w, g = spread(24 * 45, 1).view(shape).cuda(), spread(24 * 45, 2, 0.1).view(shape).cuda()
    p = torch.nn.Parameter(w.clone().contiguous(memory_format=torch.channels_last))
    flat = torch.nn.Parameter(w.permute(0, 2, 3, 1).contiguous().view(-1))  # the same memory
    opts = [AdamW([t], lr=1e-2, state_bits=bits) for t in (p, flat)]
    for i in range(3):
        p.grad = (g * (i + 1)).contiguous()
        flat.grad = (g * (i + 1)).permute(0, 2, 3, 1).contiguous().view(-1)
        for o in opts:
            o.step()
        if i == 1:
            state = opts[0].state_dict()
            opts[0] = AdamW([p], lr=5.0, state_bits=bits)
            opts[0].load_state_dict(state)
    assert torch.equal(p.detach().permute(0, 2, 3, 1).reshape(-1), flat.detach())
    for a, b in zip(opts[0].state_values(p), opts[1].state_values(flat)):
        assert a.shape == p.shape and a.stride() == p.stride() and torch.equal(a.permute(0, 2, 3, 1).reshape(-1), b)
    before = [t.clone() for t in opts[0].state_values(p)]
    p.data = p.data.contiguous()
    kept = p.detach().clone()
    with pytest.raises(ValueError, match="laid out"):
        opts[0].step()
    assert torch.equal(p, kept) and all(torch.equal(a, b) for a, b in zip(before, opts[0].state_values(p)))


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype,sizes,chunks", [
    # workgroups of 1024 threads that take four runs of 2048 elements at a time, from a few hundred runs to the most
    ("fp32", (700_001, 300, 12_345, 128, 390_625), 542), ("bf16", (5, 1_049_600, 2047), 515), ("fp16", (16_000_001, 771_000, 999), 8191),
    # 8 bits: workgroups of 256 through several runs each
    ("fp32", (129, 33_600_003, 5_000), 16411)])
def test_many_elements_over_several_tensors(dtype, sizes, chunks, bits):
    """A second step from averages that a first one left, every element of every tensor checked.  Averages in 8 bits are those of the
    definition, but where their place between two codes and the random bits make a whole number within 2^-40: there either neighbour is right."""
    assert sum(-(-n // 2048) for n in sizes) == chunks
    dt, (b1, b2) = DT[dtype], HYPER["betas"]
    p = [spread(n, 10 + i).to(dt).cuda() for i, n in enumerate(sizes)]
    m, v = ([torch.zeros(n, device="cuda") if bits == 32 else codes_of(torch.zeros(n), k) for n in sizes] for k in ("first", "second"))
    count = torch.zeros((), dtype=torch.int64, device="cuda")
    values = lambda: (m, v) if bits == 32 else F.adamw_state_values(m, v)  # noqa: E731
    for step in (1, 2):
        g = [spread(n, 40 + 10 * step + i, 0.1).to(dt).cuda() for i, n in enumerate(sizes)]
        before, (m0, v0) = [t.clone() for t in p], ([t.clone() for t in ts] for ts in values())
        F.adamw_step(p, g, m, v, count, **HYPER)
        assert count.item() == step
    for i, (m1, v1) in enumerate(zip(*values())):
        check_param(p[i], before[i], g[i], np64(m0[i]), np64(v0[i]), 2, dt)
        gd = np64(g[i])
        for which, got, old, new, b in (("first", m1, m0[i], gd, b1), ("second", v1, v0[i], gd * gd, b2)):
            x, got = b * np64(old) + (1 - b) * new, np64(got)
            if bits == 32:
                assert (np.abs(got - x) <= 4 * 2.0 ** -24 * (b * np.abs(np64(old)) + (1 - b) * np.abs(new)) + 2.0 ** -149).all()
                continue
            want = O.rounded_state(x, which, 2)
            at = np.flatnonzero(got != want)
            if at.size:
                limit, least, _ = O.FORMATS[which]
                wide = np.zeros(-(-x.size // 128) * 128)
                wide[: x.size] = np.abs(x)
                y = np.abs(x[at]) / O.least_power(wide.reshape(-1, 128).max(1), limit)[at // 128]
                grid = np.exp2(np.floor(np.log2(np.maximum(y, least))) - 3)
                z = y / grid + O.dither(x.size, 2, which)[at]
                assert (np.abs(z - np.rint(z)) < 2.0 ** -40).all()
                assert (np.abs(got[at] - want[at]) <= grid * (np.abs(x[at]) / y)).all()
