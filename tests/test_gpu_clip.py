"""The norm of many gradients and their clipping on the GPU against the formulas in 64 bits.

Tolerances.  The norm is summed in 64 bits (n 2^-53 of itself, nothing here) and rounded to 32 once: 2^-24.  The factor is rounded to 32 bits and
multiplied in 32 bits, 2^-24 each, and the result rounded to its type once, eps / 2 or half of the smallest subnormal."""
import copy
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import flash_dropout.functional as F
    from flash_dropout.optim import AdamW, clip_grad_norm_

DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SIZES = [(1,), (0,), (3,), (7, 9), (8191,), (8192,), (8193,), (16384,), (33, 65), (1, 1), (70001,), (10, 1024), (2, 3, 5, 7)]


def gradients(dtypes, sizes=SIZES, seed=0, std=1.0):
    gen = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=gen) * std * 2.0 ** float(torch.randint(-6, 3, (1,), generator=gen))).to(DT[dtypes[i % len(dtypes)]]).cuda()
            for i, s in enumerate(sizes)]


def norm64(grads, kind=2.0):
    flat = [g.detach().double().cpu().flatten().numpy() for g in grads]
    flat = np.concatenate(flat)
    return float(np.sqrt((flat ** 2).sum())) if kind == 2.0 else float(np.abs(flat).max()) if flat.size else 0.0


def close(got, ref, dtype):
    info = torch.finfo(dtype)
    tol = (2.0 ** -23 + (info.eps / 2 if dtype != torch.float32 else 0)) * ref.abs() * (1 + 2.0 ** -10) + info.smallest_normal * info.eps / 2
    return bool(((got.detach().double() - ref).abs() <= tol).all())


@pytest.mark.parametrize("dtypes", [("fp32",), ("fp16",), ("bf16",), ("fp32", "bf16", "fp16")], ids="-".join)
@pytest.mark.parametrize("kind", [2.0, math.inf])
@pytest.mark.parametrize("limit", [0.0, 0.1, 3.0, 1e9])
def test_norm_and_clip(dtypes, kind, limit):
    grads = gradients(dtypes)
    ref = norm64(grads, kind)
    by = min(1.0, limit / (ref + 1e-6))
    norm, factor = F.grad_norm(grads, kind, limit)
    assert norm.dtype == torch.float32 and norm.dim() == 0 and abs(float(norm) - ref) <= 2.0 ** -23 * ref
    assert abs(float(factor) - by) <= 2.0 ** -23 * by
    assert torch.equal(F.grad_norm(grads, kind), norm)
    before = [g.clone() for g in grads]
    versions = [g._version for g in grads]
    got = F.clip_grad_norm_(grads, limit, kind)
    assert torch.equal(got, norm)
    for g, b, v in zip(grads, before, versions):
        assert close(g, b.double() * by, g.dtype) and g._version > v
        if by == 1.0:
            assert torch.equal(g, b)


@pytest.mark.parametrize("count", [1, 175, 176, 177, 1000, 3000])
def test_many_tensors(count):
    grads = gradients(("fp32", "bf16"), [(1 + 37 * i % 20000,) for i in range(count)], seed=1)
    ref = norm64(grads)
    before = [g.clone() for g in grads]
    assert abs(float(F.clip_grad_norm_(grads, 1.0)) - ref) <= 2.0 ** -23 * ref
    by = min(1.0, 1.0 / (ref + 1e-6))
    assert all(close(g, b.double() * by, g.dtype) for g, b in zip(grads, before))


def test_a_large_tensor():
    gen = torch.Generator("cuda").manual_seed(2)
    g = torch.randn(9_000_001, generator=gen, device="cuda")
    ref = float(g.double().square().sum().sqrt())
    b = g.clone()
    assert abs(float(F.clip_grad_norm_([g], 1.0)) - ref) <= 2.0 ** -22 * ref  # (the reference's own sum is in another order)
    assert close(g, b.double() / (ref + 1e-6), torch.float32)


def test_squares_that_overflow_or_vanish_in_32_bits():
    for scale in (1e30, 1e-30):
        grads = [torch.full((5000,), scale, device="cuda"), torch.full((300,), scale, device="cuda").bfloat16()]
        ref = norm64(grads)
        assert abs(float(F.grad_norm(grads)) - ref) <= 2.0 ** -23 * ref
    big = [torch.full((100,), 3e38, device="cuda")]  # a norm beyond 32 bits is infinity, and clips by its own value
    ref = norm64(big)
    norm = F.clip_grad_norm_(big, 1.0)
    # The factor, 1 / 3e39, lies under the smallest normal number of its 32 bits: rounding it moves it by up to 2^-150 absolute, which is
    # 2^-150 * 3e39 = 2.1e-6 of itself, and not by 2^-24; the products are normal numbers.
    got = big[0].double()
    assert torch.isinf(norm) and ((got - 3e38 / ref).abs() <= (2.0 ** -150 * ref + 2.0 ** -23) * 3e38 / ref).all()


@pytest.mark.parametrize("kind", [2.0, math.inf])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_what_is_not_finite(bad, kind):
    for dtype in DT.values():
        grads = [torch.ones(9000, device="cuda", dtype=dtype), torch.ones(70, device="cuda", dtype=dtype)]
        grads[0][8200] = bad
        params = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]
        for p, g in zip(params, grads):
            p.grad = g.clone()
        with pytest.raises(RuntimeError, match="not finite"):
            clip_grad_norm_(params, 1.0, kind, error_if_nonfinite=True)
        assert all(torch.equal(p.grad, g) or math.isnan(bad) for p, g in zip(params, grads))
        norm = clip_grad_norm_(params, 1.0, kind)
        assert math.isnan(float(norm)) if math.isnan(bad) else math.isinf(float(norm))
        if math.isnan(bad):
            assert all(p.grad.isnan().all() for p in params)
        else:  # a factor of 0: 0 everywhere, NaN where infinity was
            assert not params[1].grad.any() and params[0].grad[8200].isnan() and not params[0].grad[:8200].any()


@pytest.mark.parametrize("offset", [1, 3, 8])
def test_tensors_that_begin_anywhere(offset):
    for dtype in DT.values():
        whole = torch.randn(20000, device="cuda").to(dtype)
        part, rest = whole[offset:offset + 10001], whole.clone()
        ref = norm64([part])
        assert abs(float(F.clip_grad_norm_([part], 0.5)) - ref) <= 2.0 ** -23 * ref
        assert close(part, rest[offset:offset + 10001].double() * 0.5 / (ref + 1e-6), dtype)
        assert torch.equal(whole[:offset], rest[:offset]) and torch.equal(whole[offset + 10001:], rest[offset + 10001:])


def test_layouts():
    turned = torch.randn(300, 70, device="cuda").t()  # fills its memory in another order
    last = torch.randn(4, 8, 5, 5, device="cuda").to(memory_format=torch.channels_last)
    grads = [turned, last]
    ref, before = norm64(grads), [g.clone() for g in grads]
    F.clip_grad_norm_(grads, 1.0)
    assert all(close(g, b.double() / (ref + 1e-6), torch.float32) for g, b in zip(grads, before))
    gaps, spread = torch.randn(64, 64, device="cuda")[:, :33], torch.randn(1, 64, device="cuda").expand(64, 64)
    for g in (gaps, spread):  # their norm is taken, in place they are refused
        ref = norm64([g])
        assert abs(float(F.grad_norm([g])) - ref) <= 2.0 ** -23 * ref
        with pytest.raises(ValueError, match="fill its memory"):
            F.clip_grad_norm_([g], 1.0)


def test_refusals():
    g = torch.ones(100, device="cuda")
    for bad, error, match in (([], ValueError, "at least one"), ([g.cpu()], ValueError, "one GPU"), ([g, g.cpu()], ValueError, "one GPU"),
                              ([g.double()], TypeError, "float16, bfloat16 or float32"), ([g.to_sparse()], ValueError, "sparse")):
        with pytest.raises(error, match=match):
            F.clip_grad_norm_(bad, 1.0)
        with pytest.raises(error, match=match):
            F.grad_norm(bad)
    for shared in ([g, g], [g, g[50:]], [g[:60], g[59:]]):
        with pytest.raises(ValueError, match="share memory"):
            F.clip_grad_norm_(shared, 1.0)
    F.clip_grad_norm_([g[:60], g[60:]], 1.0)
    for limit in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            F.clip_grad_norm_([g], limit)
        with pytest.raises(ValueError, match="max_norm"):
            F.grad_norm([g], 2, limit)
    with pytest.raises(ValueError, match="norm_type"):
        F.grad_norm([g], 3)
    with pytest.raises(NotImplementedError, match="traced"):
        torch.jit.trace(lambda t: F.grad_norm([t]), (g,))
    assert abs(float(F.grad_norm([g, g])) - float(F.grad_norm([g])) * 2 ** 0.5) < 1e-5


def test_equal_gradients_have_equal_norms_and_none_is_kept_for_another_call():
    a, b = gradients(("fp32", "bf16"), seed=3), gradients(("fp32", "bf16"), seed=4)
    na, nb = F.grad_norm(a).clone(), F.grad_norm(b).clone()
    for _ in range(3):
        assert torch.equal(F.grad_norm(a), na) and torch.equal(F.grad_norm(b), nb)


def test_captured_and_replayed_beside_another():
    sets = [gradients(("fp32", "bf16"), seed=5), gradients(("fp16",), seed=6)]
    for s in sets:
        F.clip_grad_norm_([g.clone() for g in s], 1.0)
    graphs, norms = [], []
    torch.cuda.synchronize()
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norms.append(F.clip_grad_norm_(s, 0.25))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in sets]
    for seed in (7, 8, 9):
        fresh = [gradients(("fp32", "bf16"), seed=seed), gradients(("fp16",), seed=seed + 10)]
        for s, f in zip(sets, fresh):
            for g, v in zip(s, f):
                g.copy_(v)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):  # both at once
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for s, f, n in zip(sets, fresh, norms):
            assert torch.equal(F.clip_grad_norm_(f, 0.25), n)
            assert all(torch.equal(g, v) for g, v in zip(s, f))


# ---- with AdamW ----------------------------------------------------------------------------------------------------------
def parameters(dtype, seed=0, sizes=((40, 30), (1000,), (257, 129), (1,))):
    gen = torch.Generator().manual_seed(seed)
    ps = [torch.nn.Parameter(torch.randn(s, generator=gen).to(dtype).cuda()) for s in sizes]
    for p in ps:
        p.grad = torch.randn(p.shape, generator=gen).to(dtype).cuda()
    return ps


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("limit", [0.5, 1e9])
def test_adamw_takes_gradients_times_the_factor(bits, limit):
    """float32 gradients scaled before the step are rounded where the step rounds them: equal parameters and averages."""
    here, there = parameters(torch.float32), parameters(torch.float32)
    a, b = AdamW(here, lr=1e-2, state_bits=bits, max_norm=limit), AdamW(there, lr=1e-2, state_bits=bits)
    for step in range(3):
        for p, q in zip(here, there):
            q.grad = p.grad.clone()
        kept = [p.grad.clone() for p in here]
        norm = clip_grad_norm_(there, limit)
        a.step()
        b.step()
        assert torch.equal(a.grad_norm, norm) and abs(float(norm) - norm64(kept)) <= 2.0 ** -23 * norm64(kept)
        for p, q, g in zip(here, there, kept):
            assert torch.equal(p, q) and torch.equal(p.grad, g)
            assert all(torch.equal(x, y) for x, y in zip(a.state_values(p), b.state_values(q)))
        for i, p in enumerate(here):
            p.grad = torch.randn_like(p) * 10.0 ** -step


@pytest.mark.parametrize("dtype", list(DT))
def test_adamw_step_with_a_factor_against_its_formula(dtype):
    dt = DT[dtype]
    p, g = ([t.detach().clone() for t in ts] for ts in (parameters(dt, 1), parameters(dt, 2)))
    m, v = [torch.zeros_like(t, dtype=torch.float32) for t in p], [torch.zeros_like(t, dtype=torch.float32) for t in p]
    factor, step = torch.tensor(0.125, device="cuda"), torch.zeros((), dtype=torch.int64, device="cuda")
    before = [t.clone() for t in p]
    F.adamw_step(p, g, m, v, step, lr=1e-2, weight_decay=0.0, grad_scale=factor)
    for t, b, x, a, s in zip(p, before, g, m, v):
        x = x.double() * 0.125
        assert ((a.double() - 0.1 * x).abs() <= 2.0 ** -22 * 0.1 * x.abs() + 1e-40).all()
        assert ((s.double() - 1e-3 * x * x).abs() <= 2.0 ** -21 * 1e-3 * x * x + 1e-40).all()
        # the first step moves by lr g / (|g| + eps): sixteen roundings of 2^-24 as in the step without a factor, three more for the factor's
        ref = b.double() - 1e-2 * x / (x.abs() + 1e-8)
        assert ((t.double() - ref).abs() <= 24 * 2.0 ** -24 * 1e-2 + (torch.finfo(dt).eps / 2 + 3 * 2.0 ** -24) * (b.double().abs() + 1e-2)).all()


def test_adamw_clips_the_joint_norm_of_its_groups_and_takes_a_changed_limit():
    ps = parameters(torch.float32, 3)
    opt = AdamW([{"params": ps[:2]}, {"params": ps[2:], "lr": 1e-3}], max_norm=1.0)
    ps[1].grad = None
    opt.step()
    ref = norm64([p.grad for p in ps if p.grad is not None])
    assert abs(float(opt.grad_norm) - ref) <= 2.0 ** -23 * ref
    before = [p.detach().clone() for p in ps]
    opt.max_norm = 0.0  # nothing of the gradients is left
    opt.param_groups[0]["weight_decay"] = opt.param_groups[1]["weight_decay"] = 0.0
    for p in ps:
        opt.state[p].clear() if p.grad is None else opt.state[p]["exp_avg"].zero_()
    opt.step()
    assert all(torch.equal(p, b) for p, b in zip(ps, before))
    again = copy.deepcopy(opt)
    assert again.max_norm == 0.0
    with pytest.raises(ValueError, match="max_norm"):
        AdamW(ps, max_norm=-1.0)
    for p in ps:
        p.grad = None
    opt.step()  # without any gradient there is nothing to do


def test_adamw_captured_with_clipping():
    ps, qs = parameters(torch.bfloat16, 4), parameters(torch.bfloat16, 4)
    a, b = AdamW(ps, lr=1e-2, max_norm=0.5), AdamW(qs, lr=1e-2, max_norm=0.5)
    a.step()
    b.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    found = a.grad_norm
    for seed in (11, 12, 13):
        for p, q, fresh in zip(ps, qs, parameters(torch.bfloat16, seed)):
            p.grad.copy_(fresh.grad)
            q.grad.copy_(fresh.grad)
        graph.replay()
        torch.cuda.synchronize()
        b.step()
        assert torch.equal(found, b.grad_norm)
        assert all(torch.equal(p, q) for p, q in zip(ps, qs))


def test_clipping_keeps_the_arguments_of_torchs():
    ps, qs = parameters(torch.float32, 5), parameters(torch.float32, 5)
    ps[0].grad = qs[0].grad = None
    ours, theirs = clip_grad_norm_(ps, 0.7), torch.nn.utils.clip_grad_norm_(qs, 0.7)
    assert abs(float(ours) - float(theirs)) <= 1e-5 * float(theirs)
    for p, q in zip(ps[1:], qs[1:]):
        torch.testing.assert_close(p.grad, q.grad, rtol=1e-5, atol=1e-8)
    one = parameters(torch.float32, 6)[1]
    assert float(clip_grad_norm_(one, 1.0, foreach=True)) > 1.0
    assert float(clip_grad_norm_([torch.nn.Parameter(torch.ones(3))], 1.0)) == 0.0


def test_a_training_step_of_the_gated_block_with_clipping():
    """Block, backward, norm, step, as they are used together: equal to the same with each part by itself."""
    from flash_dropout.layers import GatedMLP

    def models():
        torch.manual_seed(1)
        return GatedMLP(128, 256, p=0.3, variant="blockwise[hip]", block_size=64).cuda().bfloat16().train()

    one, two = models(), models()
    a, b = AdamW(one.parameters(), lr=1e-3, max_norm=0.01), AdamW(two.parameters(), lr=1e-3)
    two.load_state_dict(one.state_dict())
    gen = torch.Generator("cuda").manual_seed(2)
    for step in range(3):
        x = torch.randn(200, 128, generator=gen, device="cuda").bfloat16()
        grads = []
        for model in (one, two):
            model.zero_grad(set_to_none=True)
            y = F.hip_blockwise_dropout_gated_mlp(x, model.weight_in, model.weight_out, 64, 0.3, seed=100 + step)
            y.float().square().mean().backward()
            grads.append([p.grad for p in model.parameters()])
        assert all(torch.equal(g, h) for g, h in zip(*grads))
        a.step()
        norm, factor = F.grad_norm(grads[1], max_norm=0.01)
        F_state = [b.state[p] for p in two.parameters()]
        if step == 0:
            for p in two.parameters():
                b._init_state(p, 32, torch.zeros((), dtype=torch.int64, device="cuda"))
            F_state = [b.state[p] for p in two.parameters()]
        with torch.no_grad():
            F.adamw_step(list(two.parameters()), grads[1], [s["exp_avg"] for s in F_state], [s["exp_avg_sq"] for s in F_state], F_state[0]["step"], lr=1e-3,
                         grad_scale=factor)
        assert torch.equal(norm, a.grad_norm) and float(factor) < 1.0
        assert all(torch.equal(p, q) for p, q in zip(one.parameters(), two.parameters()))


def test_a_factor_or_a_rate_inside_what_a_step_writes_is_refused():
    p, g = torch.randn(1000, device="cuda"), torch.randn(1000, device="cuda")
    m, v, step = torch.zeros_like(p), torch.zeros_like(p), torch.zeros((), dtype=torch.int64, device="cuda")
    before = p.clone()
    for t in (p, m, v):
        for kw in ({"grad_scale": t[990]}, {"lr": t[3:4]}):
            with pytest.raises(ValueError, match="parameter 0.*factor of the gradients"):
                F.adamw_step([p], [g], [m], [v], step, **kw)
    for t in (p, m, v, g):
        with pytest.raises(ValueError, match="parameter 0.*the step"):
            F.adamw_step([p], [g], [m], [v], t[4:6].view(torch.int64)[0])
    assert torch.equal(p, before) and not m.any() and not v.any() and int(step) == 0
    factors = torch.tensor([0.0, 0.5], device="cuda")  # beside what is written, and in a gradient, which is read alone
    F.adamw_step([p], [g], [m], [v], step, lr=factors[0], grad_scale=factors[1], weight_decay=0.0)
    F.adamw_step([p], [g], [m], [v], step, lr=factors[0], grad_scale=g[5], weight_decay=0.0)
    assert torch.equal(p, before) and int(step) == 2 and bool(m.any())
