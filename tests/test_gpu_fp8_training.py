"""Layers in 8 bits, their optimizer and serving used together, and the calls that lie at the edges of what is allowed.

Tolerances are those of the single operators (tests/test_gpu_fp8.py, tests/test_gpu_adamw.py): every step below is checked from the tensors that
went into it."""
import gc

import numpy as np
import pytest
import torch

from oracle import fp8_oracle as O
from test_gpu_adamw import check_param
from test_gpu_fp8 import check_product, check_train, np64, spread, train

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import flash_dropout.functional as F
    from flash_dropout.hip import GEMM
    from flash_dropout.layers import DropoutMM
    from flash_dropout.optim import AdamW

HYPER = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_training_steps_and_then_serving(dtype, bits):
    """Two layers, three steps of AdamW, then the products with the trained weights kept in 8 bits."""
    gen = torch.Generator().manual_seed(1)
    tokens, dims, bs, p = 300, (260, 384, 140), 128, 0.5
    ws = [torch.nn.Parameter((torch.randn(dims[i + 1], dims[i], generator=gen) * dims[i] ** -0.5).to(dtype).cuda()) for i in range(2)]
    opt = AdamW(ws, **HYPER, state_bits=bits)
    for step in range(1, 4):
        x = torch.randn(tokens, dims[0], generator=gen).to(dtype).cuda().requires_grad_()
        dy = torch.randn(tokens, dims[2], generator=gen).to(dtype).cuda()
        masks = [torch.rand(-(-tokens // bs), -(-dims[i] // bs), generator=gen) < p for i in range(2)]
        h = F.hip_blockwise_dropout_matmul_fp8_mask(x, masks[0].cuda(), bs, p, ws[0])
        h.retain_grad()
        a = torch.relu(h)
        a.retain_grad()
        y = F.hip_blockwise_dropout_matmul_fp8_mask(a, masks[1].cuda(), bs, p, ws[1])
        opt.zero_grad(set_to_none=True)
        y.backward(dy)
        check_train(x, ws[0], h.grad, masks[0], bs, p, h, x.grad, ws[0].grad)
        check_train(a, ws[1], dy, masks[1], bs, p, y, a.grad, ws[1].grad)
        before = [(w.detach().clone(), *((np64(t) for t in opt.state_values(w)) if opt.state[w] else (0.0, 0.0))) for w in ws]
        opt.step()
        for w, (old, m, v) in zip(ws, before):
            m, v = (np.broadcast_to(t, tuple(w.shape)) for t in (m, v))
            check_param(w, old, w.grad, m, v, step, dtype, HYPER)
            _, m, v = O.adamw(np64(old), np64(w.grad), m, v, step, HYPER["lr"], *HYPER["betas"], HYPER["eps"], HYPER["weight_decay"])
            got = [np64(t) for t in opt.state_values(w)]
            if bits == 8:
                assert np.array_equal(got[0], O.rounded_state(m, "first", step)) and np.array_equal(got[1], O.rounded_state(v, "second", step))
            assert opt.state[w]["step"].item() == step
    kept = [F.fp8_quantize(w.detach(), (128, 128)) for w in ws]
    for rows in (1, 16, 50, 300):
        x = torch.randn(rows, dims[0], generator=gen).to(dtype).cuda()
        with torch.no_grad():
            h = F.fp8_linear(x, *kept[0])
            y = F.fp8_linear(torch.relu(h), *kept[1])
        check_product(h, *O.product(np64(x), 1, np64(ws[0]), 128), dims[0], dtype)
        check_product(y, *O.product(np64(torch.relu(h)), 1, np64(ws[1]), 128), dims[1], dtype)


@pytest.mark.parametrize("bits", [8, 32])
def test_a_captured_training_step_equals_an_eager_one(bits):
    """Layers with drawn masks, both gradients and the optimizer in one graph: parameters and averages after every replay are those of the
    same steps taken one by one."""
    def net():
        torch.manual_seed(3)
        return torch.nn.Sequential(DropoutMM(256, 384, p=0.5, variant="blockwise[hip-fp8]", block_size=128), torch.nn.ReLU(),
                                   DropoutMM(384, 256, p=0.5, variant="blockwise[hip-fp8]", block_size=128)).cuda().bfloat16()

    x, dy = torch.empty(300, 256, device="cuda").bfloat16(), torch.empty(300, 256, device="cuda").bfloat16()

    def batch(i):
        x.copy_(spread(300, 256, torch.bfloat16, 10 + i).div_(64))
        dy.copy_(spread(300, 256, torch.bfloat16, 20 + i).div_(64))

    def step(model, opt):
        opt.zero_grad(set_to_none=True)
        model(x).backward(dy)
        opt.step()

    nets = [net(), net()]
    opts = [AdamW(n.parameters(), **HYPER, state_bits=bits) for n in nets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    batch(0)
    with torch.cuda.stream(side):
        for n, o in zip(nets, opts):
            GEMM().manual_seed(9)
            step(n, o)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    nets[0].zero_grad(set_to_none=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(nets[0], opts[0])
    for i in range(1, 4):
        batch(i)
        GEMM().manual_seed(100 + i)
        graph.replay()
        torch.cuda.synchronize()
        GEMM().manual_seed(100 + i)
        step(nets[1], opts[1])
        for a, b in zip(nets[0].parameters(), nets[1].parameters()):
            assert torch.equal(a, b)
            sa, sb = opts[0].state[a], opts[1].state[b]
            assert all(torch.equal(sa[key], sb[key]) for key in sb) and sa["step"].item() == i + 1


def test_an_optimizers_first_step_is_not_captured():
    ps = [torch.nn.Parameter(torch.ones(300, device="cuda")) for _ in range(2)]
    opt = AdamW(ps, lr=1e-2)
    for q in ps:
        q.grad = torch.ones_like(q)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="first step"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    opt = AdamW(ps, lr=1e-2)
    opt.step()
    ps[0].grad = None
    with pytest.raises(RuntimeError, match="without some"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    torch.cuda.synchronize()
    opt.step()
    assert [opt.state[q]["step"].item() for q in ps] == [1, 2]


@pytest.mark.parametrize("bs", [128, 256])
def test_masks_of_many_blocks_are_drawn_like_those_of_few(bs):
    m, k, n = 2200, 2300, 40
    x, w, dy, _ = train(m, k, n, torch.float16, bs, 0.5)
    grid = (-(-m // bs), -(-k // bs))
    for seed in (77, None):
        GEMM().manual_seed(41)
        mask, _ = GEMM().random_lists(grid, 0.5, *(() if seed is None else (seed,)))
        GEMM().manual_seed(41)
        y = F.hip_blockwise_dropout_matmul_fp8(x, w, bs, 0.5, seed=seed)
        assert GEMM().rng_state()[1].item() == (seed is None)
        check_train(x, w, dy, mask, bs, 0.5, y, *torch.autograd.grad(y, (x, w), dy))


def test_everything_kept_for_the_backward_goes_through_saved_tensor_hooks():
    x, w, dy, mask = train(300, 512, 256, torch.float16, 128, 0.5)
    mask = mask.cuda()
    call = lambda: F.hip_blockwise_dropout_matmul_fp8_mask(x, mask, 128, 0.5, w)  # noqa: E731
    want = torch.autograd.grad(call(), (x, w), dy)
    gc.collect()
    before = torch.cuda.memory_allocated()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda()):
        y = call()
    gc.collect()
    assert torch.cuda.memory_allocated() - before <= -(-y.numel() * 2 // 512) * 512
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, (x, w), dy), want))
    for unpack in (lambda t: t.cpu(), lambda t: t.double(), lambda t: t[:-1]):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            y = call()
        with pytest.raises(ValueError, match="saved-tensor hook"):
            torch.autograd.grad(y, (x, w), dy)

    def strided(t):
        wide = torch.zeros(*t.shape, 2, dtype=t.dtype, device=t.device)
        wide[..., 0] = t
        return wide[..., 0]

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, strided):
        y = call()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, (x, w), dy), want))


def test_what_changes_between_forward_and_backward():
    """Input and weight are kept in 8 bits, so later writes to them change no gradient; one to the mask is an error."""
    x, w, dy, mask = train(300, 512, 256, torch.float16, 128, 0.5)
    mask = mask.cuda()
    want = torch.autograd.grad(F.hip_blockwise_dropout_matmul_fp8_mask(x, mask, 128, 0.5, w), (x, w), dy)
    y = F.hip_blockwise_dropout_matmul_fp8_mask(x, mask, 128, 0.5, w)
    with torch.no_grad():
        x.zero_()
        w.zero_()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, (x, w), dy), want))
    y = F.hip_blockwise_dropout_matmul_fp8_mask(x, mask, 128, 0.5, w)
    mask.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, (x, w), dy)


def test_forward_gradients_and_transforms_are_refused_and_traces_run():
    import torch.autograd.forward_ad as fwd

    x, w, dy, _ = train(130, 256, 140, torch.float16, 128, 0.5)
    kept = F.fp8_quantize(w.detach(), (128, 128))
    layer = lambda a, b: F.hip_blockwise_dropout_matmul_fp8(a, b, 128, 0.5, seed=5)  # noqa: E731
    served = lambda a: F.fp8_linear(a, *kept)  # noqa: E731
    with fwd.dual_level():
        for i in range(2):
            dual = [x.detach(), w.detach()]
            dual[i] = fwd.make_dual(dual[i], torch.ones_like(dual[i]))
            with pytest.raises(NotImplementedError, match="jvp"):
                layer(*dual)
        with pytest.raises(NotImplementedError, match="jvp"):
            served(fwd.make_dual(x.detach(), torch.ones_like(x)))
    for transformed in (lambda: torch.func.vmap(served)(torch.stack([x.detach()] * 2)),
                        lambda: torch.func.vmap(lambda a: layer(a, w.detach()))(torch.stack([x.detach()] * 2)),
                        lambda: torch.func.grad(lambda a: layer(a, w.detach()).float().sum())(x.detach())):
        with pytest.raises((RuntimeError, NotImplementedError, ValueError)):
            transformed()
    traced = torch.jit.trace(lambda a, b: layer(a, b) * 2, (x, w), check_trace=False)
    other = [(t.detach() * 0.5).requires_grad_() for t in (x, w)]
    got, want = traced(*other), layer(*other) * 2
    assert torch.equal(got, want)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(got, other, dy), torch.autograd.grad(want, other, dy)))
    with torch.no_grad():
        traced = torch.jit.trace(served, (x,), check_trace=False)
        assert torch.equal(traced(other[0]), served(other[0]))
        with torch.autocast("cuda", torch.bfloat16):
            cast = torch.jit.trace(served, (x.detach().float(),), check_trace=False)
            assert torch.equal(cast(other[0].float()), served(other[0].bfloat16()))
    with pytest.raises(NotImplementedError):
        traced(other[0]).float().sum().backward()


def test_the_quantizer_refuses_forward_gradients_and_transforms():
    import torch.autograd.forward_ad as fwd

    x = spread(70, 300, torch.float32)
    for block in ((1, 128), (128, 128)):
        with fwd.dual_level():
            with pytest.raises(NotImplementedError, match="jvp"):
                F.fp8_quantize(fwd.make_dual(x, torch.ones_like(x)), block)
        with pytest.raises(NotImplementedError, match="jvp"):
            torch.func.jvp(lambda a: F.fp8_dequantize(*F.fp8_quantize(a, block)), (x,), (x,))
        with pytest.raises((RuntimeError, NotImplementedError, ValueError)):
            torch.func.vmap(lambda a: F.fp8_dequantize(*F.fp8_quantize(a, block)))(torch.stack([x, x]))
    data, scales = F.fp8_quantize(x.requires_grad_())
    assert not data.requires_grad and not scales.requires_grad


def test_traces_quantize_what_they_are_given():
    """Codes, scales and values of the traced program's own inputs, whichever of its parts were traced; autocast changes none."""
    x, other = spread(70, 300, torch.float32).div_(64), spread(70, 300, torch.float32, 5).div_(64)
    w = torch.nn.Parameter(spread(140, 300, torch.float16, 2).div_(64))

    def values(a):
        data, scales = F.fp8_quantize(a)
        return data.float(), scales.float(), F.fp8_dequantize(data, scales, a.shape[1], torch.bfloat16)

    def served(a, b):  # (a weight that wants a gradient does not pass it on to its codes)
        return F.fp8_linear(a, *F.fp8_quantize(b, (128, 128)))

    traced = torch.jit.trace(values, (x,), check_trace=False)
    for a in (other, other[:31]):
        assert all(torch.equal(s, t) for s, t in zip(traced(a), values(a)))
    with torch.autocast("cuda", torch.bfloat16):
        cast = torch.jit.trace(values, (x,), check_trace=False)
        assert all(torch.equal(s, t) for s, t in zip(cast(other), values(other)))
    assert all(torch.equal(s, t) for s, t in zip(cast(other), values(other)))
    traced = torch.jit.trace(served, (x.half(), w), check_trace=False)
    for _ in range(2):
        assert torch.equal(traced(other.half(), w), served(other.half(), w))
        with torch.no_grad():
            w.mul_(3)
    p = torch.nn.Parameter(torch.zeros(3, device="cuda"))
    p.grad = torch.ones_like(p)
    opt = AdamW([p], state_bits=8)
    opt.step()
    with pytest.raises(NotImplementedError, match="cannot be traced"):
        torch.jit.trace(lambda a: opt.step() or a, (x,), check_trace=False)
    assert opt.state[p]["step"].item() == 1


def test_under_autocast_kept_weights_take_inputs_in_32_bits():
    x = spread(40, 256, torch.float32).div_(64)
    kept = F.fp8_quantize(spread(140, 256, torch.float16, 2), (128, 128))
    with torch.no_grad(), torch.autocast("cuda", torch.bfloat16):
        y = F.fp8_linear(x, *kept)
    assert torch.equal(y, F.fp8_linear(x.bfloat16(), *kept)) and y.dtype == torch.bfloat16


@pytest.mark.parametrize("m,k,n", [(130, 4097 * 128 + 40, 16), (4097 * 128 + 40, 130, 16), (130, 260, 4097 * 128 + 40)])
def test_reductions_of_more_blocks_than_a_list_holds(m, k, n):
    """Whole numbers up to 4: sums of half a million products stay below 2^24 and exact in 32 bits."""
    gen = torch.Generator(device="cuda").manual_seed(m)
    make = lambda *size: torch.randint(-4, 5, size, generator=gen, device="cuda").bfloat16()  # noqa: E731
    x, w, dy = make(m, k).requires_grad_(), make(n, k).requires_grad_(), make(m, n)
    mask = torch.rand(-(-m // 128), -(-k // 128), generator=gen, device="cuda") < 0.5
    y = F.hip_blockwise_dropout_matmul_fp8_mask(x, mask, 128, 0.5, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    keep = ~mask.repeat_interleave(128, 0)[:m].repeat_interleave(128, 1)[:, :k]
    xk, wd, dyd = (x.detach() * keep).double(), w.detach().double(), dy.double()
    assert torch.equal(y, (2 * xk @ wd.t()).bfloat16())
    assert torch.equal(dx, (2 * (dyd @ wd) * keep).bfloat16())
    assert torch.equal(dw, (2 * dyd.t() @ xk).bfloat16())


def test_very_wide_matrices_there_and_back():
    cols = (1 << 22) + 200
    x = spread(2, 1, torch.float32).expand(2, cols) * torch.arange(1, cols + 1, device="cuda").float().remainder(97)
    for block in ((1, 128), (128, 128)):
        data, scales = F.fp8_quantize(x, block)
        values = F.fp8_dequantize(data, scales, cols)
        most = x.new_zeros(2, -(-cols // 128) * 128)
        most[:, :cols] = x.abs()
        most = most.view(2, -1, 128).amax(2)
        if block[0] == 128:
            most = most.amax(0, keepdim=True).expand(2, -1)
        # half of 2^-3 of the value, or half of 2^-9 of its block's scale, which is less than 2^-7 of the block's largest
        assert ((values - x).abs() <= x.abs() * 2.0 ** -4 + most.repeat_interleave(128, 1)[:, :cols] * 2.0 ** -17).all()
    with pytest.raises(NotImplementedError):
        F.fp8_linear(torch.zeros(1, cols, device="cuda").half(), *F.fp8_quantize(x.half(), (128, 128)))


def test_codes_that_start_anywhere():
    x, w = spread(70, 256, torch.float16).div_(64), spread(140, 256, torch.float16, 1).div_(64)
    data, scales = F.fp8_quantize(w, (128, 128))
    want, values = F.fp8_linear(x, data, scales), F.fp8_dequantize(data, scales)
    buf = torch.empty(data.numel() + 16, dtype=torch.uint8, device="cuda")
    for offset in (1, 8):
        there = buf[offset : offset + data.numel()].view(torch.float8_e4m3fn).view(data.shape)
        there.view(torch.uint8).copy_(data.view(torch.uint8))
        for rows in (4, 70):
            assert torch.equal(F.fp8_linear(x[:rows], there, scales), F.fp8_linear(x[:rows], data, scales))
        assert torch.equal(F.fp8_dequantize(there, scales), values)
    assert torch.equal(F.fp8_linear(x, data, scales), want)


def test_calls_on_two_streams_at_once():
    """Each call has buffers of its own: results are those of calls one after the other."""
    sets = [train(500, 1024, 700, torch.float16, 128, 0.5, seed=s) for s in (1, 2)]
    masks = [s[3].cuda() for s in sets]
    params = [[torch.nn.Parameter(s[1].detach().clone()) for s in sets] for _ in range(2)]

    def run(i, w):
        x, _, dy, _ = sets[i]
        opt = AdamW([w], **HYPER, state_bits=8)
        for _ in range(4):
            y = F.hip_blockwise_dropout_matmul_fp8_mask(x, masks[i], 128, 0.5, w)
            dx, w.grad = torch.autograd.grad(y, (x, w), dy)
            opt.step()
        return y, dx, w.grad, F.fp8_linear(x.detach(), *F.fp8_quantize(w.detach(), (128, 128)))

    want = [run(i, params[0][i]) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            got.append(run(i, params[1][i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(got[i], want[i])) and torch.equal(params[0][i], params[1][i])


@pytest.mark.parametrize("bits", [8, 32])
def test_gradients_whose_squares_are_next_to_nothing(bits):
    """Without eps a first step moves a parameter by lr, whatever the gradient's size: of 2.7e-19 the second average is 2^-130, which fp32
    holds to 2^-20, and its root to 8 of the 2^-24 that the update is held to 24 of (the first average's and the update's own take 12)."""
    n = 300
    g = torch.where(torch.arange(n) % 3 == 0, -2.7e-19, 2.7e-19).cuda()
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    p.grad = g.clone()
    AdamW([p], lr=0.5, betas=(0.9, 0.99), eps=0.0, weight_decay=0.0, state_bits=bits).step()
    assert ((p.detach() + 0.5 * g.sign()).abs() <= 24 * 2.0 ** -24 * 0.5).all()


@pytest.mark.parametrize("optimizer", ["adamw", "adamw-8bit"])
@pytest.mark.parametrize("name", ["mlp-784", "vit-ffn"])
def test_the_model_harness_runs_layers_in_8_bits_and_the_optimizer(name, optimizer):
    from benchmark import model as bm

    cls, make_x = bm.MODELS[name]
    torch.manual_seed(0)
    x = make_x().cuda().half()
    for graph in (False, True):
        net = cls("blockwise[hip-fp8]", 0.5, 128).cuda().half().train()
        opt = AdamW(net.parameters(), lr=1e-4, state_bits=bm.OPTIMIZERS[optimizer])
        before = [q.detach().clone() for q in net.parameters()]
        assert len(bm.time_model(net, x, warmup=0.0, rep=0.0, graph=graph, optimizer=opt)) >= 5
        assert all(not torch.equal(a, b) for a, b in zip(before, net.parameters()))
        assert {opt.state[q]["step"].item() for q in net.parameters()} != {0}


def test_captured_serving_replays():
    """Quantizing, both routes of the product with kept weights, and the product of two quantized matrices in one graph, on new inputs."""
    w = spread(1030, 2000, torch.bfloat16, 1).div_(64)
    few, many = torch.empty(5, 2000, device="cuda").bfloat16(), torch.empty(300, 2000, device="cuda").bfloat16()
    kept = F.fp8_quantize(w, (128, 128))

    def run():
        q = F.fp8_quantize(many)
        return (*(t.view(torch.uint8) for t in q), F.fp8_dequantize(*q, 2000), F.fp8_linear(few, *kept), F.fp8_linear(many, *kept), GEMM().gemm_fp8(*q, *kept))

    def batch(i):
        few.copy_(spread(5, 2000, torch.bfloat16, 10 + i).div_(64))
        many.copy_(spread(300, 2000, torch.bfloat16, 20 + i).div_(64))

    batch(0)
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for i in range(1, 4):
        batch(i)
        graph.replay()
        torch.cuda.synchronize()
        want = run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_scales_that_are_no_number():
    """A scale's byte 255 stands for NaN: all of its block is."""
    x, w = spread(140, 256, torch.float16).div_(64), spread(300, 256, torch.float16, 1).div_(64)
    data, scales = F.fp8_quantize(w, (128, 128))
    want = [F.fp8_linear(x[:rows], data, scales) for rows in (4, 140)]
    values = F.fp8_dequantize(data, scales)
    scales.view(torch.uint8)[1, 1] = 255
    again = F.fp8_dequantize(data, scales)
    assert again[128:256, 128:].isnan().all()
    again[128:256, 128:] = values[128:256, 128:]
    assert torch.equal(again, values)
    for rows, y in zip((4, 140), want):
        got = F.fp8_linear(x[:rows], data, scales)
        assert got[:, 128:256].isnan().all() and torch.equal(got[:, :128], y[:, :128]) and torch.equal(got[:, 256:], y[:, 256:])


@pytest.mark.parametrize("rows", [1, 5, 16, 17, 32, 33, 64])
@pytest.mark.parametrize("n,k", [(4110, 2200), (4097, 130), (8200, 2048), (500, 2200), (4112, 4100)])
def test_few_rows_of_wide_and_narrow_layers(n, k, rows):
    """Whole numbers up to 8, exact in 8 bits and in fp32 sums: 16 and 32 outputs a workgroup, four and sixteen waves, each with a ragged end."""
    gen = torch.Generator(device="cuda").manual_seed(n + k)
    make = lambda *size: torch.randint(-8, 9, size, generator=gen, device="cuda").bfloat16()  # noqa: E731
    w, buf = make(n, k), make(rows, k + 3)
    kept = F.fp8_quantize(w, (128, 128))
    for x in (buf[:, :k].contiguous(), buf[:, 3:]):
        assert torch.equal(F.fp8_linear(x, *kept), (x.double() @ w.double().t()).bfloat16())
