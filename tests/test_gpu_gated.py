"""The gated feed-forward block on the GPU against its formulas in 64 bits: element by element within the bounds that oracle/gated_oracle.py
derives from the roundings, and within the package's bar of 1e-2 in the relative Frobenius norm."""
import math
import os
import subprocess
import sys

import pytest
import torch

from _util import REL_FRO_TOL, rel_fro
from oracle import gated_oracle as O

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import flash_dropout.functional as F
    from flash_dropout.hip import _loader
    from flash_dropout.layers import GatedMLP

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
NAMES = ("y", "dx", "dw_in", "dw_out")


def operands(m, k, f, n, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    make = lambda r, c, std: (torch.randn(r, c, generator=gen) * std).to(DT[dtype]).cuda()
    return make(m, k, 1.0), make(2 * f, k, k ** -0.5), make(n, f, f ** -0.5), make(m, n, 0.1)


def masks_of(m, k, f, bs, p, seed=5):
    gen = torch.Generator().manual_seed(seed)
    return [(torch.rand(-(-m // bs), -(-c // bs), generator=gen) < p).cuda() for c in (k, f)]


def run(x, w_in, w_out, dy, act, bs=None, p=0.0, masks=None):
    leaves = [t.detach().requires_grad_() for t in (x, w_in, w_out)]
    y = F.gated_mlp(*leaves, act) if bs is None else F.hip_blockwise_dropout_gated_mlp(*leaves, bs, p, act, masks=masks)
    return dict(zip(NAMES, (y, *torch.autograd.grad(y, leaves, dy))))


def check(got, ref):
    for name in got:
        value, bound = ref[name]
        g = got[name].detach().double()
        assert g.shape == value.shape, name
        over = ((g - value).abs() > bound) | ~torch.isfinite(g)
        assert not over.any(), (name, int(over.sum()), over.nonzero()[0].tolist(), float((g - value).abs().max()))
        if value.numel() > 200 and float(value.abs().max()) > 1e-3:
            assert rel_fro(g, value) < REL_FRO_TOL, name


SIZES = [(1, 64, 64, 64), (1, 1024, 4096, 1024), (2, 8, 8, 8), (3, 1, 1, 1), (1, 130, 1, 5), (5, 77, 33, 19), (16, 512, 1024, 512), (17, 512, 1000, 200),
         (33, 264, 136, 72), (64, 256, 512, 256), (65, 256, 512, 256), (128, 128, 64, 128), (130, 200, 96, 72), (257, 320, 704, 320), (301, 1025, 777, 640),
         (512, 1024, 2048, 1024), (1100, 392, 1304, 264)]


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_block(size, act):
    for dtype in ("fp16", "bf16"):
        ops = operands(*size, dtype)
        check(run(*ops, act), O.reference(*ops, act, DT[dtype]))
        with torch.no_grad():
            y = F.gated_mlp(*ops[:3], act)
        check({"y": y}, O.reference(*ops, act, DT[dtype]))


@pytest.mark.parametrize("bs,p", [(64, 0.5), (64, 0.1), (128, 0.3), (32, 0.5), (96, 0.25), (64, 0.9)])
@pytest.mark.parametrize("size", [(64, 64, 64, 64), (130, 200, 96, 72), (301, 1025, 777, 640), (1024, 512, 1024, 512), (70, 640, 1300, 130)],
                         ids=lambda s: "x".join(map(str, s)))
def test_dropped_blocks(size, bs, p):
    for dtype, act in (("fp16", "gelu"), ("bf16", "silu"), ("bf16", "relu")):
        ops = operands(*size, dtype, seed=1)
        masks = masks_of(*size[:3], bs, p)
        got = run(*ops, act, bs, p, masks)
        check(got, O.reference(*ops, act, DT[dtype], masks, bs, (p, p)))


def test_large_products():
    ops = operands(2048, 1024, 4096, 1024, "bf16", seed=2)
    check(run(*ops, "silu"), O.reference(*ops, "silu", torch.bfloat16))
    masks = masks_of(2048, 1024, 4096, 64, 0.5)
    check(run(*ops, "gelu", 64, 0.5, masks), O.reference(*ops, "gelu", torch.bfloat16, masks, 64, (0.5, 0.5)))


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("size", [(128, 256, 320, 64), (300, 136, 200, 88), (1024, 1024, 1024, 256)])
def test_rows_and_operands_with_nothing_kept(size, which):
    m, k, f, n = size
    ops = operands(*size, "bf16", seed=3)
    none = [torch.zeros(-(-m // 64), -(-c // 64), dtype=torch.bool, device="cuda") for c in (k, f)]
    for rows in (slice(0, 1), slice(None)):
        masks = [t.clone() for t in none]
        masks[which][rows] = True
        got = run(*ops, "silu", 64, (0.5, 0.0), masks)
        check(got, O.reference(*ops, "silu", torch.bfloat16, masks, 64, (0.5, 0.0)))
        assert not got["y"][:64].any() and not got["dx"][:64].any()
        if rows == slice(None):
            assert not got["dw_in"].any() and not got["dw_out"].any()


def test_what_stands_in_dropped_blocks_reaches_nothing():
    size = (192, 256, 320, 128)
    ops = operands(*size, "fp16", seed=4)
    masks = masks_of(192, 256, 320, 64, 0.4)
    ref = run(*ops, "gelu", 64, 0.4, masks)
    x = ops[0].clone()
    drop = masks[0].repeat_interleave(64, 0).repeat_interleave(64, 1)
    x[drop] = float("nan")
    got = run(x, *ops[1:], "gelu", 64, 0.4, masks)
    for name in NAMES:
        assert torch.equal(got[name], ref[name]), name
    # hidden activations that overflow in a dropped block
    w_in = ops[1].clone()
    w_in[64:128] *= 30000  # the gate's columns 64 .. 127
    masks[1][:, 1] = True
    got, ref = (run(ops[0], w, *ops[2:], "gelu", 64, 0.4, masks) for w in (w_in, ops[1]))
    for name in ("y", "dw_out"):
        assert torch.equal(got[name], ref[name]), name
    assert not got["dw_in"][64:128].any() and torch.equal(got["dx"], ref["dx"])


def test_layouts_of_operands():
    ops = operands(72, 136, 200, 56, "bf16", seed=6)
    ref = O.reference(*ops, "silu", torch.bfloat16)
    turned = [t.t().contiguous().t() for t in ops]
    check(run(*turned, "silu"), ref)
    wide = [torch.cat((t, t), 1)[:, : t.shape[1]] for t in ops]
    check(run(*wide, "silu"), ref)
    off = [torch.cat((t[:, :3], t), 1)[:, 3:] for t in ops]
    check(run(*off, "silu"), ref)
    got = run(ops[0][:1].expand(72, 136), *ops[1:], "silu")
    check(got, O.reference(ops[0][:1].expand(72, 136), *ops[1:], "silu", torch.bfloat16))
    for few in (1, 7):  # the few rows of serving, strided
        part = [ops[0][:few], *ops[1:3], ops[3][:few]]
        with torch.no_grad():
            for xs in (part[0], wide[0][:few], off[0][:few], turned[0][:few]):
                for ws in (ops, wide, off, turned):
                    check({"y": F.gated_mlp(xs, ws[1], ws[2])}, O.reference(*part, "silu", torch.bfloat16))


@pytest.mark.parametrize("p", [0.0, 0.4])
@pytest.mark.parametrize("size", [(96, 128, 192, 64), (97, 130, 99, 33), (1030, 512, 768, 520)], ids=lambda s: "x".join(map(str, s)))
def test_only_the_wanted_gradients(size, p):
    ops = operands(*size, "fp16", seed=7)
    masks = masks_of(*size[:3], 64, p) if p else None
    full = run(*ops, "silu", 64, p, masks)
    for wanted in range(1, 8):
        leaves = [t.detach().requires_grad_(bool(wanted >> i & 1)) for i, t in enumerate(ops[:3])]
        y = F.hip_blockwise_dropout_gated_mlp(*leaves, 64, p, masks=masks)
        y.backward(ops[3])
        for t, name in zip(leaves, NAMES[1:]):
            if not t.requires_grad:
                assert t.grad is None
            else:  # (a gradient by itself may be summed in another order than beside another)
                assert rel_fro(t.grad.double(), full[name].double()) < 2.0 ** -10, name


def test_no_rows():
    _, w_in, w_out, _ = operands(1, 64, 96, 32, "bf16")
    leaves = [torch.empty(0, 64, dtype=torch.bfloat16, device="cuda").requires_grad_(), w_in.requires_grad_(), w_out.requires_grad_()]
    y = F.gated_mlp(*leaves)
    assert y.shape == (0, 32)
    y.sum().backward()
    assert leaves[0].grad.shape == (0, 64) and not leaves[1].grad.any() and not leaves[2].grad.any()


def test_draws():
    ops = operands(256, 256, 512, 128, "bf16", seed=8)
    draw = lambda **kw: F.hip_blockwise_dropout_gated_mlp(*ops[:3], 64, 0.5, "silu", **kw)
    assert torch.equal(draw(seed=3), draw(seed=3)) and not torch.equal(draw(seed=3), draw(seed=4))
    assert not torch.equal(draw(), draw())
    # the input's mask is drawn from the seed, the hidden activations' from the next: blocks of either with one row of inputs tell which they are
    both = masks_of(256, 256, 512, 64, 0.5)
    a, b = (draw(masks=[both[0], None], seed=s) for s in (11, 11))
    assert torch.equal(a, b) and not torch.equal(a, draw(masks=[both[0], None], seed=12))
    # nothing dropped where p is 0
    y = F.hip_blockwise_dropout_gated_mlp(*ops[:3], 64, 0.0)
    assert torch.equal(y, F.gated_mlp(*ops[:3]))
    half = F.hip_blockwise_dropout_gated_mlp(*ops[:3], 64, (0.0, 0.5), masks=[None, both[1]])
    check({"y": half}, O.reference(*ops, "silu", torch.bfloat16, (None, both[1]), 64, (0.0, 0.5)))


@pytest.mark.parametrize("p", [0.0, 0.4])
@pytest.mark.parametrize("size", [(1, 256, 512, 256), (24, 200, 333, 120), (512, 256, 768, 256)], ids=lambda s: "x".join(map(str, s)))
def test_captured_and_replayed(size, p):
    ops = operands(*size, "bf16", seed=9)
    masks = masks_of(*size[:3], 64, p) if p else None
    static = [t.clone() for t in ops]
    leaves = [t.requires_grad_() for t in static[:3]]

    def step():
        y = F.hip_blockwise_dropout_gated_mlp(*leaves, 64, p, "silu", masks=masks)
        return (y, *torch.autograd.grad(y, leaves, static[3]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (20, 21, 22):
        fresh = operands(*size, "bf16", seed=seed)
        with torch.no_grad():
            for t, v in zip(static, fresh):
                t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        eager = run(*fresh, "silu", 64, p, masks)
        for name, t in zip(NAMES, out):
            assert torch.equal(t, eager[name]), name


def test_other_streams_and_calls_beside_each_other():
    cases = [operands(16, 512, 1024, 512, "bf16", seed=30), operands(300, 256, 512, 128, "bf16", seed=31)]
    refs = [run(*c, "silu") for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[] for _ in cases]
    for _ in range(4):
        for i, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                got[i].append(run(*c, "silu"))
    torch.cuda.synchronize()
    for i, ref in enumerate(refs):
        for g in got[i]:
            assert all(torch.equal(g[name], ref[name]) for name in NAMES)


def test_autocast_and_leading_dimensions():
    layer = GatedMLP(128, 320, p=0.0, variant="blockwise[hip]", block_size=64).cuda()
    x = torch.randn(4, 33, 128, device="cuda")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = layer(x)
    assert y.shape == (4, 33, 128) and y.dtype == torch.bfloat16
    y.float().square().mean().backward()
    assert layer.weight_in.grad.shape == (640, 128) and layer.weight_out.grad.dtype == torch.float32


@pytest.mark.parametrize("variant", ["none", "vanilla", "blockwise[naive]", "blockwise[hip]"])
def test_layer_variants_agree_without_dropout(variant):
    torch.manual_seed(0)
    layer = GatedMLP(192, 256, 64, p=0.3, variant=variant, activation="gelu", block_size=64).cuda().bfloat16()
    x = torch.randn(100, 192, device="cuda").bfloat16()
    ref, bound = O.reference(x, layer.weight_in, layer.weight_out, torch.zeros(100, 64, device="cuda"), "gelu", torch.bfloat16)["y"]
    y = layer.eval()(x)
    # (torch's products, activation and multiplication round once more each)
    assert ((y.double() - ref).abs() <= (bound if variant == "blockwise[hip]" else 3 * bound)).all()
    layer.train()(x.requires_grad_()).float().square().sum().backward()
    assert x.grad.isfinite().all() and layer.weight_in.grad.any() and layer.weight_out.grad.any()


def test_backward_twice_and_changed_tensors():
    ops = operands(64, 64, 64, 64, "bf16", seed=12)
    leaves = [t.requires_grad_() for t in ops[:3]]
    y = F.gated_mlp(*leaves)
    y.backward(ops[3], retain_graph=True)
    first = [t.grad.clone() for t in leaves]
    for t in leaves:
        t.grad = None
    y.backward(ops[3])
    assert all(torch.equal(t.grad, g) for t, g in zip(leaves, first))
    with pytest.raises(RuntimeError):
        y.backward(ops[3])
    y = F.gated_mlp(*leaves)
    with torch.no_grad():
        leaves[1].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(ops[3])


def test_traced():
    x, w_in, w_out, _ = operands(64, 64, 96, 64, "bf16", seed=13)
    traced = torch.jit.trace(lambda a, b, c: F.gated_mlp(a, b, c, "gelu"), (x, w_in, w_out), check_trace=False)
    other = operands(64, 64, 96, 64, "bf16", seed=14)[:3]
    assert torch.equal(traced(*other), F.gated_mlp(*other, "gelu"))


def test_refusals():
    x, w_in, w_out, _ = operands(8, 64, 96, 32, "bf16")
    with pytest.raises(ValueError, match="both projections"):
        F.gated_mlp(x, w_in[:-1], w_out)
    with pytest.raises(ValueError, match="reduction dims"):
        F.gated_mlp(x[:, :-1], w_in, w_out)
    with pytest.raises(TypeError, match="same dtype"):
        F.gated_mlp(x, w_in, w_out.half())
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        F.gated_mlp(x.float(), w_in.float(), w_out.float())
    with pytest.raises(ValueError, match="must not be empty"):
        F.gated_mlp(x, w_in[:0], w_out[:, :0])
    with pytest.raises(ValueError, match="on the GPU|same device"):
        F.gated_mlp(x, w_in, w_out.cpu())
    with pytest.raises(ValueError, match="mask shape"):
        F.hip_blockwise_dropout_gated_mlp(x, w_in, w_out, 64, 0.5, masks=[torch.zeros(2, 1, dtype=torch.bool, device="cuda"), None], seed=1)
    with pytest.raises(NotImplementedError, match="forward mode"):
        with torch.autograd.forward_ad.dual_level():
            F.gated_mlp(torch.autograd.forward_ad.make_dual(x, x), w_in, w_out)


def few(x, w_in, w_out, act, pitches=(0, 0, 0, 0)):
    """The two launches for few rows, whatever is expected to be faster, between rows and bytes that must stay as they are."""
    (m, k), (n, f) = x.shape, w_out.shape
    lib, guard = _loader.load(), 7777.0

    def wide(t, more):
        big = torch.full((t.shape[0], t.shape[1] + more), guard, dtype=x.dtype, device="cuda")
        big[:, : t.shape[1]] = t
        return big

    xs, ws, os_ = (wide(t, p) for t, p in zip((x, w_in, w_out), pitches))
    y = torch.full((m + 2, n + pitches[3]), guard, dtype=x.dtype, device="cuda")
    need = lib.sd_gated_mlp_few_workspace_bytes(m, f, n)
    scratch = torch.full((need + 64,), 0x5a, dtype=torch.uint8, device="cuda")
    rc = lib.sd_gated_mlp_few(xs.data_ptr(), xs.stride(0), ws.data_ptr(), ws.stride(0), os_.data_ptr(), os_.stride(0), y[1:].data_ptr(), y.stride(0), m, k, f, n,
                              {"relu": 1, "gelu": 2, "silu": 3}[act], 1 if x.dtype == torch.bfloat16 else 0, scratch.data_ptr(), need,
                              torch.cuda.current_stream().cuda_stream)
    assert rc == 0, lib.sd_last_error()
    assert (y[0] == guard).all() and (y[-1] == guard).all() and (y[:, n:] == guard).all() and (scratch[need:] == 0x5a).all()
    return y[1:-1, :n]


@pytest.mark.parametrize("m", [1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 50, 64])
def test_few_rows(m):
    for i, (k, f, n) in enumerate(((64, 64, 64), (1, 1, 1), (63, 65, 3), (1024, 4096, 1024), (130, 5461, 300), (2048, 333, 2048), (200, 9000, 100))):
        dtype, act = ("bf16", "fp16")[i % 2], ("silu", "gelu", "relu")[i % 3]
        ops = operands(m, k, f, n, dtype, seed=40 + i)
        ref = O.reference(*ops, act, DT[dtype])
        check({"y": few(*ops[:3], act)}, ref)
        check({"y": few(*ops[:3], act, (3, 1, 5, 2))}, ref)


@pytest.mark.parametrize("m,k,f,n,plan", [(24, 1024, 4096, 1024, ",16 shares=4"), (48, 512, 8192, 2048, ",32 shares=4"), (16, 64, 8192, 2048, "shares=2"),
                                          (8, 64, 8193, 2047, "shares=2"), (24, 64, 8255, 2040, "shares=4")])
def test_few_rows_share_out_a_reduction(m, k, f, n, plan):
    ops = operands(m, k, f, n, "bf16", seed=45)
    got = few(*ops[:3], "silu", (0, 0, 1, 3))
    assert plan in _loader.load().sd_last_kernel_detail().decode()
    check({"y": got}, O.reference(*ops, "silu", torch.bfloat16))
    assert torch.equal(few(*ops[:3], "silu"), few(*ops[:3], "silu"))


def test_few_rows_keep_the_hidden_activations_to_more_than_their_type():
    """Up to 8 rows only the result is rounded to 16 bits: half a step of it, and the 32-bit sums' errors of the reference's bounds without u in them."""
    ops = operands(8, 512, 1024, 512, "bf16", seed=50)
    exact = O.reference(*ops, "silu", torch.bfloat16)["y"][0]
    wide = O.reference(*(t.double() for t in ops), "silu", torch.float32)["y"]  # (h in two halves is off by 2^-16 of itself, u^2)
    h = O.act((ops[0].double() @ ops[1].double().t())[:, :1024], "silu")[0] * (ops[0].double() @ ops[1].double().t())[:, 1024:]
    bound = wide[1] + 2.0 ** -8 * exact.abs() * 1.01 + 2.0 ** -16 * (h.abs() @ ops[2].double().abs().t())
    got = few(*ops[:3], "silu").double()
    assert ((got - exact).abs() <= bound).all()
    assert float(((got - exact).norm() / exact.norm())) < 2.0 ** -8 / 3 ** 0.5 * 1.05  # a uniform rounding error's, no more


def test_rows_behind_two_to_the_31_elements():
    m, k, f, n = 66000, 64, 16384 + 320, 64  # [G | U] has 2.2e9 elements
    gen = torch.Generator("cuda").manual_seed(51)
    make = lambda r, c, std: (torch.randn(r, c, generator=gen, device="cuda") * std).bfloat16()
    x, w_in, w_out, dy = make(m, k, 1.0), make(2 * f, k, k ** -0.5), make(n, f, f ** -0.5), make(m, n, 0.1)
    got = run(x, w_in, w_out, dy, "silu")
    for rows in (slice(0, 100), slice(m - 130, m)):
        ref = O.reference(x[rows], w_in, w_out, dy[rows], "silu", torch.bfloat16)
        check({name: got[name][rows] for name in ("y", "dx")}, ref)
    assert all(got[name].isfinite().all() for name in NAMES)


def test_product_and_gate_apart():
    """What is left to the kernel that takes any layout: the gate in passes of its own, in a process that is told to."""
    code = """
import sys
sys.path[:0] = [%r, %r, %r]
import torch
import test_gpu_gated as T
from oracle import gated_oracle as O
for size, p in (((64, 128, 192, 64), 0.0), ((130, 77, 99, 50), 0.0), ((130, 200, 332, 72), 0.4), ((70, 65, 130, 33), 0.4)):
    ops = T.operands(*size, "bf16", seed=60)
    masks = T.masks_of(*size[:3], 64, p) if p else (None, None)
    got = T.run(*ops, "gelu", 64, p, list(masks)) if p else T.run(*ops, "gelu")
    T.check(got, O.reference(*ops, "gelu", torch.bfloat16, masks, 64, (p, p)))
print("apart: right")
""" % tuple(os.path.join(os.path.dirname(os.path.abspath(__file__)), d) for d in (".", "..", os.path.join("..", "sparse-dropout_amd")))
    done = subprocess.run([sys.executable, "-c", code], env={**os.environ, "SPARSEDROP_FORCE_GENERIC": "1"}, capture_output=True, text=True, timeout=100)
    assert done.returncode == 0 and "apart: right" in done.stdout, done.stdout + done.stderr


@pytest.mark.parametrize("policy", [1, 2])
def test_either_size_of_tile(policy):
    """The large and the middle shapes on sizes that would not be given to them: ragged in every extent, dropped and not."""
    lib = _loader.load()
    was = lib.sd_set_tile_policy(policy)
    try:
        for i, size in enumerate(((257, 328, 712, 320), (64, 64, 64, 64), (300, 130, 1000, 136), (512, 512, 512, 512))):
            ops = operands(*size, "bf16", seed=70 + i)
            check(run(*ops, "silu"), O.reference(*ops, "silu", torch.bfloat16))
            for bs in (64, 32):
                masks = masks_of(*size[:3], bs, 0.4, seed=i)
                check(run(*ops, "gelu", bs, 0.4, masks), O.reference(*ops, "gelu", torch.bfloat16, masks, bs, (0.4, 0.4)))
    finally:
        lib.sd_set_tile_policy(was)


def test_saved_tensors_that_come_back_elsewhere():
    """Hooks that hand back copies in another layout (offloading does)."""
    ops = operands(65, 130, 99, 33, "bf16", seed=80)
    masks = masks_of(65, 130, 99, 64, 0.3)
    ref = run(*ops, "silu", 64, 0.3, masks)
    back = lambda t: t.t().contiguous().t() if t.dim() == 2 and t.is_floating_point() else t.clone()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: back(t.cuda())):
        got = run(*ops, "silu", 64, 0.3, masks)
    for name in NAMES:
        assert torch.equal(got[name], ref[name]), name


def test_a_gradient_in_any_layout_or_type():
    ops = operands(130, 64, 96, 40, "bf16", seed=81)
    leaves = [t.detach().requires_grad_() for t in ops[:3]]
    ref = run(*ops, "silu")
    for dy in (ops[3].t().contiguous().t(), torch.cat((ops[3], ops[3]), 1)[:, :40], torch.cat((ops[3][:, :1], ops[3]), 1)[:, 1:]):
        y = F.gated_mlp(*leaves)
        for g, name in zip(torch.autograd.grad(y, leaves, dy), NAMES[1:]):
            assert torch.equal(g, ref[name]), name
    y = F.gated_mlp(*leaves)
    y.float().sum().backward()  # an expanded gradient
    ones = run(*ops[:3], torch.ones(130, 40, device="cuda").bfloat16(), "silu")
    assert all(torch.equal(t.grad, ones[name]) for t, name in zip(leaves, NAMES[1:]))


@pytest.mark.parametrize("m", [3, 24, 40, 200])
@pytest.mark.parametrize("k,f,n", [(100, 77, 33), (65, 130, 64), (63, 62, 40), (136, 200, 72)])
def test_what_is_not_finite_stays_in_its_row(m, k, f, n):
    """An infinity or a NaN of a row reaches no other, wherever in the row it stands (the last elements are read with those in front of them)."""
    ops = operands(m, k, f, n, "fp16", seed=90)
    with torch.no_grad():
        ref = F.gated_mlp(*ops[:3], "relu")
        for bad in (math.inf, math.nan):
            for at in {0, k // 2, k - 2, k - 1}:
                x = ops[0].clone()
                x[1, at] = bad
                y = F.gated_mlp(x, *ops[1:3], "relu")
                others = torch.arange(m, device="cuda") != 1
                assert torch.equal(y[others], ref[others]), (bad, at)
                assert not torch.isfinite(y[1]).any(), (bad, at)


@pytest.mark.parametrize("m", [2, 20, 64])
@pytest.mark.parametrize("k,f,n", [(63, 65, 3), (129, 100, 66), (70, 64, 33), (5, 7, 3)])
def test_few_rows_read_nothing_beside_their_rows(m, k, f, n):
    """NaN in front of, behind and between all rows, which begin at every place of 16 bytes."""
    assert _loader.load().sd_gated_mlp_few_taken(m, k, f, n)
    ops = operands(m, k, f, n, "bf16", seed=91)
    ref = O.reference(*ops, "silu", torch.bfloat16)
    for before in range(8):
        views = []
        for t in ops[:3]:
            for behind in (1, 2):
                wide = torch.full((t.shape[0] + 2, before + t.shape[1] + behind), math.nan, dtype=t.dtype, device="cuda")
                inner = wide[1:-1, before:before + t.shape[1]]
                inner.copy_(t)
                views.append(inner)
        for shift in (0, 1):
            with torch.no_grad():
                check({"y": F.gated_mlp(*views[shift::2], "silu")}, ref)


@pytest.mark.parametrize("size", [(40, 140000, 64, 64), (8, 64, 140000, 40), (72, 64, 140000, 40)], ids=lambda s: "x".join(map(str, s)))
def test_very_long_reductions(size):
    """More blocks than a workgroup of the tile kernels walks: the gate in a pass of its own, or the reduction in parts."""
    ops = operands(*size, "bf16", seed=92)
    ref = O.reference(*ops, "silu", torch.bfloat16)
    check(run(*ops, "silu"), ref)
    with torch.no_grad():
        check({"y": F.gated_mlp(*ops[:3], "silu")}, ref)
    masks = masks_of(*size[:3], 64, 0.5)
    check(run(*ops, "gelu", 64, 0.5, masks), O.reference(*ops, "gelu", torch.bfloat16, masks, 64, (0.5, 0.5)))


def test_few_rows_captured_and_replayed():
    """Two graphs of the few rows of serving beside each other: either has a workspace of its own."""
    calls = []
    for i, size in enumerate(((1, 1024, 4096, 1024), (24, 333, 777, 100))):
        ops = operands(*size, "bf16", seed=93 + i)
        static = [t.clone() for t in ops[:3]]
        with torch.no_grad():
            F.gated_mlp(*static)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                y = F.gated_mlp(*static)
        calls.append((size, static, graph, y))
    side = torch.cuda.Stream()
    for seed in (95, 96, 97):
        refs = []
        for size, static, _, _ in calls:
            fresh = operands(*size, "bf16", seed=seed)
            with torch.no_grad():
                for t, v in zip(static, fresh):
                    t.copy_(v)
                refs.append(F.gated_mlp(*fresh[:3]))
        torch.cuda.synchronize()
        calls[0][2].replay()
        with torch.cuda.stream(side):
            calls[1][2].replay()
        torch.cuda.synchronize()
        for (_, _, _, y), ref in zip(calls, refs):
            assert torch.equal(y, ref)
