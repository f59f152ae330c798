"""Values of the gated feed-forward block where they are not ordinary numbers, and what saved-tensor hooks hand back."""
import math

import pytest
import torch

from oracle import gated_oracle as O
from test_gpu_gated import DT, NAMES, check, masks_of, operands, run

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import flash_dropout.functional as F
    from flash_dropout.hip import _loader

ACTS = {"relu": 1, "gelu": 2, "silu": 3}


@pytest.fixture(params=[0, 1, 2], ids=["auto", "large", "middle"])
def tiles(request):
    lib = _loader.load()
    was = lib.sd_set_tile_policy(request.param)
    yield
    lib.sd_set_tile_policy(was)


def gate_apart(a, act, dh=None):
    """The gate as a pass of its own: H, or [dG | dU]."""
    lib, (m, f) = _loader.load(), (a.shape[0], a.shape[1] // 2)
    dtype, stream = int(a.dtype == torch.bfloat16), torch.cuda.current_stream().cuda_stream
    out = torch.empty(m, f if dh is None else 2 * f, dtype=a.dtype, device="cuda")
    if dh is None:
        rc = lib.sd_gated_forward(a.data_ptr(), 2 * f, f, out.data_ptr(), f, f, m, f, ACTS[act], dtype, stream)
    else:
        rc = lib.sd_gated_backward(dh.data_ptr(), f, a.data_ptr(), 2 * f, f, out.data_ptr(), 2 * f, 2 * f, m, f, ACTS[act], dtype, stream)
    assert rc == 0, lib.sd_last_error()
    return out


# ---- a NaN that only the gate has --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("m", [1, 8, 9, 24, 64, 200])
def test_nan_in_a_gate_reaches_every_output_of_serving(m, dtype, act):
    x, w_in, w_out, _ = operands(m, 136, 200, 72, dtype, seed=100)
    w_in[77, 5] = math.nan  # the gate's: U is finite everywhere
    with torch.no_grad():
        assert F.gated_mlp(x, w_in, w_out, act).isnan().all()


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("p", [0.0, 0.4])
@pytest.mark.parametrize("size", [(70, 136, 200, 72), (130, 77, 99, 50), (320, 256, 512, 128)], ids=lambda s: "x".join(map(str, s)))
def test_nan_in_a_gate_reaches_what_depends_on_it(size, p, act, tiles):
    m, k, f, n = size
    x, w_in, w_out, dy = operands(*size, "bf16", seed=101)
    masks = masks_of(m, k, f, 64, p) if p else None
    ref = run(x, w_in, w_out, dy, act, 64 if p else None, p, masks)
    wide = [~t.repeat_interleave(64, 0).repeat_interleave(64, 1) for t in masks] if p else [torch.ones(m, c, dtype=torch.bool, device="cuda") for c in (k, f)]
    both = wide[0][:m, 5:6] & wide[1][:m, :f]  # the gate is NaN there, if it is this column's, and H kept
    bad = int(both.any(0).nonzero()[-1])
    kept = both[:, bad]
    w_in[bad, 5] = math.nan
    got = run(x, w_in, w_out, dy, act, 64 if p else None, p, masks)
    assert got["y"][kept].isnan().all() and torch.equal(got["y"][~kept], ref["y"][~kept])
    away = torch.arange(k, device="cuda") != 5  # (column 5 of dx has the NaN of W_in itself as a factor)
    assert torch.equal(got["dx"][~kept][:, away], ref["dx"][~kept][:, away])
    assert got["dx"][kept][wide[0][:m, :k][kept]].isnan().all()
    assert got["dw_out"][:, bad].isnan().all() and got["dw_in"][bad].isnan().any() and got["dw_in"][f + bad].isnan().any()
    others = torch.arange(f, device="cuda") != bad
    assert torch.equal(got["dw_out"][:, others], ref["dw_out"][:, others])
    assert torch.equal(got["dw_in"][others.repeat(2)], ref["dw_in"][others.repeat(2)])


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("f", [40, 37])
def test_nan_in_a_gate_by_itself(f, act):
    for dtype in DT.values():
        a = torch.randn(50, 2 * f, device="cuda").to(dtype)
        dh = torch.randn(50, f, device="cuda").to(dtype)
        dh[dh == 0] = 1
        ref = gate_apart(a, act), gate_apart(a, act, dh)
        nan = torch.rand(50, f, device="cuda") < 0.2
        nan[:, -1] = True
        a[:, :f][nan] = math.nan
        h, da = gate_apart(a, act), gate_apart(a, act, dh)
        assert torch.equal(h.isnan(), nan) and torch.equal(h[~nan], ref[0][~nan])
        twice = torch.cat((nan, nan), 1)
        assert torch.equal(da.isnan(), twice) and torch.equal(da[~twice], ref[1][~twice])


# ---- infinite weights ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("m,k,f,n", [(1, 136, 200, 72), (5, 65, 99, 33), (8, 136, 200, 72), (8, 64, 8193, 2047), (9, 136, 200, 72), (24, 64, 4096, 1024), (200, 136, 200, 72)])
def test_infinite_output_weights_give_infinite_outputs(m, k, f, n, dtype):
    """An output with one infinite weight is an infinity of the sign of its product, with two NaN where the signs differ; others are as they were."""
    x, w_in, w_out, _ = operands(m, k, f, n, dtype, seed=102)
    h = (O.act((x.double() @ w_in.double().t())[:, :f], "silu")[0] * (x.double() @ w_in.double().t())[:, f:])
    # (the hidden columns furthest from 0 in every row: 16 bits hold their signs)
    one, two = h.abs().amin(0).topk(2).indices.tolist()
    assert float(h[:, [one, two]].abs().min()) > 2.0 ** -20
    with torch.no_grad():
        ref = F.gated_mlp(x, w_in, w_out)
        w_out[3, one], w_out[7, two], w_out[n - 1, one], w_out[n - 1, two] = math.inf, -math.inf, math.inf, math.inf
        y = F.gated_mlp(x, w_in, w_out)
    assert torch.equal(y[:, 3].double(), math.inf * h[:, one].sign()) and torch.equal(y[:, 7].double(), -math.inf * h[:, two].sign())
    both = math.inf * h[:, one].sign() + math.inf * h[:, two].sign()
    assert torch.equal(y[:, n - 1].isnan(), both.isnan()) and torch.equal(y[:, n - 1][~both.isnan()].double(), both[~both.isnan()])
    others = torch.ones(n, dtype=torch.bool, device="cuda")
    others[[3, 7, n - 1]] = False
    assert torch.equal(y[:, others], ref[:, others])


# ---- projections beyond fp16 ------------------------------------------------------------------------------------------------------
# The forward's gate is computed from 32-bit sums and the backward's from G and U in 16 bits, where what lies beyond 65504 is infinite.  Where an
# activation is flat (0 or 1 its slope, to the last of 32 bits) gradients do not depend on how far out G lies: calls with G inside of fp16 and beyond it
# have equal ones, bit by bit.
def far_operands(size, which, unit, value, seed=103):
    """Hidden column `unit` of G (which 0) or of U (1) is about value, up to a few times that, in every row."""
    m, k, f, n = size
    x, w_in, w_out, dy = operands(*size, "fp16", seed=seed)
    x = x.abs() + 0.5
    w_in[which * f + unit] = value / (1.3 * k)
    return x, w_in, w_out, dy


def equal_gradients(a, b, unit, f, names=NAMES, halves=(0, 1)):
    rows = torch.ones(2 * f, dtype=torch.bool, device="cuda")
    for half in (0, 1):
        rows[half * f + unit] = half in halves
    for name in names:
        x, y = (t[name][rows] if name == "dw_in" else t[name] for t in (a, b))
        assert y.isfinite().all(), name
        assert torch.equal(x, y), name


@pytest.mark.parametrize("p", [0.0, 0.4])
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("size", [(70, 136, 200, 72), (130, 77, 99, 50), (320, 256, 512, 128)], ids=lambda s: "x".join(map(str, s)))
def test_a_gate_far_below_zero_has_no_gradient(size, act, p, tiles):
    f, unit = size[2], 21
    masks = masks_of(*size[:3], 64, p) if p else None
    got = []
    for value in (-20000.0, -200000.0):
        x, w_in, w_out, dy = far_operands(size, 0, unit, value)
        assert (w_in[unit].isfinite().all()) and float((x.double() @ w_in[unit].double()).max()) < value / 3
        got.append(run(x, w_in, w_out, dy, act, 64 if p else None, p, masks))
    # dx sums products of gradients that are 0 with weights that differ
    equal_gradients(*got, unit, f)
    assert not got[1]["dw_in"][unit].any() and not got[1]["dw_in"][f + unit].any()


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("size", [(70, 136, 200, 72), (130, 77, 99, 50), (320, 256, 512, 128)], ids=lambda s: "x".join(map(str, s)))
def test_a_gate_far_above_zero_has_a_slope_of_one(size, act, tiles):
    """dG = dH U; act(G) itself, which dU is a multiple of, is not held."""
    f, unit = size[2], 21
    got = []
    for value in (20000.0, 200000.0):
        x, w_in, w_out, dy = far_operands(size, 0, unit, value)
        w_in[f + unit] *= 2.0 ** -10
        got.append(run(x, w_in, w_out, dy, act))
    assert got[0]["dw_in"][unit].any()
    equal_gradients(*got, unit, f, names=("dw_in",), halves=(0,))


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("size", [(70, 136, 200, 72), (130, 77, 99, 50), (320, 256, 512, 128)], ids=lambda s: "x".join(map(str, s)))
def test_behind_a_closed_gate_the_other_projection_may_be_anything(size, act, tiles):
    f, unit = size[2], 21
    got = []
    for value in (20000.0, 200000.0):
        x, w_in, w_out, dy = far_operands(size, 1, unit, value)
        w_in[unit] = -200.0 / size[1]  # the gate: under -100 in every row, where the slope is 0
        assert float((x.double() @ w_in[unit].double()).max()) < -110
        got.append(run(x, w_in, w_out, dy, act))
    equal_gradients(*got, unit, f)
    assert not got[1]["dw_in"][unit].any() and not got[1]["dw_in"][f + unit].any()


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("f", [40, 37])
def test_infinite_projections_of_a_gate_by_itself(f, act):
    for dtype in DT.values():
        a = torch.randn(30, 2 * f, device="cuda").to(dtype)
        dh = torch.randn(30, f, device="cuda").to(dtype)
        dh[dh == 0] = 1
        g, u = a[:, :f], a[:, f:]
        g[0], g[1], g[2], g[3] = -math.inf, math.inf, -math.inf, -200.0
        u[2], u[3], u[4] = math.inf, -math.inf, math.nan
        g[4], g[5], u[5] = -200.0, 200.0, math.inf
        da = gate_apart(a, act, dh)
        dg, du = da[:, :f], da[:, f:]
        assert not dg[[0, 2, 3]].any() and not du[[0, 2, 3]].any()
        assert torch.equal(dg[1].double(), (dh[1].double() * u[1].double()).to(dtype).double()) and du[1].isinf().all()
        assert dg[4].isnan().all() and not du[4].any()
        assert dg[5].isinf().all() and torch.equal(du[5].double(), (dh[5].double() * 200).to(dtype).double())
        assert da[6:].isfinite().all()


# ---- saved-tensor hooks ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("p", [0.0, 0.3])
@pytest.mark.parametrize("size", [(70, 136, 200, 72), (65, 130, 99, 33), (130, 77, 104, 56), (130, 80, 99, 50)], ids=lambda s: "x".join(map(str, s)))
def test_what_a_hook_hands_back_is_used(size, p):
    """Twice a saved operand gives twice the gradients that it is a factor of, whatever the widths."""
    m, k, f, n = size
    ops = operands(*size, "bf16", seed=104)
    masks = masks_of(m, k, f, 64, p) if p else None
    ref = run(*ops, "silu", 64 if p else None, p, masks)
    for i, name in ((0, "dw_in"), (1, "dx")):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t * 2 if t.shape == ops[i].shape and t.dtype == torch.bfloat16 else t):
            got = run(*ops, "silu", 64 if p else None, p, masks)
        for other in NAMES:
            assert torch.equal(got[other], ref[other] * 2 if other == name else ref[other]), (name, other)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t * 2 if t.shape == (n, f) and t.dtype == torch.bfloat16 else t):
        got = run(*ops, "silu", 64 if p else None, p, masks)
    assert torch.equal(got["dx"], ref["dx"] * 2) and torch.equal(got["dw_in"], ref["dw_in"] * 2) and torch.equal(got["dw_out"], ref["dw_out"])


@pytest.mark.parametrize("size", [(4000, 1024, 1040, 520), (4000, 1025, 1041, 523)], ids=lambda s: "x".join(map(str, s)))
def test_offloading_leaves_nothing_of_the_forward_on_the_gpu(size):
    ops = operands(*size, "bf16", seed=105)
    leaves = [t.requires_grad_() for t in ops[:3]]
    with torch.no_grad():
        F.gated_mlp(*leaves)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda()):
        y = F.gated_mlp(*leaves)
    assert torch.cuda.memory_allocated() - before <= y.numel() * 2 + (1 << 16)
    y.backward(ops[3])
    ref = run(*ops, "silu")
    assert all(torch.equal(t.grad, ref[name]) for t, name in zip(leaves, NAMES[1:]))


# ---- rows behind two to the 31 elements --------------------------------------------------------------------------------------------
def test_weight_gradients_of_rows_behind_two_to_the_31_elements():
    """Only the last rows have a gradient, so the weights' gradients are those of these rows alone."""
    m, k, f, n, last = 66000, 64, 16384 + 320, 64, 200  # [G | U] has 2.2e9 elements
    gen = torch.Generator("cuda").manual_seed(106)
    make = lambda r, c, std: (torch.randn(r, c, generator=gen, device="cuda") * std).bfloat16()
    x, w_in, w_out, dy = make(m, k, 1.0), make(2 * f, k, k ** -0.5), make(n, f, f ** -0.5), make(m, n, 0.1)
    dy[:-last] = 0
    got = run(x, w_in, w_out, dy, "silu")
    assert not got["dx"][:-last].any()
    ref = O.reference(x[-last:], w_in, w_out, dy[-last:], "silu", torch.bfloat16)
    check({"y": got["y"][-last:], "dx": got["dx"][-last:], "dw_in": got["dw_in"], "dw_out": got["dw_out"]}, ref)
