"""Values of the gated feed-forward block where they are not ordinary numbers."""
import math

import pytest
import torch

from oracle import gated_oracle as O
from test_gpu_gated import DT, masks_of, operands, run

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
