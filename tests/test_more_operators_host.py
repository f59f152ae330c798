"""What the gated block and the clipping refuse before they reach the GPU, and the gated block's oracle against differences."""
import ctypes
import math

import pytest
import torch

from flash_dropout import functional as F
from flash_dropout.hip import _loader
from flash_dropout.layers import GatedMLP
from flash_dropout.optim import AdamW, clip_grad_norm_
from oracle import gated_oracle as O

fake = 0x1000


def test_gate_calls_refuse_bad_arguments():
    lib = _loader.load()
    ok = dict(A=fake, lda=16, up=8, H=fake, ldh=8, h_cols=8, M=4, F=8, act=3, dtype=1)
    fwd = lambda **kw: lib.sd_gated_forward(*{**ok, **kw}.values(), None)
    for bad, message in ((dict(A=None), b"null pointer"), (dict(lda=15), b"pitch"), (dict(up=7), b"U begins"), (dict(ldh=7), b"pitch"), (dict(H=None), b"null pointer"),
                         (dict(h_cols=9, ldh=16), b"zeros up to"), (dict(h_cols=7), b"zeros up to"), (dict(M=-1), b"extents"), (dict(F=1 << 30), b"extents"),
                         (dict(act=0), b"act must be"), (dict(act=4), b"act must be"), (dict(dtype=2), b"dtype")):
        assert fwd(**bad) == 1 and message in lib.sd_last_error(), bad
    assert fwd(M=0, A=None, H=None) == 0
    ok_back = dict(dH=fake, ldd=8, A=fake, lda=16, up=8, dA=fake, ldda=16, da_cols=16, M=4, F=8, act=2, dtype=0)
    bwd = lambda **kw: lib.sd_gated_backward(*{**ok_back, **kw}.values(), None)
    for bad, message in ((dict(dH=None), b"null gradient"), (dict(ldd=7), b"pitch"), (dict(dA=None), b"null pointer"), (dict(ldda=15), b"pitch"), (dict(lda=8), b"pitch"),
                         (dict(da_cols=17, ldda=24), b"zeros up to")):
        assert bwd(**bad) == 1 and message in lib.sd_last_error(), bad


def test_gated_products_refuse_bad_arguments():
    lib = _loader.load()
    ok = dict(X=fake, xr=64, xc=1, W=fake, wr=64, wc=1, H=fake, ldh=32, h_cols=32, A=fake, lda=64, up=32, rows=None, cols=None, M=128, F=32, K=64, bs=64, scale=1.0, act=3,
              dtype=1)
    call = lambda **kw: lib.sd_gated_matmul(*{**ok, **kw}.values(), None)
    for bad, message in ((dict(act=0), b"act must be"), (dict(up=31), b"U begins"), (dict(lda=63), b"pitch"), (dict(rows=fake), b"both be given"), (dict(scale=math.nan), b"NaN"),
                         (dict(rows=fake, cols=fake, bs=0), b"positive"), (dict(xr=63), b"row stride"), (dict(wr=63), b"row stride"), (dict(W=None), b"null pointer"),
                         (dict(ldh=31), b"row stride"), (dict(h_cols=33, ldh=40), b"next multiple of 8"), (dict(h_cols=31), b"next multiple of 8"), (dict(dtype=2), b"dtype")):
        assert call(**bad) == 1 and message in lib.sd_last_error(), bad
    assert call(rows=fake, cols=fake, bs=48) == 2 and call(K=0) == 2 and call(M=0) == 0 and call(F=0, h_cols=0) == 0
    ok = dict(X=fake, xr=64, xc=1, W=fake, wr=64, wc=1, H=fake, ldh=32, h_cols=32, A=fake, lda=64, up=32, mask=fake, mr=1, mc=1, state=None, seed=0, offset=0, p=0.5, out=None,
              rp=fake, ci=fake, cp=fake, ri=fake, M=128, F=32, K=64, bs=64, act=3, dtype=1)
    call = lambda **kw: lib.sd_gated_dropout_matmul_forward(*{**ok, **kw}.values(), None)
    for bad, message in ((dict(p=1.0), b"p must be"), (dict(p=-0.1), b"p must be"), (dict(rp=None), b"CSR list arrays"), (dict(mask=None), b"null mask_out"), (dict(M=0), b"empty"),
                         (dict(mr=2, mc=2), b"row or column major"), (dict(mask=None, out=fake, state=fake + 4), b"aligned device pointer"), (dict(act=5), b"act must be")):
        assert call(**bad) == 1 and message in lib.sd_last_error(), bad
    assert call(bs=48) == 2
    ok = dict(dY=fake, gr=16, gc=1, W=fake, wr=32, wc=1, A=fake, lda=64, up=32, dA=fake, ldda=64, cols=64, H=fake, hr=32, hc=1, dW=fake, dr=32, dc=1, rp=None, ci=None, cp=None,
              ri=None, M=128, F=32, N=16, bs=64, p=0.0, act=3, dtype=1, ws=None, nbytes=0)
    call = lambda **kw: lib.sd_gated_matmul_gradient(*{**ok, **kw}.values(), None)
    for bad, message in ((dict(p=1.0), b"p must be"), (dict(A=None), b"null [G | U]"), (dict(dA=None), b"null pointer"), (dict(ldda=63), b"pitch"), (dict(cols=65, ldda=72), b"multiple of 8"),
                         (dict(rp=fake, ci=fake), b"CSC lists"), (dict(cp=fake), b"both be given"), (dict(hr=31), b"stride"), (dict(gr=15), b"row stride"), (dict(act=0), b"act")):
        assert call(**bad) == 1 and message in lib.sd_last_error(), bad
    assert call(N=0) == 2 and call(M=0) == 0


def test_few_rows_refuse_bad_arguments():
    lib = _loader.load()
    assert lib.sd_gated_mlp_few_workspace_bytes(1, 64, 16) == 2 * 16 * 64 and lib.sd_gated_mlp_few_workspace_bytes(9, 65, 3) == 2 * 9 * 192
    assert lib.sd_gated_mlp_few_workspace_bytes(24, 4096, 1024) == 2 * 24 * 65 * 64 + 4 * 4 * 24 * 1024  # a reduction in four shares
    assert [lib.sd_gated_mlp_few_workspace_bytes(*a) for a in ((0, 64, 8), (65, 64, 8), (4, 0, 8), (4, 1 << 29, 8), (4, 64, 0), (4, 64, 1 << 29))] == [0] * 6
    assert lib.sd_gated_mlp_few_taken(1, 1024, 4096, 1024) == 1 and lib.sd_gated_mlp_few_taken(16, 8192, 8192, 8192) == 1
    assert [lib.sd_gated_mlp_few_taken(*a) for a in ((0, 64, 64, 64), (65, 64, 64, 64), (4, 0, 64, 64), (4, 64, 1 << 29, 64), (64, 2048, 8192, 2048))] == [0] * 5
    need = lib.sd_gated_mlp_few_workspace_bytes(4, 64, 16)
    ok = dict(X=fake, ldx=32, Wi=fake, ldwi=32, Wo=fake, ldwo=64, Y=fake, ldy=16, M=4, K=32, F=64, N=16, act=3, dtype=0, ws=fake, nbytes=need)
    call = lambda **kw: lib.sd_gated_mlp_few(*{**ok, **kw}.values(), None)
    for bad, message in ((dict(K=0), b"extents"), (dict(M=-1), b"extents"), (dict(F=1 << 29), b"extents"), (dict(dtype=2), b"dtype"), (dict(act=0), b"act"), (dict(X=None), b"null"),
                         (dict(ldx=31), b"pitch"), (dict(ldwi=31), b"pitch"), (dict(ldwo=63), b"pitch"), (dict(ldy=15), b"pitch"), (dict(nbytes=need - 1), b"too small"),
                         (dict(ws=fake + 8), b"aligned")):
        assert call(**bad) == 1 and message in lib.sd_last_error(), bad
    assert call(M=0) == 0 and call(M=65) == 2 and b"at most 64" in lib.sd_last_error()


def test_norm_calls_refuse_bad_arguments():
    lib = _loader.load()
    n = 3

    def call(fn, sizes=(5, 0, 8193), types=(0, 1, 2), pointers=(fake, None, fake), kind=2, limit=1.0, norm=fake, ws=fake, nbytes=1 << 20, count=n):
        p, s, t = (ctypes.c_void_p * n)(*pointers), (ctypes.c_int64 * n)(*sizes), (ctypes.c_int32 * n)(*types)
        if fn == "clip":
            return lib.sd_clip_grads(count, p, s, t, kind, limit, norm, ws, nbytes, None)
        return lib.sd_grad_norm(count, p, s, t, kind, limit, norm, fake, ws, nbytes, None)

    need = lib.sd_grad_norm_workspace_bytes(n, (ctypes.c_int64 * n)(5, 0, 8193))
    assert need == 8 * 3 and lib.sd_grad_norm_workspace_bytes(0, None) == 0
    assert lib.sd_grad_norm_workspace_bytes(1, (ctypes.c_int64 * 1)(1 << 40)) == 8 * 1024
    for fn in ("norm", "clip"):
        for bad, message in ((dict(sizes=(5, -1, 2)), b"negative size"), (dict(types=(0, 1, 3)), b"dtype"), (dict(pointers=(None, None, fake)), b"null pointer"),
                             (dict(kind=1), b"norm_type"), (dict(limit=-1.0), b"max_norm"), (dict(limit=math.nan), b"max_norm"), (dict(norm=None), b"null norm"),
                             (dict(ws=None), b"workspace too small"), (dict(nbytes=need - 1), b"workspace too small"), (dict(ws=fake + 4), b"8-byte aligned"),
                             (dict(count=-1), b"negative count")):
            assert call(fn, **bad) == 1 and message in lib.sd_last_error(), (fn, bad)
        assert call(fn, sizes=(1 << 42, 0, 1)) == 2 and b"too large" in lib.sd_last_error()


def test_python_refusals():
    x, w_in, w_out = torch.ones(4, 8), torch.ones(12, 8), torch.ones(8, 6)
    with pytest.raises(ValueError, match="gate is one of"):
        F.gated_mlp(x, w_in, w_out, "tanh")
    with pytest.raises(ValueError, match="must be on the GPU"):
        F.gated_mlp(x, w_in, w_out)
    for p in (1.0, -0.1, (0.5,), (0.5, 1.0), (0.1, 0.2, 0.3)):
        with pytest.raises(ValueError, match="p must be"):
            F.hip_blockwise_dropout_gated_mlp(x, w_in, w_out, 64, p)
    with pytest.raises(ValueError, match="masks are"):
        F.hip_blockwise_dropout_gated_mlp(x, w_in, w_out, 64, 0.5, masks=[None])
    with pytest.raises(ValueError, match="activation"):
        GatedMLP(8, 16, activation="tanh")
    with pytest.raises(ValueError, match="Unknown variant"):
        GatedMLP(8, 16, variant="other")(x)
    with pytest.raises(ValueError, match="one GPU"):
        F.grad_norm([x])
    with pytest.raises(ValueError, match="norm_type"):
        F.clip_grad_norm_([x], 1.0, 1.0)
    with pytest.raises(ValueError, match="at least one"):
        F.grad_norm([])
    assert float(clip_grad_norm_([torch.nn.Parameter(x)], 1.0)) == 0.0
    assert AdamW([torch.nn.Parameter(x)], max_norm=2.0).max_norm == 2.0


def test_layer_on_the_cpu():
    torch.manual_seed(0)
    for variant in ("none", "vanilla", "blockwise[naive]"):
        layer = GatedMLP(24, 40, 16, p=0.0, variant=variant, activation="silu", block_size=32).double()
        x = torch.randn(3, 5, 24).double()
        for mode in (layer.train(), layer.eval()):
            y = mode(x)
            assert y.shape == (3, 5, 16)
            ref = O.block(x.reshape(-1, 24), layer.weight_in, layer.weight_out, "silu", 1.0, 1.0)
            torch.testing.assert_close(y.reshape(-1, 16), ref)


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("dropped", [False, True])
def test_oracle_gradients_against_differences(act, dropped):
    """Central differences in 64 bits: off by h^2 / 6 of a third derivative and 2^-52 / h of the value, under 1e-6 of it with h = 1e-5; ReLU's kinks lie
    further than that from any of these 0.9 k values."""
    gen = torch.Generator().manual_seed(3)
    m, k, f, n, bs = 7, 5, 6, 4, 2
    x, w_in, w_out, dy = (torch.randn(s, generator=gen, dtype=torch.float64) for s in ((m, k), (2 * f, k), (n, f), (m, n)))
    masks = [torch.rand(-(-m // bs), -(-c // bs), generator=gen) < 0.4 for c in (k, f)] if dropped else (None, None)
    ps = (0.4, 0.4) if dropped else (0.0, 0.0)
    ref = O.reference(x, w_in, w_out, dy, act, torch.float16, masks, bs, ps)
    by = [O.keep(masks[i], bs, m, c, ps[i], x) for i, c in enumerate((k, f))]
    value = lambda: float((O.block(x, w_in, w_out, act, *by) * dy).sum())
    torch.testing.assert_close(ref["y"][0], O.block(x, w_in, w_out, act, *by))
    for name, t in (("dx", x), ("dw_in", w_in), ("dw_out", w_out)):
        flat, grad = t.view(-1), ref[name][0].reshape(-1)
        for i in range(flat.numel()):
            h, was = 1e-5, float(flat[i])
            flat[i] = was + h
            up = value()
            flat[i] = was - h
            down = value()
            flat[i] = was
            assert abs((up - down) / (2 * h) - float(grad[i])) < 1e-6 * (1 + abs(float(grad[i]))), (name, i)
