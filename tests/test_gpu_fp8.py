"""Matrices in 8 bits and their products on the GPU, against their definitions in 64 bits.

Tolerances.  Quantized values and scales are exact.  A product of two of them is exact in 64 bits; of the kernel's sum over K terms each
addition in fp32 is off by at most 2^-23 of the sum of magnitudes S, so all by at most K * 2^-23 * S.  The matrix cores add eight
consecutive products at a time, each cut to a multiple of 2^-13 of the power of two that the largest sum of two exponents stands for:
seven of them lose at most 2^-13 of that, which is less than the eight's part of S, together 7 * 2^-13 * S, where S takes codes below
the least normal one, and zeros, as that, because their exponent is its.  The result is rounded once: by half a step of its
type, or half of the type's least number.  That is much where S is far from the result, so a whole matrix is held to more: what
is cut off has either sign, a third of 2^-26 of the largest one's square on average; seven in eight products, of results whose own square is the sum
of all products' squares on average, are off by at most sqrt(7 / 3) * 2^-13 = 1.9e-4 of their norm, and 2^-11 allows for the spread.
Small whole numbers, whose products no cut touches, come out exactly."""
import numpy as np
import pytest
import torch

from oracle import fp8_oracle as O

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import flash_dropout.functional as F
    from flash_dropout.hip import GEMM
    from flash_dropout.layers import DropoutMM

DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def np64(t):
    return t.detach().double().cpu().numpy()


def check_product(got, ref, sums, terms, dtype):
    got = np64(got)
    assert got.shape == ref.shape
    info = torch.finfo(dtype)
    tol = info.eps / 2 * np.abs(ref) + (terms * 2.0 ** -23 + 7 * 2.0 ** -13) * sums * (1 + info.eps) + info.smallest_normal * info.eps / 2
    # (from half a step above the largest number on, a value rounds to infinity: a quarter of eps, the largest being 2 - eps times a power)
    over = np.isinf(got) & (np.sign(got) == np.sign(ref)) & (np.abs(ref) + tol >= info.max * (1 + info.eps / 4))
    with np.errstate(invalid="ignore"):
        bad = ~(np.abs(got - ref) <= tol) & ~(np.isnan(ref) & np.isnan(got)) & ~over
    if got.size >= 1000 and np.isfinite(got).all():
        norm = np.linalg.norm(ref)
        assert np.linalg.norm(got - ref) <= (info.eps / 2 + 2.0 ** -11) * norm + info.smallest_normal * info.eps * got.size ** 0.5
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), got[bad][:4], ref[bad][:4])


def spread(rows, cols, dtype, seed=0, device="cuda"):
    """Values over many binades: normal times powers of two, a few columns large, some zeros, one block of zeros."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=gen) * 2.0 ** torch.randint(-12, 6, (rows, cols), generator=gen)
    x[torch.rand(rows, cols, generator=gen) < 0.05] = 0
    x[:, : min(cols, 3)] *= 64
    if rows > 2 and cols > 130:
        x[1, 128:] = 0
    return x.to(dtype).to(device)


def expand(scales, side, rows, cols):
    return np.repeat(np.repeat(scales, side, 0), 128, 1)[:rows, :cols]


# ---- quantizing -------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("block", [(1, 128), (128, 128)])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 127), (128, 128), (129, 257), (77, 1025), (300, 64), (16, 4096), (1000, 130)])
def test_codes_and_scales_are_those_of_the_definition(rows, cols, block, dtype):
    x = spread(rows, cols, DT[dtype])
    data, scales = F.fp8_quantize(x, block)
    values, want = O.quantize(np64(x), block[0])
    wide = -(-cols // 128) * 128
    assert data.dtype == torch.float8_e4m3fn and tuple(data.shape) == (rows, wide)
    assert scales.dtype == torch.float8_e8m0fnu and tuple(scales.shape) == want.shape
    assert np.array_equal(np64(scales.float()), want)
    assert np.array_equal(np64(data.float())[:, :cols] * expand(want, block[0], rows, cols), values)
    assert not data[:, cols:].float().any()
    assert np.array_equal(np64(F.fp8_dequantize(data, scales, cols)), values)
    for out in (torch.float16, torch.bfloat16):  # rounded once, to nearest
        assert torch.equal(F.fp8_dequantize(data, scales, cols, out), torch.from_numpy(values).float().to(out).cuda())


def test_every_code_and_every_half_between_two_of_them():
    table = np.unique(np.abs(O.state_table("first")[np.isfinite(O.state_table("first"))]))
    mids = (table[1:] + table[:-1]) / 2
    tests = np.concatenate([table, mids, np.nextafter(mids.astype(np.float32), np.float32(0)), np.nextafter(mids.astype(np.float32), np.float32(1e9)), [2.0 ** -11]])
    tests = np.concatenate([tests, -tests])
    rows = -(-len(tests) // 127)
    x = torch.zeros(rows, 128)
    x[:, 0] = 448  # every row's scale is 1
    flat = np.zeros(rows * 127)
    flat[: len(tests)] = tests
    x[:, 1:] = torch.from_numpy(flat.reshape(rows, 127)).float()
    data, scales = F.fp8_quantize(x.cuda())
    assert (scales.float() == 1).all()
    assert np.array_equal(np64(data.float()), O.quantize(x.double().numpy(), 1)[0])


@pytest.mark.parametrize("dtype,values", [
    ("fp32", [0.0, 1e-45, 2.0 ** -127, 2.0 ** -126, 448.0, 448.0 * 2 ** 5, 449.0, 3.4e38, 2.0 ** -140]),
    ("bf16", [0.0, 1e-38, 448.0, 450.0, 3.3e38]),
    ("fp16", [0.0, 6e-8, 448.0, 448.25, 65504.0]),
])
def test_scales_at_the_borders(dtype, values):
    x = torch.zeros(len(values), 128, dtype=DT[dtype])
    for i, v in enumerate(values):
        x[i, 5] = v
        x[i, 6] = -v / 3
    data, scales = F.fp8_quantize(x.cuda())
    want, powers = O.quantize(x.double().numpy(), 1)
    assert np.array_equal(np64(scales.view(torch.uint8).float()), np.log2(powers) + 127)
    got = np64(data.float()) * powers
    assert np.array_equal(got, want)


@pytest.mark.parametrize("block", [(1, 128), (128, 128)])
def test_what_is_not_finite_becomes_nan_and_changes_no_scale(block):
    x = spread(130, 300, torch.float32)
    x[3, 7], x[4, 200], x[129, 299] = float("inf"), float("nan"), float("-inf")
    x[5] = float("nan")
    data, scales = F.fp8_quantize(x, block)
    values, want = O.quantize(np64(x), block[0])
    assert np.array_equal(np64(scales.float()), want)
    assert np.array_equal(np64(F.fp8_dequantize(data, scales, 300)), values, equal_nan=True)


@pytest.mark.parametrize("block", [(1, 128), (128, 128)])
@pytest.mark.parametrize("layout", ["columns", "slice", "odd offset", "expanded", "every other"])
def test_layouts(layout, block):
    base = spread(400, 600, torch.bfloat16)
    x = {"columns": base.t(), "slice": base[3:260, 8:400], "odd offset": base[1:, 1:300], "expanded": base[:1].expand(200, 600),
         "every other": base[::2, ::2]}[layout]
    data, scales = F.fp8_quantize(x, block)
    values, want = O.quantize(np64(x), block[0])
    assert np.array_equal(np64(scales.float()), want)
    assert np.array_equal(np64(F.fp8_dequantize(data, scales, x.shape[1])), values)


def test_empty_matrices():
    for shape in ((0, 200), (5, 0), (0, 0)):
        data, scales = F.fp8_quantize(torch.zeros(shape, device="cuda"))
        assert data.shape[0] == shape[0] and scales.shape[0] == shape[0]
        assert tuple(F.fp8_dequantize(data, scales, shape[1]).shape) == shape
    assert tuple(F.fp8_linear(torch.zeros(0, 128, device="cuda").half(), *F.fp8_quantize(torch.ones(5, 128, device="cuda"), (128, 128))).shape) == (0, 5)
    assert tuple(F.fp8_linear(torch.zeros(3, 128, device="cuda").half(), *F.fp8_quantize(torch.ones(0, 128, device="cuda"), (128, 128))).shape) == (3, 0)
    y = F.fp8_linear(torch.zeros(3, 0, device="cuda").half(), *F.fp8_quantize(torch.ones(4, 0, device="cuda"), (128, 128)))
    assert tuple(y.shape) == (3, 4) and not y.any()


# ---- serving ----------------------------------------------------------------------------------------------------------------
def serve(m, k, n, dtype, seed=0):
    x, w = spread(m, k, dtype, seed), spread(n, k, dtype, seed + 1)
    return x, w, *O.product(np64(x), 1, np64(w), 128)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 128, 16), (1, 4096, 1024), (2, 129, 17), (5, 1000, 130), (15, 257, 300), (16, 2200, 77), (17, 300, 129),
                                   (31, 128, 1), (64, 4096, 256), (128, 128, 128), (200, 2048, 640), (257, 513, 383), (1000, 384, 1000)])
def test_linear_with_kept_weights(m, k, n, dtype):
    x, w, ref, sums = serve(m, k, n, DT[dtype])
    y = F.fp8_linear(x / 64, *F.fp8_quantize(w, (128, 128)))
    check_product(y, ref / 64, sums / 64, k, DT[dtype])


@pytest.mark.parametrize("m", [3, 100])
def test_linear_takes_any_layout_of_its_operands(m):
    x, w, ref, sums = serve(m, 300, 200, torch.bfloat16)
    data, scales = F.fp8_quantize(w, (128, 128))
    want = F.fp8_linear(x, data, scales)
    check_product(want, ref, sums, 300, torch.bfloat16)
    wide = torch.zeros(m, 400, dtype=x.dtype, device="cuda")
    wide[:, 7:307] = x
    padded = torch.zeros(200, 512, dtype=torch.uint8, device="cuda")
    padded[:, :384] = data.view(torch.uint8)
    for xx, d, s in ((x.t().contiguous().t(), data, scales), (wide[:, 7:307], data, scales), (x, padded[:, :384].view(torch.float8_e4m3fn), scales),
                     (x, data, scales.view(torch.uint8).t().contiguous().t().view(torch.float8_e8m0fnu))):
        assert torch.equal(F.fp8_linear(xx, d, s), want)


@pytest.mark.parametrize("m", [4, 40])
def test_nan_stays_in_its_rows_and_columns(m):
    x, w, ref, sums = serve(m, 260, 140, torch.float16)
    x, ref, sums = x / 64, ref / 64, sums / 64
    x[1, 3] = float("nan")
    x[2, 5] = float("inf")
    data, scales = F.fp8_quantize(w, (128, 128))
    y = F.fp8_linear(x, data, scales)
    assert y[1:3].isnan().all()
    rest = [i for i in range(m) if i not in (1, 2)]
    check_product(y[rest], *O.product(np64(x[rest]), 1, np64(w), 128), 260, torch.float16)


@pytest.mark.parametrize("b_block", [(1, 128), (128, 128)])
@pytest.mark.parametrize("m,k,n", [(1, 128, 1), (130, 300, 257), (64, 8192, 64), (300, 1024, 520)])
def test_product_of_two_quantized_matrices(m, k, n, b_block):
    a, b = spread(m, k, torch.float32, 1), spread(n, k, torch.float32, 2)
    ref, sums = O.product(np64(a), 1, np64(b), b_block[0])
    for dtype in (torch.bfloat16, torch.float16):
        c = GEMM().gemm_fp8(*F.fp8_quantize(a / 256), *F.fp8_quantize(b, b_block), dtype)
        check_product(c, ref / 256, sums / 256, k, dtype)
    data, scales = F.fp8_quantize(a / 256)
    assert torch.equal(GEMM().gemm_fp8(data, scales.view(torch.uint8).contiguous().view(torch.float8_e8m0fnu), *F.fp8_quantize(b, b_block), torch.float16), c)


@pytest.mark.parametrize("k", [100, 128, 1000])
@pytest.mark.parametrize("m,n,a_rows,b_rows", [(700, 640, slice(500, 700), slice(512, 640)), (513, 300, slice(4, 513), slice(0, 127)),
                                               # 128 x 128 and 256 x 256 tiles that end inside; one that starts off a word
                                               (300, 500, slice(8, 263), slice(128, 387)), (8200, 8192, slice(4097, 8200), slice(4096, 8192)),
                                               (8192, 8300, slice(4000, 8192), slice(128, 8300))])
def test_products_of_some_rows_of_quantized_matrices(m, n, k, a_rows, b_rows):
    """Codes and scales are sliced where they lie; the results are those rows and columns of the product of matrices of their own."""
    a, b = spread(m, k, torch.float32, 1) / 256, spread(n, k, torch.float32, 2)
    for b_block in ((1, 128), (128, 128)):
        if b_block[0] == 128:
            b_rows = slice(b_rows.start // 128 * 128, b_rows.stop)
        qa, qb = F.fp8_quantize(a), F.fp8_quantize(b, b_block)
        sb = slice(b_rows.start // b_block[0], -(-b_rows.stop // b_block[0]))
        c = GEMM().gemm_fp8(qa[0][a_rows], qa[1][a_rows], qb[0][b_rows], qb[1][sb], torch.float16)
        own_a, own_b = (qa[0][a_rows].clone(), qa[1][a_rows].contiguous()), (qb[0][b_rows].clone(), qb[1][sb].contiguous())
        assert torch.equal(c, GEMM().gemm_fp8(*own_a, *own_b, torch.float16))
        rows, cols = torch.arange(m)[a_rows][::61], torch.arange(n)[b_rows][::53]
        va, vb = F.fp8_dequantize(*qa, k)[rows.cuda()], F.fp8_dequantize(*qb, k)[cols.cuda()]
        sums = O.magnitudes(np64(a), 1)[rows] @ O.magnitudes(np64(b), b_block[0])[cols].T
        picked = c[(rows - a_rows.start).cuda()][:, (cols - b_rows.start).cuda()]
        check_product(picked, np64(va) @ np64(vb).T, sums, k, torch.float16)


# ---- training ---------------------------------------------------------------------------------------------------------------
def train(m, k, n, dtype, bs, p, seed=0, mask=None):
    gen = torch.Generator().manual_seed(seed)
    x = spread(m, k, dtype, seed).div_(64).requires_grad_()
    w = spread(n, k, dtype, seed + 1).div_(64).requires_grad_()
    dy = spread(m, n, dtype, seed + 2).div_(64)
    if mask is None:
        mask = torch.rand(-(-m // bs), -(-k // bs), generator=gen) < p
    return x, w, dy, mask


def check_train(x, w, dy, mask, bs, p, y, dx, dw):
    m, k, n = *x.shape, w.shape[0]
    (ry, rdx, rdw), (sy, sdx, sdw) = O.train(np64(x), np64(w), np64(dy), mask.cpu().numpy(), bs, p)
    check_product(y, ry, sy, k + 1, x.dtype)  # (one more: the scale is rounded to 32 bits)
    if dx is not None:
        check_product(dx, rdx, sdx, n + 1, x.dtype)
    if dw is not None:
        check_product(dw, rdw, sdw, m + 1, x.dtype)


SHAPES = [(1, 1, 1), (128, 256, 256), (127, 129, 130), (300, 257, 77), (513, 640, 10), (1000, 384, 512), (64, 2048, 300), (2100, 130, 260), (256, 512, 1024)]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("bs,p", [(128, 0.0), (128, 0.5), (256, 0.3), (384, 0.6)])
def test_a_layer_and_its_gradients(m, k, n, bs, p, dtype):
    x, w, dy, mask = train(m, k, n, DT[dtype], bs, p)
    y = F.hip_blockwise_dropout_matmul_fp8_mask(x, mask.cuda(), bs, p, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    check_train(x, w, dy, mask, bs, p, y, dx, dw)


def whole(rows, cols, seed, dtype):
    """Whole numbers from -8 to 8: exact in 8 bits whatever block they are in, and so are their products and sums."""
    gen = torch.Generator().manual_seed(seed)
    return torch.randint(-8, 9, (rows, cols), generator=gen).to(dtype).cuda()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("m,k,n", SHAPES + [(700, 900, 1100), (2600, 1300, 400), (257, 4000, 513),
                                                       # 256 x 256 tiles for the forward, the input gradient and the weight gradient
                                                       (4001, 299, 4195), (3970, 4195, 299), (299, 4195, 4001), (4096, 4224, 128)])
@pytest.mark.parametrize("bs,p", [(128, 0.0), (128, 0.5), (256, 0.5), (384, 0.5)])
def test_whole_numbers_come_out_exactly(m, k, n, bs, p, dtype):
    dt = DT[dtype]
    x, w, dy = whole(m, k, 1, dt).requires_grad_(), whole(n, k, 2, dt).requires_grad_(), whole(m, n, 3, dt)
    mask = torch.rand(-(-m // bs), -(-k // bs), generator=torch.Generator().manual_seed(m + k)) < p
    y = F.hip_blockwise_dropout_matmul_fp8_mask(x, mask.cuda(), bs, p, w)
    got = (y, *torch.autograd.grad(y, (x, w), dy))
    s, keep = 1 / (1 - p), torch.from_numpy(O.keep_matrix(mask.numpy(), bs, m, k)).cuda()
    xd, wd, dyd = x.detach().double(), w.detach().double(), dy.double()
    for a, b in zip(got, (s * (xd * keep) @ wd.t(), s * (dyd @ wd) * keep, s * dyd.t() @ (xd * keep))):
        assert torch.equal(a, b.to(dt))
    data, scales = F.fp8_quantize(w.detach(), (128, 128))
    for rows in {min(m, r) for r in (1, 7, 16, 17, m)}:
        assert torch.equal(F.fp8_linear(x.detach()[:rows], data, scales), (xd[:rows] @ wd.t()).to(dt))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("m,k,n,bs,p,kernel", [
    # kept blocks of a row two at a time, with rows of none and of odd numbers
    (4777, 6601, 131, 128, 0.875, "fp8:duo"), (4777, 6601, 131, 256, 0.875, "fp8:duo"), (4800, 6656, 300, 384, 0.875, "fp8:duo"),
    (8192, 8192, 260, 128, 0.75, "fp8:duo"),
    # pairs of row blocks: hardly anything to leave out, few rounds, rows whose full ends share XCDs
    (4777, 6601, 131, 128, 0.25, "fp8:big"), (4096, 4096, 256, 128, 0.75, "fp8:big"), (4096, 8192, 256, 128, 0.5, "fp8:big"),
    (4200, 4099, 140, 256, 0.5, "fp8:big")])
def test_input_gradients_of_large_layers_on_the_tiles_that_pay(m, k, n, bs, p, kernel, dtype):
    dt = DT[dtype]
    x, w, dy = whole(m, k, 1, dt).requires_grad_(), whole(n, k, 2, dt), whole(m, n, 3, dt)
    mask = torch.rand(-(-m // bs), -(-k // bs), generator=torch.Generator().manual_seed(m + k)) < p
    mask[1] = True
    y = F.hip_blockwise_dropout_matmul_fp8_mask(x, mask.cuda(), bs, p, w)
    with torch.autograd.set_multithreading_enabled(False):  # (the last kernel is known by thread)
        dx, = torch.autograd.grad(y, x, dy)
    assert GEMM().last_kernel_detail().startswith(kernel)
    keep = torch.from_numpy(O.keep_matrix(mask.numpy(), bs, m, k)).cuda()
    # (exact sums, scaled in 32 bits)
    want = (dy.double() @ w.double()).float().mul_(1 / (1 - p)).double() * keep
    assert torch.equal(dx, want.to(dt))


@pytest.mark.parametrize("kind", ["all", "rows", "columns", "one kept"])
def test_masks_that_leave_rows_and_columns_empty(kind):
    m, k, n, bs = 520, 600, 300, 128
    mask = torch.zeros(5, 5, dtype=torch.bool)
    if kind == "all":
        mask[:] = True
    elif kind == "rows":
        mask[1::2] = True
    elif kind == "columns":
        mask[:, ::2] = True
    else:
        mask[:] = True
        mask[4, 3] = False
    x, w, dy, _ = train(m, k, n, torch.float16, bs, 0.5, mask=mask)
    with torch.no_grad():  # a dropped block is not read
        keep = torch.from_numpy(O.keep_matrix(mask.numpy(), bs, m, k)).cuda() > 0
        x[~keep] = float("nan")
    for mk in (mask.cuda(), mask.t().contiguous().t().cuda()):
        y = F.hip_blockwise_dropout_matmul_fp8_mask(x, mk, bs, 0.5, w)
        dx, dw = torch.autograd.grad(y, (x, w), dy)
        check_train(x, w, dy, mask, bs, 0.5, y, dx, dw)
        assert not dx[~keep].any()


@pytest.mark.parametrize("layout", ["x columns", "w columns", "dy columns", "dy expanded", "slices", "every other"])
def test_layouts_of_a_layers_operands(layout):
    m, k, n, bs, p = 300, 260, 140, 128, 0.4
    x, w, dy, mask = train(m, k, n, torch.bfloat16, bs, p)
    turned = lambda t: t.detach().t().contiguous().t()
    if layout == "x columns":
        x = turned(x).requires_grad_()
    elif layout == "w columns":
        w = turned(w).requires_grad_()
    elif layout == "dy columns":
        dy = turned(dy)
    elif layout == "dy expanded":
        dy = dy[:1].expand(m, n)
    elif layout == "slices":
        big = torch.zeros(m, k + 9, dtype=x.dtype, device="cuda")
        big[:, 5:5 + k] = x.detach()
        x = big[:, 5:5 + k].requires_grad_()
    else:
        big = torch.zeros(2 * n, 2 * k, dtype=x.dtype, device="cuda")
        big[::2, ::2] = w.detach()
        w = big[::2, ::2].requires_grad_()
    y = F.hip_blockwise_dropout_matmul_fp8_mask(x, mask.cuda(), bs, p, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    check_train(x, w, dy, mask, bs, p, y, dx, dw)


@pytest.mark.parametrize("wrt", ["x", "w", "neither"])
def test_only_the_gradients_that_are_asked_for(wrt):
    x, w, dy, mask = train(200, 300, 150, torch.float16, 128, 0.3)
    x.requires_grad_(wrt == "x")
    w.requires_grad_(wrt == "w")
    y = F.hip_blockwise_dropout_matmul_fp8_mask(x, mask.cuda(), 128, 0.3, w)
    assert y.requires_grad == (wrt != "neither")
    g = {}
    if wrt != "neither":
        g["dx" if wrt == "x" else "dw"], = torch.autograd.grad(y, x if wrt == "x" else w, dy)
    check_train(x, w, dy, mask, 128, 0.3, y, g.get("dx"), g.get("dw"))


def test_draws_are_those_of_the_16_bit_layer():
    x, w, dy, _ = train(500, 700, 260, torch.float16, 128, 0.5)
    mask, _ = GEMM().random_lists((4, 6), 0.5, 1234)
    y = F.hip_blockwise_dropout_matmul_fp8(x, w, 128, 0.5, seed=1234)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    check_train(x, w, dy, mask, 128, 0.5, y, dx, dw)
    mask, _ = GEMM().random_lists((2, 3), 0.5, 99)
    xt = x.detach().t().contiguous().t().requires_grad_()
    y = F.hip_blockwise_dropout_matmul_fp8(xt, w, 256, 0.5, seed=99)
    check_train(x, w, dy, mask, 256, 0.5, y, *torch.autograd.grad(y, (xt, w), dy))
    # from the generator's state: one draw a call
    GEMM().manual_seed(7)
    first = [F.hip_blockwise_dropout_matmul_fp8(x, w, 128, 0.5).detach() for _ in range(2)]
    assert not torch.equal(*first)
    assert GEMM().rng_state()[1].item() == 2
    GEMM().manual_seed(7)
    for want in first:
        assert torch.equal(F.hip_blockwise_dropout_matmul_fp8(x, w, 128, 0.5), want)


def test_gradients_against_differences():
    """Of the quantized matrices: a change of an input by one code's step moves the result along the gradient, to the second order
    (the product is linear in either operand, so there is none) but for the roundings of both."""
    m, k, n, bs, p = 256, 256, 128, 128, 0.5
    x, w, dy, mask = train(m, k, n, torch.float16, bs, p)
    with torch.no_grad():  # operands that are their own values in 8 bits, along rows and columns alike
        x.copy_(torch.randint(-8, 9, (m, k)).half())
        w.copy_(torch.randint(-8, 9, (n, k)).half())
        x[:, 0] = x[0] = 8
        x[:, 128] = x[128] = 8
        w[0, 0] = w[0, 128] = 8
    dy = torch.randint(-4, 5, (m, n)).half().cuda()
    f = lambda: (F.hip_blockwise_dropout_matmul_fp8_mask(x, mask.cuda(), bs, p, w).double() * dy.double()).sum()
    dx, dw = torch.autograd.grad(F.hip_blockwise_dropout_matmul_fp8_mask(x, mask.cuda(), bs, p, w), (x, w), dy)
    for t, g, i, j in ((x, dx, 5, 7), (x, dx, 200, 131), (w, dw, 100, 3), (w, dw, 7, 250)):
        with torch.no_grad():
            before = f()
            old = t[i, j].clone()
            t[i, j] = old + (1 if old < 8 else -1)
            step = (t[i, j] - old).double()
            after = f()
            t[i, j] = old
        # y is whole numbers below 2^11 times 2, exact in fp16 up to 2048: half a step of 2 otherwise, on the results that moved
        moved = n if t is x else m
        tol = moved * 4 * 2.0 + 1e-3 * abs(float(g[i, j]))
        assert abs(float(after - before) - float(g[i, j].double() * step)) <= tol


def test_the_layer_module_and_autocast():
    layer = DropoutMM(256, 384, p=0.25, variant="blockwise[hip-fp8]", block_size=128).cuda()
    x = torch.randn(2, 100, 256, device="cuda", requires_grad=True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        GEMM().manual_seed(3)
        y = layer(x)
    assert y.dtype == torch.bfloat16 and tuple(y.shape) == (2, 100, 384)
    y.float().square().mean().backward()
    assert x.grad.dtype == torch.float32 and layer.weight.grad.dtype == torch.float32
    GEMM().manual_seed(3)
    mask, _ = GEMM().random_lists((2, 2), 0.25)
    xb, wb = x.detach().reshape(200, 256).bfloat16(), layer.weight.detach().bfloat16()
    dy = (2 * y.detach().float() / y.numel()).bfloat16().reshape(200, 384)
    check_train(xb, wb, dy, mask, 128, 0.25, y.reshape(200, 384), x.grad.reshape(200, 256).bfloat16(), layer.weight.grad.bfloat16())
    layer.eval()
    with torch.no_grad():
        assert torch.equal(layer(x), torch.nn.functional.linear(x, layer.weight))


def test_a_captured_step_replays():
    torch.manual_seed(11)
    x, w, dy, _ = train(300, 512, 256, torch.float16, 128, 0.5)
    F.hip_blockwise_dropout_matmul_fp8(x, w, 128, 0.5)  # (makes the generator's state)
    xs, ws = x.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(F.hip_blockwise_dropout_matmul_fp8(xs, ws, 128, 0.5), (xs, ws), dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = F.hip_blockwise_dropout_matmul_fp8(xs, ws, 128, 0.5)
        dx, dw = torch.autograd.grad(y, (xs, ws), dy)
    GEMM().manual_seed(5)
    seen = []
    for i in range(3):
        GEMM().rng_state()[1] = i
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (y, dx, dw)]
        GEMM().rng_state()[1] = i
        want = F.hip_blockwise_dropout_matmul_fp8(xs, ws, 128, 0.5)
        for a, b in zip(got, (want, *torch.autograd.grad(want, (xs, ws), dy))):
            assert torch.equal(a, b)
        seen.append(got[0])
    assert not torch.equal(seen[0], seen[1])


def test_on_another_stream():
    x, w, dy, mask = train(300, 512, 256, torch.float16, 128, 0.5)
    mask = mask.cuda()
    want = F.hip_blockwise_dropout_matmul_fp8_mask(x, mask, 128, 0.5, w)
    wants = torch.autograd.grad(want, (x, w), dy)
    data, scales = F.fp8_quantize(w.detach(), (128, 128))
    served = F.fp8_linear(x.detach(), data, scales), F.fp8_linear(x.detach()[:4], data, scales)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = F.hip_blockwise_dropout_matmul_fp8_mask(x, mask, 128, 0.5, w)
        gots = torch.autograd.grad(got, (x, w), dy)
        d, s = F.fp8_quantize(w.detach(), (128, 128))
        again = F.fp8_linear(x.detach(), d, s), F.fp8_linear(x.detach()[:4], d, s)
    side.synchronize()
    for a, b in zip((want, *wants, *served), (got, *gots, *again)):
        assert torch.equal(a, b)


# ---- refusals ---------------------------------------------------------------------------------------------------------------
def test_refusals():
    x = torch.zeros(10, 256, device="cuda").half()
    w = torch.zeros(20, 256, device="cuda").half()
    mask = torch.zeros(1, 2, dtype=torch.bool, device="cuda")
    data, scales = F.fp8_quantize(w, (128, 128))
    with pytest.raises(ValueError):
        F.fp8_quantize(x, (64, 64))
    with pytest.raises(TypeError):
        F.fp8_quantize(x.double())
    with pytest.raises(ValueError):
        F.fp8_quantize(x[0])
    with pytest.raises(NotImplementedError):
        F.hip_blockwise_dropout_matmul_fp8(x, w, 64, 0.5)
    with pytest.raises(ValueError):
        F.hip_blockwise_dropout_matmul_fp8(x, w, 128, 1.0)
    with pytest.raises(ValueError):
        F.hip_blockwise_dropout_matmul_fp8_mask(x, mask[:, :1], 128, 0.5, w)
    with pytest.raises(TypeError):
        F.hip_blockwise_dropout_matmul_fp8_mask(x, mask.float(), 128, 0.5, w)
    with pytest.raises(TypeError):
        F.hip_blockwise_dropout_matmul_fp8_mask(x.float(), mask, 128, 0.5, w.float())
    with pytest.raises(TypeError):
        F.hip_blockwise_dropout_matmul_fp8_mask(x.bfloat16(), mask, 128, 0.5, w)
    with pytest.raises(ValueError):
        F.hip_blockwise_dropout_matmul_fp8_mask(x[:, :128], mask[:, :1], 128, 0.5, w)
    with pytest.raises(NotImplementedError):
        F.fp8_linear(x.clone().requires_grad_(), data, scales)
    with pytest.raises(TypeError):
        F.fp8_linear(x.float(), data, scales)
    with pytest.raises(ValueError):
        F.fp8_linear(x[:, :100], data, scales)
    with pytest.raises(ValueError):
        F.fp8_linear(x, data, scales[:, :1])
    with pytest.raises(TypeError):
        F.fp8_linear(x, data.view(torch.uint8), scales)
    with pytest.raises(NotImplementedError):
        F.fp8_linear(x, *F.fp8_quantize(w))
    with pytest.raises(NotImplementedError):
        GEMM().gemm_fp8(*F.fp8_quantize(torch.zeros(300, 128, device="cuda"), (128, 128)), *F.fp8_quantize(torch.zeros(300, 128, device="cuda")))
    with pytest.raises(ValueError):
        F.fp8_dequantize(data, scales, 100)
    y = F.hip_blockwise_dropout_matmul_fp8_mask(x.requires_grad_(), mask, 128, 0.5, w)
    torch.autograd.grad(y, x, torch.zeros_like(y))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, x, torch.zeros_like(y))
