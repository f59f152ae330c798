"""What the products in 8 bits and AdamW refuse before anything runs on a GPU, and the sizes that they ask for."""
import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

from oracle import fp8_oracle as O

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture(scope="module")
def lib():
    from flash_dropout.hip import _loader

    return _loader.load()


FAKE = ctypes.c_void_p(0x1000)
ODD = ctypes.c_void_p(0x1008)
INVALID, UNSUPPORTED = 1, 2


def refused(lib, rc, code, text):
    assert rc == code and text in lib.sd_last_error(), (rc, lib.sd_last_error())


def test_sizes(lib):
    # codes with rows of whole 128-blocks, then the scales, to whole 16 bytes
    assert lib.sd_fp8_matrix_bytes(1, 1, 0) == 128 + 16
    assert lib.sd_fp8_matrix_bytes(17, 129, 0) == 17 * 256 + 2 * 32
    assert lib.sd_fp8_matrix_bytes(300, 300, 1) == 300 * 384 + 16
    assert lib.sd_fp8_matrix_bytes(0, 5, 0) == lib.sd_fp8_matrix_bytes(5, 0, 1) == 0
    assert lib.sd_fp8_matrix_bytes(70000, 70000, 0) > 2 ** 32
    for bad in ((-1, 1), (1, -1), (1 << 31, 1), (1, 1 << 31)):
        assert lib.sd_fp8_matrix_bytes(*bad, 0) == -1
        assert lib.sd_fp8_gemm_workspace_bytes(*bad, 1) == lib.sd_fp8_linear_workspace_bytes(1, *bad) == -1
        assert lib.sd_fp8_dropout_matmul_workspace_bytes(*bad, 1, 0) == -1
    # a few tokens take no workspace, more the input in 8 bits at least
    assert lib.sd_fp8_linear_workspace_bytes(16, 8192, 8192) == 0
    assert lib.sd_fp8_linear_workspace_bytes(65, 512, 512) >= lib.sd_fp8_matrix_bytes(65, 512, 0)
    # a reduction that does not fit a workgroup's list of kept blocks is cut into parts, whose sums are 4 bytes each
    m, n, k = 128 * 4097, 256, 256
    assert lib.sd_fp8_dropout_matmul_workspace_bytes(m, n, k, 1) >= lib.sd_fp8_matrix_bytes(m, n, 0) + 2 * 4 * n * k


def test_quantizer_refusals(lib):
    def q(x=FAKE, sr=256, sc=1, rows=10, cols=256, dtype=0, block=1, data=FAKE, ld=256, scales=FAKE, ssr=1, ssk=16):
        return lib.sd_fp8_quantize(x, sr, sc, rows, cols, dtype, block, data, ld, ctypes.cast(scales, ctypes.c_void_p), ssr, ssk, None)

    refused(lib, q(rows=-1), INVALID, b"negative")
    refused(lib, q(rows=1 << 31), INVALID, b"too large")
    refused(lib, q(dtype=3), INVALID, b"dtype")
    refused(lib, q(block=64), INVALID, b"1 x 128 or 128 x 128")
    refused(lib, q(x=None), INVALID, b"null pointer")
    refused(lib, q(sr=512, sc=2), INVALID, b"row or column major")
    refused(lib, q(sr=100), INVALID, b"row stride")
    refused(lib, q(data=None), INVALID, b"null pointer")
    refused(lib, q(data=ODD), INVALID, b"16 bytes")
    refused(lib, q(ld=264), INVALID, b"16 bytes")
    refused(lib, q(cols=250, ld=240), INVALID, b"whole 128-blocks")
    refused(lib, q(ssr=0), INVALID, b"positive")
    refused(lib, q(rows=1 << 30, cols=1 << 20, sr=1 << 20, ld=1 << 20, ssk=1 << 30), UNSUPPORTED, b"one launch")
    assert q(rows=0) == 0 and q(cols=0) == 0

    def d(data=FAKE, ld=256, scales=FAKE, block=1, rows=10, cols=256, out=FAKE, out_ld=256, dtype=0):
        return lib.sd_fp8_dequantize(data, ld, scales, 1, 16, block, rows, cols, out, out_ld, dtype, None)

    refused(lib, d(cols=-1), INVALID, b"negative")
    refused(lib, d(dtype=9), INVALID, b"dtype")
    refused(lib, d(block=2), INVALID, b"1 x 128 or 128 x 128")
    refused(lib, d(data=None), INVALID, b"null pointer")
    refused(lib, d(data=ODD), INVALID, b"16 bytes")
    refused(lib, d(ld=128), INVALID, b"does not hold")
    refused(lib, d(out=None), INVALID, b"null pointer")
    refused(lib, d(out_ld=255), INVALID, b"row stride")
    assert d(rows=0) == 0


def test_product_refusals(lib):
    def g(a=FAKE, lda=256, sa=FAKE, sal=16, b=FAKE, ldb=256, sb=FAKE, sbr=2, sbk=1, block=128, c=FAKE, csr=20, csc=1, M=10, N=20, K=256, dtype=0):
        return lib.sd_fp8_gemm(a, lda, sa, sal, b, ldb, sb, sbr, sbk, block, c, csr, csc, M, N, K, dtype, None, 0, None)

    refused(lib, g(M=-1), INVALID, b"negative")
    refused(lib, g(dtype=2), INVALID, b"dtype")
    refused(lib, g(block=32), INVALID, b"1 x 128 or 128 x 128")
    refused(lib, g(a=None), INVALID, b"null pointer")
    refused(lib, g(sa=None), INVALID, b"null pointer")
    refused(lib, g(b=ODD), INVALID, b"16 bytes")
    refused(lib, g(lda=250), INVALID, b"16 bytes")
    refused(lib, g(ldb=128), INVALID, b"does not hold")
    refused(lib, g(csr=19), INVALID, b"row stride")
    refused(lib, g(K=0), INVALID, b"empty reduction")
    refused(lib, g(sal=9), INVALID, b"A's scales")
    refused(lib, g(sal=18), INVALID, b"A's scales")
    refused(lib, g(sbk=0), INVALID, b"positive")
    refused(lib, g(block=1, sbr=1, sbk=18), INVALID, b"B's scales")
    refused(lib, g(block=1, sbr=2, sbk=32), INVALID, b"B's scales")
    refused(lib, g(lda=(1 << 22) + 128), UNSUPPORTED, b"pitch")
    refused(lib, g(lda=1 << 22, ldb=1 << 22, K=1 << 22, sal=1 << 16), UNSUPPORTED, b"too many scales")
    assert g(M=0) == 0 and g(N=0, csr=1) == 0

    def f(x=FAKE, ldx=256, w=FAKE, ldw=256, sw=FAKE, swr=2, swk=1, y=FAKE, ldy=20, M=10, N=20, K=256, dtype=0, ws=None, bytes_=0):
        return lib.sd_fp8_linear(x, ldx, w, ldw, sw, swr, swk, y, ldy, M, N, K, dtype, ws, bytes_, None)

    refused(lib, f(x=None), INVALID, b"null pointer")
    refused(lib, f(ldx=255), INVALID, b"row stride")
    refused(lib, f(w=ODD), INVALID, b"16 bytes")
    refused(lib, f(ldw=128), INVALID, b"does not hold")
    refused(lib, f(sw=None), INVALID, b"null pointer")
    refused(lib, f(ldy=19), INVALID, b"row stride")
    refused(lib, f(K=0), INVALID, b"empty reduction")
    refused(lib, f(swk=0), INVALID, b"positive")
    refused(lib, f(dtype=2), INVALID, b"dtype")
    refused(lib, f(M=100), INVALID, b"workspace")
    need = lib.sd_fp8_linear_workspace_bytes(100, 20, 256)
    refused(lib, f(M=100, ws=FAKE, bytes_=need - 1), INVALID, b"workspace")
    refused(lib, f(M=100, ws=ODD, bytes_=need), INVALID, b"workspace")
    refused(lib, f(K=(1 << 22) + 1, ldx=1 << 23, ldw=1 << 23), UNSUPPORTED, b"pitch")


def test_layer_refusals(lib):
    def fwd(x=FAKE, xsr=256, xsc=1, w=FAKE, y=FAKE, ysr=20, mask=FAKE, msr=2, msc=1, state=None, p=0.5, out=None, xt=None, wt=None, M=10, N=20,
            K=256, bs=128, dtype=0, ws=FAKE, bytes_=1 << 40):
        return lib.sd_fp8_dropout_matmul_forward(x, xsr, xsc, w, 256, 1, y, ysr, 1, mask, msr, msc, state, 0, 0, p, out, xt, wt, M, N, K, bs, dtype,
                                                 ws, bytes_, None)

    refused(lib, fwd(M=-5), INVALID, b"negative")
    refused(lib, fwd(M=0), INVALID, b"empty operand")
    refused(lib, fwd(dtype=2), INVALID, b"dtype")
    for p in (-0.1, 1.0, float("nan")):
        refused(lib, fwd(p=p), INVALID, b"p must be")
    refused(lib, fwd(bs=0), INVALID, b"positive")
    refused(lib, fwd(bs=192), UNSUPPORTED, b"multiples of 128")
    refused(lib, fwd(M=(1 << 22) + 1), UNSUPPORTED, b"too long")
    refused(lib, fwd(x=None), INVALID, b"null pointer")
    refused(lib, fwd(xsr=2, xsc=3), INVALID, b"row or column major")
    refused(lib, fwd(ysr=10), INVALID, b"row stride")
    refused(lib, fwd(xt=ODD), INVALID, b"16 bytes")
    refused(lib, fwd(msr=2, msc=3), INVALID, b"row or column major")
    refused(lib, fwd(mask=None), INVALID, b"mask_out")
    refused(lib, fwd(mask=None, out=FAKE, state=ctypes.c_void_p(0x1004)), INVALID, b"aligned")
    need = lib.sd_fp8_dropout_matmul_workspace_bytes(10, 20, 256, 0)
    refused(lib, fwd(bytes_=need - 1), INVALID, b"workspace")
    refused(lib, fwd(ws=None), INVALID, b"workspace")

    def bwd(dy=FAKE, mask=FAKE, xt=FAKE, wt=FAKE, dx=FAKE, dw=FAKE, M=10, N=20, K=256, bs=128, p=0.5, ws=FAKE, bytes_=1 << 40):
        return lib.sd_fp8_dropout_matmul_backward(dy, N, 1, mask, 2, 1, xt, wt, dx, K, 1, dw, K, 1, M, N, K, bs, p, 0, ws, bytes_, None)

    refused(lib, bwd(N=0), INVALID, b"no outputs")
    refused(lib, bwd(dx=None, dw=None), INVALID, b"neither gradient")
    refused(lib, bwd(mask=None), INVALID, b"mask")
    refused(lib, bwd(dy=None), INVALID, b"null pointer")
    refused(lib, bwd(wt=None), INVALID, b"needs WT")
    refused(lib, bwd(xt=ODD), INVALID, b"needs XT")
    refused(lib, bwd(bs=100), UNSUPPORTED, b"multiples of 128")
    refused(lib, bwd(bytes_=lib.sd_fp8_dropout_matmul_workspace_bytes(10, 20, 256, 1) - 1), INVALID, b"workspace")


def test_adamw_refusals(lib):
    pointers = (ctypes.c_void_p * 1)(0x1000)
    nothing = (ctypes.c_void_p * 1)(None)
    sizes = (ctypes.c_int64 * 1)(5)

    def step(count=1, p=pointers, g=pointers, m=pointers, v=pointers, ms=pointers, vs=pointers, n=sizes, at=FAKE, lr_at=None, lr=1e-3, b1=0.9,
             b2=0.99, eps=1e-8, decay=0.1, dtype=2, bits=8):
        return lib.sd_adamw_step(count, p, g, m, v, ms, vs, n, at, lr_at, lr, b1, b2, eps, decay, dtype, bits, 1, None)

    refused(lib, step(count=-1), INVALID, b"negative count")
    refused(lib, step(dtype=3), INVALID, b"dtype")
    refused(lib, step(bits=16), INVALID, b"8 or in 32 bits")
    refused(lib, step(at=None), INVALID, b"step")
    refused(lib, step(at=ctypes.c_void_p(0x1004)), INVALID, b"step")
    for kw, text in ((dict(lr=-1.0), b"lr"), (dict(lr=float("nan")), b"lr"), (dict(lr=float("inf")), b"lr"), (dict(b1=1.0), b"betas"), (dict(b2=-0.1), b"betas"),
                     (dict(eps=-1e-8), b"eps"), (dict(eps=1e-39), b"eps"), (dict(eps=float("nan")), b"eps"), (dict(eps=1e37), b"eps"),
                     (dict(decay=-0.1), b"weight_decay")):
        refused(lib, step(**kw), INVALID, text)
    refused(lib, step(n=None), INVALID, b"null array")
    refused(lib, step(g=None), INVALID, b"null array")
    refused(lib, step(m=nothing), INVALID, b"null pointer")
    refused(lib, step(vs=nothing), INVALID, b"scales")
    refused(lib, step(ms=None), INVALID, b"scales")
    refused(lib, step(n=(ctypes.c_int64 * 1)(-5)), INVALID, b"negative size")
    refused(lib, step(n=(ctypes.c_int64 * 1)(1 << 43)), UNSUPPORTED, b"too large")
    second = (ctypes.c_int32 * 1)(0)
    values = lambda count=1, c=pointers, n=sizes: lib.sd_adamw_state_values(count, c, pointers, pointers, n, second, None)  # noqa: E731
    refused(lib, values(count=-1), INVALID, b"negative count")
    refused(lib, values(c=None), INVALID, b"null array")
    refused(lib, values(c=nothing), INVALID, b"null pointer")
    refused(lib, values(n=(ctypes.c_int64 * 1)(-1)), INVALID, b"negative size")
    assert values(count=0) == 0


def test_operands_on_the_cpu_are_refused():
    import flash_dropout.functional as F
    from flash_dropout.hip import GEMM
    from flash_dropout.layers import DropoutMM
    from flash_dropout.optim import AdamW

    x = torch.zeros(4, 256, dtype=torch.float16)
    data, scales = torch.zeros(4, 256).to(torch.float8_e4m3fn), torch.ones(1, 2).to(torch.float8_e8m0fnu)
    for call in (lambda: F.fp8_quantize(x), lambda: F.fp8_dequantize(data, scales), lambda: F.fp8_linear(x, data, scales),
                 lambda: GEMM().gemm_fp8(data, scales, data, scales),
                 lambda: F.hip_blockwise_dropout_matmul_fp8_mask(x, torch.zeros(1, 2, dtype=torch.bool), 128, 0.5, x),
                 lambda: F.hip_blockwise_dropout_matmul_fp8(x, x, 128, 0.5, seed=1),
                 lambda: F.adamw_step([x], [x], [x.float()], [x.float()], torch.zeros((), dtype=torch.int64)),
                 lambda: F.adamw_state_values([(torch.zeros(4, dtype=torch.uint8), torch.zeros(1, dtype=torch.uint8))] * 2,
                                              [(torch.zeros(4, dtype=torch.uint8), torch.zeros(1, dtype=torch.uint8))] * 2)):
        with pytest.raises(ValueError):
            call()
    for bs in (0, -128, 1.5, (128, 256)):
        with pytest.raises(ValueError):
            F.hip_blockwise_dropout_matmul_fp8(x, x, bs, 0.5)
    p = torch.nn.Parameter(torch.zeros(3))
    for kw in (dict(eps=1e-39), dict(eps=1e37), dict(eps=-1.0), dict(lr=-1e-3), dict(betas=(0.9, 1.0)), dict(weight_decay=-1.0), dict(state_bits=16)):
        with pytest.raises(ValueError):
            AdamW([p], **kw)
    p.grad = torch.zeros(3)
    with pytest.raises(ValueError):
        AdamW([p]).step()
    with pytest.raises(ValueError, match="8 or in 32"):
        AdamW([dict(params=[p], state_bits=4)]).step()
    assert DropoutMM(4, 4, variant="blockwise[hip-fp8]", block_size=128).eval()(torch.zeros(2, 4)).shape == (2, 4)


def test_the_states_random_bits_leave_averages_right_on_average():
    """A value's two neighbours come up with the probabilities that its place says: over 4096 elements and 16 steps a share of 1/4 is
    off by more than 6 sqrt(1/4 * 3/4 / 65536) = 0.0102 once in 10^8 draws."""
    n, steps = 4096, range(1, 17)
    for which, step_between in (("first", 2.0), ("second", 2.0)):
        x = O.np.full(n, 16 + step_between / 4)  # a quarter of the way from 16 to 18
        x[::128] = 448.0 if which == "first" else 61440.0  # scales of 1
        got = O.np.stack([O.rounded_state(x, which, s) for s in steps])
        got = O.np.delete(got, O.np.arange(0, n, 128), 1)
        assert set(O.np.unique(got)) == {16.0, 18.0}
        assert abs((got == 18.0).mean() - 0.25) <= 0.0104  # (a 128th of them are the large ones)


def test_scales_that_lie_far_apart_are_refused(lib):
    """The tiles read them by 32-bit offsets; strides over one block are nobody's business."""
    def g(N, K, sbr, sbk):
        return lib.sd_fp8_gemm(FAKE, 1 << 20, FAKE, 16, FAKE, 1 << 20, FAKE, sbr, sbk, 128, FAKE, N, 1, 10, N, K, 0, None, 0, None)

    def f(N, K, swr, swk, ws=FAKE):
        return lib.sd_fp8_linear(FAKE, K, FAKE, 1 << 20, FAKE, swr, swk, FAKE, N, 100, N, K, 0, ws, 1 << 40, None)

    for call in (g, f):
        for N, K, sr, sk in ((300, 256, 1 << 30, 1), (256, 128, 1 << 31, 1), (1000, 256, 1 << 40, 1), (1 << 20, 1 << 20, 1 << 62, 1),
                             (300, 300, 1 << 29, (1 << 29) + 1), (128 << 10, 128, (1 << 21) + 4096, 1)):
            refused(lib, call(N, K, sr, sk), UNSUPPORTED, b"too far")
    refused(lib, f(128, 256, 1 << 40, 1, None), INVALID, b"workspace")
    refused(lib, f(256, 256, (1 << 31) - 3, 1, None), INVALID, b"workspace")


def test_drop_rates_that_round_to_one_draw_no_mask(lib):
    """The draw compares in 32 bits and would drop everything; a mask that is given has no rate to be drawn by."""
    def fwd(p, mask, out, ws):
        return lib.sd_fp8_dropout_matmul_forward(FAKE, 256, 1, FAKE, 256, 1, FAKE, 20, 1, mask, 2, 1, None, 0, 0, p, out, None, None, 10, 20, 256, 128, 0,
                                                 ws, 1 << 40, None)

    for p in (1 - 2.0 ** -26, 1 - 2.0 ** -53):
        refused(lib, fwd(p, None, FAKE, FAKE), INVALID, b"in 32 bits")
        refused(lib, fwd(p, FAKE, None, None), INVALID, b"workspace")
    refused(lib, fwd(1 - 2.0 ** -24, None, FAKE, None), INVALID, b"workspace")


_SCALE_READS = r"""
#include <stdio.h>
#include <initializer_list>
#include "fp8_scales.h"

static long n_words = 0, n_cut = 0;

// What the lanes of a tile of `tile` rows from `first` on ask for, a word each in every 128-block, of scales that are not followed by
// anything: a word is read if it ends within the bound, whole words only.
static bool holds(int64_t nk, int64_t ld, int64_t rows, int64_t first, int64_t tile) {
  const int64_t left = sd::row_scales_left(nk, ld, rows, first), end = (nk - 1) * ld + rows;
  for (int64_t k = 0; k < nk; ++k)
    for (int64_t lane = 0; lane < tile / 4; ++lane) {
      const int64_t off = k * ld + 4 * lane, row = first + 4 * lane;
      const bool read = off + 4 <= left;
      ++n_words;
      n_cut += !read;
      if (read && first + off >= end) return false;  // the word holds nothing that is there
      if (!read && row < rows) return false;         // a row of the matrix is missing
    }
  return true;
}

int main() {
  for (int64_t nk : {1, 2, 3, 9})
    for (int64_t rows = 1; rows <= 600; rows += rows < 270 ? 1 : 37)
      for (int64_t more : {0, 4, 12, 16, 128, 7916})
        for (int64_t tile : {128, 256})
          for (int64_t first = 0; first < rows; first += tile) {
            const int64_t ld = (rows + 3) / 4 * 4 + more;
            if (holds(nk, ld, rows, first, tile)) continue;
            printf("%ld blocks of %ld rows, %ld apart, tile of %ld from %ld\n", (long)nk, (long)rows, (long)ld, (long)tile, (long)first);
            return 1;
          }
  return n_words < 1000000 || n_cut < 10000;
}
"""


def test_row_scales_are_not_read_behind_their_end(tmp_path):
    """Scales of some rows of a larger matrix (csrc/fp8_scales.h): the last 128-block's row of them may be the end of the memory."""
    (tmp_path / "sweep.cpp").write_text(_SCALE_READS)
    subprocess.run(["g++", "-O2", "-std=c++17", f"-I{ROOT / 'sparse-dropout_amd' / 'csrc'}", str(tmp_path / "sweep.cpp"), "-o",
                    str(tmp_path / "sweep")], check=True)
    proc = subprocess.run([str(tmp_path / "sweep")], capture_output=True, text=True, timeout=100)
    assert proc.returncode == 0, proc.stdout


def test_traces_record_the_quantizer_and_refuse_the_optimizer(monkeypatch):
    """Around stand-ins for the native calls, whose results are filled behind torch's back."""
    import flash_dropout.functional as F
    from flash_dropout.functional import adamw, fp8_blocks
    from flash_dropout.hip import GEMM
    from flash_dropout.optim import AdamW

    class Bridge:
        @staticmethod
        def fp8_quantize(x, rows):
            data, scales = torch.empty(x.shape), torch.empty(x.shape[0], 1)
            data.numpy()[:], scales.numpy()[:] = x.detach().numpy(), rows
            return data.to(torch.float8_e4m3fn), scales.to(torch.float8_e8m0fnu)

        @staticmethod
        def fp8_dequantize(data, scales, cols, dtype):
            out = torch.empty(data.shape[0], cols)
            out.numpy()[:] = data.float().numpy()[:, :cols] * scales.float().numpy()
            return out.to(dtype)

        adamw_step = adamw_state_values = staticmethod(lambda *args: [])

    for module in (fp8_blocks, adamw):
        monkeypatch.setattr(module._loader, "bridge", lambda: Bridge)

    def f(x):
        data, scales = F.fp8_quantize(x, block=(128, 128))
        return data.float(), scales.float(), F.fp8_dequantize(data, scales, x.shape[1], torch.float64) * 2

    make = lambda start: torch.arange(start, start + 8.0).view(2, 4)  # noqa: E731
    for wanted in (False, True):  # (the results carry no gradient, traced or not)
        traced = torch.jit.trace(f, (make(0).requires_grad_(wanted),), check_trace=False)
        got, want = traced(make(4).requires_grad_(wanted)), f(make(4).requires_grad_(wanted))
        assert all(torch.equal(a, b) and not a.requires_grad and not b.requires_grad for a, b in zip(got, want))
        assert want[2].dtype == torch.float64 and want[2][1, 3] == 2 * 128 * 11
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.zeros(3)
    step = torch.zeros((), dtype=torch.int64)
    for call in (lambda x: F.adamw_step([x], [x], [x], [x], step) or x, lambda x: F.adamw_state_values([(x, x)], [(x, x)]) and x,
                 lambda x: AdamW([p]).step() or x, lambda x: GEMM().gemm_fp8(x, x, x, x)):
        with pytest.raises(NotImplementedError, match="cannot be traced"):
            torch.jit.trace(call, (torch.zeros(3),), check_trace=False)
    F.adamw_step([p], [p], [p], [p], step)


def _steps_taken(params, bits):
    """An optimizer as it is after seven steps, its averages numbered by their place in memory."""
    from flash_dropout.optim import AdamW

    opt = AdamW(params, state_bits=bits)
    for p in params:
        opt._init_state(p, bits, torch.full((), 7, dtype=torch.int64))
        state = opt.state[p]
        for key in ("exp_avg", "exp_avg_sq"):
            flat = torch.as_strided(state[key], (p.numel(),), (1,))
            flat.copy_(torch.arange(p.numel()) % 100 + (key == "exp_avg_sq"))
    return opt


def _layouts():
    w = torch.zeros(2, 3, 2, 2)
    return {"rows": w, "channels last": w.contiguous(memory_format=torch.channels_last), "turned": torch.zeros(2, 2, 3, 2).permute(3, 2, 0, 1)}


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("saved", ["rows", "channels last", "turned"])
@pytest.mark.parametrize("loaded", ["rows", "channels last", "turned"])
def test_saved_averages_stay_with_their_elements(saved, loaded, bits, tmp_path):
    """Averages in 32 bits take their parameter's layout; those in 8, whose codes share scales along the memory, are refused in another one."""
    from flash_dropout.optim import AdamW

    make = lambda kind: [torch.nn.Parameter(_layouts()[kind]), torch.nn.Parameter(torch.zeros(5)), torch.nn.Parameter(torch.zeros(4, 1, 3))]  # noqa: E731
    old, new = make(saved), make(loaded)
    opt, again = _steps_taken(old, bits), AdamW(new, state_bits=bits, lr=5.0)
    torch.save(opt.state_dict(), tmp_path / "s.pt")
    state_dict = torch.load(tmp_path / "s.pt", weights_only=True)
    if bits == 8 and saved != loaded:
        with pytest.raises(ValueError, match="fit none of"):
            again.load_state_dict(state_dict)
        assert not again.state and again.param_groups[0]["lr"] == 5.0
        return
    again.load_state_dict(state_dict)
    for p, q in zip(old, new):
        for key in ("exp_avg", "exp_avg_sq"):
            a, b = opt.state[p][key], again.state[q][key]
            assert torch.equal(a, b) and a.shape == b.shape and b.dtype == a.dtype and b.stride() == q.stride()
        assert again.state[q]["step"].item() == 7 and again.state[q]["step"].dtype == torch.int64


def test_strides_of_extents_of_one_are_no_layout():
    from flash_dropout.optim import AdamW

    p, q = (torch.nn.Parameter(torch.as_strided(torch.zeros(12), (4, 1, 3), strides)) for strides in ((3, 3, 1), (3, 100, 1)))
    opt, again = _steps_taken([p], 8), AdamW([q], state_bits=8)
    again.load_state_dict(opt.state_dict())
    assert torch.equal(again.state[q]["exp_avg"], opt.state[p]["exp_avg"]) and again.state[q]["exp_avg"].stride() == q.stride()


def test_codes_saved_without_a_shape_are_of_contiguous_parameters():
    from flash_dropout.optim import AdamW

    opt = _steps_taken([torch.nn.Parameter(_layouts()["rows"])], 8)
    state_dict = opt.state_dict()
    for key in ("exp_avg", "exp_avg_sq"):
        state_dict["state"][0][key] = state_dict["state"][0][key].view(-1)
    for kind in ("rows", "channels last"):
        p = torch.nn.Parameter(_layouts()[kind])
        again = AdamW([p], state_bits=8)
        if kind == "rows":
            again.load_state_dict(state_dict)
            assert torch.equal(again.state[p]["exp_avg"].view(-1), state_dict["state"][0]["exp_avg"])
        else:
            with pytest.raises(ValueError, match="fit none of"):
                again.load_state_dict(state_dict)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [8, 32])
def test_a_state_of_torchs_optimizer_is_loaded(bits, dtype):
    """Averages in 32 bits whatever the parameters' type, the settings that torch's has no name for as they were, parameters without a state too."""
    from flash_dropout.optim import AdamW

    make = lambda: [torch.nn.Parameter(torch.ones(3, 5, dtype=dtype)), torch.nn.Parameter(torch.ones(4, dtype=dtype))]  # noqa: E731
    theirs, ours = make(), make()
    other = torch.optim.AdamW(theirs, lr=0.25, betas=(0.5, 0.75), eps=1e-6, weight_decay=0.125)
    theirs[0].grad = torch.full((3, 5), 0.5, dtype=dtype)
    for _ in range(2):
        other.step()
    opt = AdamW(ours, state_bits=bits)
    opt.load_state_dict(other.state_dict())
    group = opt.param_groups[0]
    assert {k: group[k] for k in ("lr", "betas", "eps", "weight_decay", "state_bits")} == dict(lr=0.25, betas=(0.5, 0.75), eps=1e-6, weight_decay=0.125, state_bits=bits)
    state = opt.state[ours[0]]
    for key in ("exp_avg", "exp_avg_sq"):
        assert state[key].dtype == torch.float32 and torch.equal(state[key], other.state[theirs[0]][key].float())
    assert state["step"].item() == 2 and state["step"].dtype == torch.int64 and not opt.state.get(ours[1])
    ours[1].grad = torch.ones(4, dtype=dtype)
    with pytest.raises(ValueError, match="on the GPU"):  # (a step as far as it goes here)
        opt.step()
    assert ("exp_avg_scale" in opt.state[ours[1]]) == (bits == 8)
    for key in ("amsgrad", "maximize"):
        other = torch.optim.AdamW(theirs, **{key: True})
        opt = AdamW(ours, state_bits=bits)
        with pytest.raises(ValueError, match=key):
            opt.load_state_dict(other.state_dict())
        assert key not in opt.param_groups[0]


@pytest.mark.parametrize("bits", [8, 32])
def test_hooks_around_a_load_see_what_is_loaded(bits):
    """One in front may replace the state, one behind finds the averages as they were saved."""
    import copy

    from flash_dropout.optim import AdamW

    make = lambda: [torch.nn.Parameter(torch.zeros(300, dtype=torch.bfloat16)), torch.nn.Parameter(torch.zeros(2, dtype=torch.bfloat16))]  # noqa: E731
    opt, ours = _steps_taken(make(), bits), make()
    again, seen = AdamW(ours, state_bits=bits), []

    def replace(_, given):
        given = copy.deepcopy(given)
        for state in given["state"].values():
            state["exp_avg"] += 3
            state["step"] += 1
        return given

    again.register_load_state_dict_pre_hook(replace)
    again.register_load_state_dict_post_hook(lambda o: seen.append([(o.state[p]["exp_avg"].clone(), o.state[p]["step"].item()) for p in ours]))
    saved = opt.state_dict()
    for _ in range(2):
        again.load_state_dict(saved)
    for p, (average, step), state in zip(ours * 2, seen[0] + seen[1], [*saved["state"].values()] * 2):
        assert torch.equal(average, state["exp_avg"] + 3) and average.dtype == state["exp_avg"].dtype and step == 8
    assert again.state[ours[0]]["step"] is again.state[ours[1]]["step"]
