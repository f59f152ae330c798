// extern "C" surface of the products in 8 bits and of AdamW: argument validation, the layout of buffers and dispatch.  No kernels here.
#include "fp8.h"

#include <cfloat>

namespace sd {

int launch_dequantize(const uint8_t* data, int64_t ld, const uint8_t* scales, int64_t s_r, int64_t s_k, int square, int64_t rows,
                      int64_t cols, void* out, int64_t out_ld, int dtype, hipStream_t stream);
int launch_adamw(int count, void* const* p, const void* const* g, void* const* m, void* const* v, uint8_t* const* ms, uint8_t* const* vs,
                 const int64_t* n, int64_t* step, const float* lr_at, double lr, double beta1, double beta2, double eps, double decay,
                 int dtype, int bits, bool moves_on, const float* grad_scale, hipStream_t stream);
int launch_state_values(int count, const uint8_t* const* codes, const uint8_t* const* scales, float* const* out, const int64_t* n,
                        const int32_t* second, hipStream_t stream);

namespace {

constexpr int64_t kMaxDim = 1LL << 31;
// 255 rows of a tile and a row's bytes within a 32-bit offset
constexpr int64_t kMaxPitch = 1LL << 22;

int64_t up(int64_t v, int64_t to) { return ceil_div(v, to) * to; }
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// A matrix in 8 bits in one buffer: codes with a pitch of whole 128-blocks, then scales.  Not square: a row of scales for each
// 128-block, of a multiple of 16 bytes; square: a row for each 128 rows.
struct Packed {
  int64_t rows, nk, ld, s_ld, codes, bytes;
  bool square;
  Packed(int64_t rows_, int64_t cols, bool square_) : rows(rows_), nk(ceil_div(cols, kFp8Block)), square(square_) {
    ld = nk * kFp8Block;
    codes = rows * ld;
    s_ld = square ? nk : up(rows, 16);
    bytes = codes + up(square ? ceil_div(rows, kFp8Block) * nk : nk * s_ld, 16);
  }
  uint8_t* scales(void* at) const { return static_cast<uint8_t*>(at) + codes; }
  Fp8Form form(void* at) const {
    if (at == nullptr) return Fp8Form{};
    return Fp8Form{static_cast<uint8_t*>(at), ld, scales(at), square ? s_ld : 1, square ? 1 : s_ld};
  }
};

int check_sizes(const char* fn, int64_t rows, int64_t cols) {
  SD_REQUIRE(rows >= 0 && cols >= 0, "%s: negative dimension", fn);
  SD_REQUIRE(rows < kMaxDim && cols < kMaxDim, "%s: dimension too large", fn);
  return SD_OK;
}
// what the products' 32-bit offsets reach: a reduction of K over operands of `rows` rows at most
int check_reach(const char* fn, int64_t rows, int64_t K) {
  if (up(K, kFp8Block) > kMaxPitch) return fail(SD_ERR_UNSUPPORTED, "%s: a reduction of %lld is too long (at most %lld)", fn, (long long)K, (long long)kMaxPitch);
  if (ceil_div(K, kFp8Block) * up(rows, 16) >= (1LL << 31)) return fail(SD_ERR_UNSUPPORTED, "%s: a %lld x %lld operand has too many scales", fn, (long long)rows, (long long)K);
  return SD_OK;
}
// the last of 128 x 128 blocks' scales within the tiles' 32-bit offsets
int check_square_scales(const char* fn, int64_t rows, int64_t nk, int64_t sr, int64_t sk) {
  const int64_t r = ceil_div(rows, kFp8Block) - 1, k = nk - 1, most = (1LL << 31) - 2;
  const bool far = (r > 0 && sr > most) || (k > 0 && sk > most) || (r > 0 ? r * sr : 0) + (k > 0 ? k * sk : 0) > most;
  return far ? fail(SD_ERR_UNSUPPORTED, "%s: scales %lld and %lld apart reach too far", fn, (long long)sr, (long long)sk) : SD_OK;
}
int check_matrix(const char* fn, const char* name, const void* p, int64_t sr, int64_t sc, int64_t rows, int64_t cols) {
  SD_REQUIRE(p != nullptr || rows == 0 || cols == 0, "%s: %s: null pointer", fn, name);
  SD_REQUIRE(sr == 1 || sc == 1, "%s: %s must be row or column major (strides %lld, %lld)", fn, name, (long long)sr, (long long)sc);
  SD_REQUIRE(sr >= 1 && sc >= 1, "%s: %s: strides must be positive", fn, name);
  if (sc == 1 && rows > 1) SD_REQUIRE(sr >= cols, "%s: %s: row stride %lld < %lld columns", fn, name, (long long)sr, (long long)cols);
  if (sr == 1 && sc != 1 && cols > 1) SD_REQUIRE(sc >= rows, "%s: %s: column stride %lld < %lld rows", fn, name, (long long)sc, (long long)rows);
  return SD_OK;
}
int check_codes(const char* fn, const char* name, const void* data, int64_t ld, const uint8_t* scales, int64_t rows, int64_t cols) {
  SD_REQUIRE(rows == 0 || cols == 0 || (data != nullptr && scales != nullptr), "%s: %s: null pointer", fn, name);
  SD_REQUIRE(aligned16(data) && ld % 16 == 0, "%s: %s: codes must start on 16 bytes, rows too (pitch %lld)", fn, name, (long long)ld);
  SD_REQUIRE(ld >= up(cols, kFp8Block), "%s: %s: a pitch of %lld does not hold %lld columns in whole 128-blocks", fn, name, (long long)ld, (long long)cols);
  return SD_OK;
}
int check_pitch(const char* fn, int64_t ld) {
  return ld <= kMaxPitch ? SD_OK : fail(SD_ERR_UNSUPPORTED, "%s: a pitch of %lld is too large (at most %lld)", fn, (long long)ld, (long long)kMaxPitch);
}
int check_dtype(const char* fn, int dtype) {
  SD_REQUIRE(dtype == SD_F16 || dtype == SD_BF16, "%s: dtype must be SD_F16 or SD_BF16 (got %d)", fn, dtype);
  return SD_OK;
}

// the job that brings a row- or column-major [rows, cols] matrix into 8 bits: `plain` codes [rows][cols], `turned` [cols][rows]
QuantJob quant_job(const void* x, int64_t sr, int64_t sc, int64_t rows, int64_t cols, Fp8Form plain, Fp8Form turned, bool square) {
  QuantJob j = {};
  j.src = x;
  j.square = square ? 1 : 0;
  if (sc == 1) {
    j.ld = sr;
    j.rows = (int32_t)rows;
    j.cols = (int32_t)cols;
    j.along = plain;
    j.across = turned;
  } else {  // the transpose of a row-major matrix
    j.ld = sc;
    j.rows = (int32_t)cols;
    j.cols = (int32_t)rows;
    j.along = turned;
    j.across = plain;
    j.mask_t = 1;
  }
  return j;
}

Fp8Gemm product(const Packed& a, void* pa, const Packed& b, void* pb, void* c, int64_t csr, int64_t csc, int64_t M, int64_t N, int64_t K,
                float scale, void* part, int64_t part_bytes) {
  Fp8Gemm g = {};
  g.a = static_cast<uint8_t*>(pa);
  g.lda = a.ld;
  g.sa = a.scales(pa);
  g.sa_ld = a.s_ld;
  g.b = static_cast<uint8_t*>(pb);
  g.ldb = b.ld;
  g.sb = b.scales(pb);
  g.sb_square = b.square ? 1 : 0;
  g.sb_r = b.s_ld;
  g.sb_k = b.square ? 1 : b.s_ld;
  g.c = static_cast<uint16_t*>(c);
  g.c_sr = csr;
  g.c_sc = csc;
  g.M = M;
  g.N = N;
  g.K = K;
  g.scale = scale;
  g.split = 1;
  g.keep = 1.f;
  g.part = static_cast<float*>(part);
  g.part_bytes = part_bytes;
  return g;
}

int check_workspace(const char* fn, const void* ws, int64_t have, int64_t need) {
  SD_REQUIRE(need == 0 || (ws != nullptr && have >= need && aligned16(ws)), "%s: workspace too small or not on 16 bytes (%lld bytes, %lld needed)", fn,
             (long long)have, (long long)need);
  return SD_OK;
}

}  // namespace
}  // namespace sd

using namespace sd;

extern "C" {

int64_t sd_fp8_matrix_bytes(int64_t rows, int64_t cols, int square) {
  if (rows < 0 || cols < 0 || rows >= kMaxDim || cols >= kMaxDim) return -1;
  return Packed(rows, cols, square != 0).bytes;
}

int sd_fp8_quantize(const void* x, int64_t sr, int64_t sc, int64_t rows, int64_t cols, int dtype, int64_t block_rows, void* data,
                    int64_t data_ld, uint8_t* scales, int64_t ssr, int64_t ssk, void* stream) {
  if (int rc = check_sizes("fp8_quantize", rows, cols)) return rc;
  SD_REQUIRE(dtype == SD_F16 || dtype == SD_BF16 || dtype == SD_F32, "fp8_quantize: dtype must be SD_F16, SD_BF16 or SD_F32 (got %d)", dtype);
  SD_REQUIRE(block_rows == 1 || block_rows == kFp8Block, "fp8_quantize: blocks are of 1 x 128 or 128 x 128 (got %lld rows)", (long long)block_rows);
  if (int rc = check_matrix("fp8_quantize", "x", x, sr, sc, rows, cols)) return rc;
  if (rows == 0 || cols == 0) return SD_OK;
  SD_REQUIRE(data != nullptr && scales != nullptr, "fp8_quantize: null pointer");
  SD_REQUIRE(aligned16(data) && data_ld % 16 == 0 && data_ld >= up(cols, kFp8Block),
             "fp8_quantize: codes must start on 16 bytes, rows too, and their pitch hold whole 128-blocks (got %lld)", (long long)data_ld);
  SD_REQUIRE(ssr >= 1 && ssk >= 1, "fp8_quantize: scales: strides must be positive");
  QuantJobs js = {};
  js.n = 1;
  js.job[0] = quant_job(x, sr, sc, rows, cols, Fp8Form{static_cast<uint8_t*>(data), data_ld, scales, ssr, ssk}, Fp8Form{}, block_rows != 1);
  return launch_quantize(js, dtype, (hipStream_t)stream);
}

int sd_fp8_dequantize(const void* data, int64_t data_ld, const uint8_t* scales, int64_t ssr, int64_t ssk, int64_t block_rows, int64_t rows,
                      int64_t cols, void* out, int64_t out_ld, int dtype, void* stream) {
  if (int rc = check_sizes("fp8_dequantize", rows, cols)) return rc;
  SD_REQUIRE(dtype == SD_F16 || dtype == SD_BF16 || dtype == SD_F32, "fp8_dequantize: dtype must be SD_F16, SD_BF16 or SD_F32 (got %d)", dtype);
  SD_REQUIRE(block_rows == 1 || block_rows == kFp8Block, "fp8_dequantize: blocks are of 1 x 128 or 128 x 128 (got %lld rows)", (long long)block_rows);
  if (int rc = check_codes("fp8_dequantize", "data", data, data_ld, scales, rows, cols)) return rc;
  SD_REQUIRE(ssr >= 1 && ssk >= 1, "fp8_dequantize: scales: strides must be positive");
  SD_REQUIRE(out != nullptr || rows == 0 || cols == 0, "fp8_dequantize: null pointer");
  SD_REQUIRE(rows <= 1 || out_ld >= cols, "fp8_dequantize: row stride %lld < %lld columns", (long long)out_ld, (long long)cols);
  if (rows == 0 || cols == 0) return SD_OK;
  return launch_dequantize(static_cast<const uint8_t*>(data), data_ld, scales, ssr, ssk, block_rows != 1, rows, cols, out, out_ld, dtype, (hipStream_t)stream);
}

int64_t sd_fp8_gemm_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M < 0 || N < 0 || K < 0 || M >= kMaxDim || N >= kMaxDim || K >= kMaxDim) return -1;
  return fp8_gemm_scratch(M, N, K, kFp8Dense);
}

int sd_fp8_gemm(const void* A, int64_t lda, const uint8_t* SA, int64_t sa_ld, const void* B, int64_t ldb, const uint8_t* SB, int64_t sbr,
                int64_t sbk, int64_t b_block_rows, void* C, int64_t csr, int64_t csc, int64_t M, int64_t N, int64_t K, int dtype,
                void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check_sizes("fp8_gemm", M, N)) return rc;
  if (int rc = check_sizes("fp8_gemm", M, K)) return rc;
  if (int rc = check_dtype("fp8_gemm", dtype)) return rc;
  SD_REQUIRE(b_block_rows == 1 || b_block_rows == kFp8Block, "fp8_gemm: B's blocks are of 1 x 128 or 128 x 128 (got %lld rows)", (long long)b_block_rows);
  if (int rc = check_codes("fp8_gemm", "A", A, lda, SA, M, K)) return rc;
  if (int rc = check_codes("fp8_gemm", "B", B, ldb, SB, N, K)) return rc;
  if (int rc = check_pitch("fp8_gemm", lda > ldb ? lda : ldb)) return rc;
  if (int rc = check_matrix("fp8_gemm", "C", C, csr, csc, M, N)) return rc;
  if (M == 0 || N == 0) return SD_OK;
  SD_REQUIRE(K > 0, "fp8_gemm: empty reduction");
  auto rows_of_scales = [](const void* s, int64_t ld, int64_t rows) { return ld >= rows && ld % 4 == 0 && reinterpret_cast<uintptr_t>(s) % 4 == 0; };
  SD_REQUIRE(rows_of_scales(SA, sa_ld, M), "fp8_gemm: A's scales must start on 4 bytes, a multiple of 4 and at least %lld apart (got %lld)", (long long)M, (long long)sa_ld);
  if (b_block_rows == 1)
    SD_REQUIRE(sbr == 1 && rows_of_scales(SB, sbk, N), "fp8_gemm: B's scales must start on 4 bytes, a multiple of 4 and at least %lld apart (got %lld)", (long long)N, (long long)sbk);
  else
    SD_REQUIRE(sbr >= 1 && sbk >= 1, "fp8_gemm: B's scales: strides must be positive");
  const int64_t nk = ceil_div(K, kFp8Block);
  if (nk * sa_ld >= (1LL << 31) || nk * sbk >= (1LL << 31)) return fail(SD_ERR_UNSUPPORTED, "fp8_gemm: too many scales");
  if (b_block_rows != 1)
    if (int rc = check_square_scales("fp8_gemm", N, nk, sbr, sbk)) return rc;
  const bool ws_ok = workspace != nullptr && workspace_bytes > 0 && aligned16(workspace);
  Fp8Gemm g = {};
  g.a = static_cast<const uint8_t*>(A);
  g.lda = lda;
  g.sa = SA;
  g.sa_ld = sa_ld;
  g.b = static_cast<const uint8_t*>(B);
  g.ldb = ldb;
  g.sb = SB;
  g.sb_r = sbr;
  g.sb_k = sbk;
  g.sb_square = b_block_rows != 1 ? 1 : 0;
  g.c = static_cast<uint16_t*>(C);
  g.c_sr = csr;
  g.c_sc = csc;
  g.M = M;
  g.N = N;
  g.K = K;
  g.scale = 1.f;
  g.split = 1;
  g.keep = 1.f;
  g.part = ws_ok ? static_cast<float*>(workspace) : nullptr;
  g.part_bytes = ws_ok ? workspace_bytes : 0;
  return launch_fp8_gemm(g, kFp8Dense, dtype, (hipStream_t)stream);
}

int64_t sd_fp8_linear_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M < 0 || N < 0 || K < 0 || M >= kMaxDim || N >= kMaxDim || K >= kMaxDim) return -1;
  if (fp8_few_takes(M, N, K)) return 0;
  return Packed(M, K, false).bytes + fp8_gemm_scratch(M, N, K, kFp8Dense);
}

int sd_fp8_linear(const void* X, int64_t ldx, const void* W, int64_t ldw, const uint8_t* SW, int64_t swr, int64_t swk, void* Y, int64_t ldy,
                  int64_t M, int64_t N, int64_t K, int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check_sizes("fp8_linear", M, N)) return rc;
  if (int rc = check_sizes("fp8_linear", M, K)) return rc;
  if (int rc = check_dtype("fp8_linear", dtype)) return rc;
  if (int rc = check_matrix("fp8_linear", "X", X, ldx, 1, M, K)) return rc;
  if (int rc = check_codes("fp8_linear", "W", W, ldw, SW, N, K)) return rc;
  if (int rc = check_pitch("fp8_linear", ldw)) return rc;
  if (int rc = check_matrix("fp8_linear", "Y", Y, ldy, 1, M, N)) return rc;
  if (M == 0 || N == 0) return SD_OK;
  SD_REQUIRE(K > 0, "fp8_linear: empty reduction");
  SD_REQUIRE(swr >= 1 && swk >= 1, "fp8_linear: scales: strides must be positive");
  if (int rc = check_reach("fp8_linear", M, K)) return rc;
  if (ceil_div(K, kFp8Block) * swk >= (1LL << 31)) return fail(SD_ERR_UNSUPPORTED, "fp8_linear: too many scales");
  if (fp8_few_takes(M, N, K)) {
    const Fp8Few f = {static_cast<const uint16_t*>(X), ldx, static_cast<const uint8_t*>(W), ldw, SW, swr, swk, static_cast<uint16_t*>(Y), ldy,
                      (int32_t)M, (int32_t)N, (int32_t)K};
    return launch_fp8_few(f, dtype, (hipStream_t)stream);
  }
  if (int rc = check_square_scales("fp8_linear", N, ceil_div(K, kFp8Block), swr, swk)) return rc;
  if (int rc = check_workspace("fp8_linear", workspace, workspace_bytes, sd_fp8_linear_workspace_bytes(M, N, K))) return rc;
  const Packed x(M, K, false);
  QuantJobs js = {};
  js.n = 1;
  js.job[0] = quant_job(X, ldx, 1, M, K, x.form(workspace), Fp8Form{}, false);
  if (int rc = launch_quantize(js, dtype, (hipStream_t)stream)) return rc;
  Fp8Gemm g = product(x, workspace, x, workspace, Y, ldy, 1, M, N, K, 1.f, static_cast<uint8_t*>(workspace) + x.bytes, workspace_bytes - x.bytes);
  g.b = static_cast<const uint8_t*>(W);
  g.ldb = ldw;
  g.sb = SW;
  g.sb_r = swr;
  g.sb_k = swk;
  g.sb_square = 1;
  return launch_fp8_gemm(g, kFp8Dense, dtype, (hipStream_t)stream);
}

int64_t sd_fp8_dropout_matmul_workspace_bytes(int64_t M, int64_t N, int64_t K, int backward) {
  if (M < 0 || N < 0 || K < 0 || M >= kMaxDim || N >= kMaxDim || K >= kMaxDim) return -1;
  if (!backward) return Packed(M, K, false).bytes + Packed(N, K, true).bytes + fp8_gemm_scratch(M, N, K, kFp8Dsd);
  return Packed(M, N, false).bytes + Packed(N, M, false).bytes + fp8_gemm_scratch(K, N, M, kFp8Dsd);
}

static int check_dropout(const char* fn, int64_t M, int64_t N, int64_t K, int64_t bs, double p, int dtype) {
  if (int rc = check_sizes(fn, M, N)) return rc;
  if (int rc = check_sizes(fn, M, K)) return rc;
  if (int rc = check_dtype(fn, dtype)) return rc;
  SD_REQUIRE(p >= 0.0 && p < 1.0, "%s: p must be in [0, 1) (got %g)", fn, p);
  SD_REQUIRE(bs > 0, "%s: block_size must be positive", fn);
  if (bs % kFp8Block) return fail(SD_ERR_UNSUPPORTED, "%s: block_size %lld: products in 8 bits take multiples of 128", fn, (long long)bs);
  SD_REQUIRE(M > 0 && K > 0, "%s: empty operand", fn);
  if (int rc = check_reach(fn, M, K)) return rc;
  if (int rc = check_reach(fn, M, N)) return rc;
  if (int rc = check_reach(fn, K, M)) return rc;
  return check_reach(fn, N, M);
}

int sd_fp8_dropout_matmul_forward(const void* X, int64_t xsr, int64_t xsc, const void* W, int64_t wsr, int64_t wsc, void* Y, int64_t ysr,
                                  int64_t ysc, const uint8_t* mask, int64_t msr, int64_t msc, uint64_t* rng_state, uint64_t seed,
                                  uint64_t offset, double p, uint8_t* mask_out, void* XT, void* WT, int64_t M, int64_t N, int64_t K,
                                  int64_t bs, int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* fn = "fp8_dropout_matmul_forward";
  if (int rc = check_dropout(fn, M, N, K, bs, p, dtype)) return rc;
  if (int rc = check_matrix(fn, "X", X, xsr, xsc, M, K)) return rc;
  if (int rc = check_matrix(fn, "W", W, wsr, wsc, N, K)) return rc;
  if (int rc = check_matrix(fn, "Y", Y, ysr, ysc, M, N)) return rc;
  SD_REQUIRE(aligned16(XT) && aligned16(WT), "%s: XT and WT must start on 16 bytes", fn);
  if (mask) {
    SD_REQUIRE(msr >= 1 && msc >= 1 && (msr == 1 || msc == 1), "%s: mask must be row or column major", fn);
  } else {
    SD_REQUIRE((float)p < 1.f, "%s: p must be in [0, 1) in 32 bits to draw a mask (got %.17g)", fn, p);
    SD_REQUIRE(mask_out != nullptr, "%s: null mask_out", fn);
    SD_REQUIRE(rng_state == nullptr || reinterpret_cast<uintptr_t>(rng_state) % 8 == 0, "%s: state must be an aligned device pointer", fn);
  }
  if (int rc = check_workspace(fn, workspace, workspace_bytes, sd_fp8_dropout_matmul_workspace_bytes(M, N, K, 0))) return rc;
  const Packed x(M, K, false), w(N, K, true), xt(K, M, false), wt(K, N, true);
  uint8_t *const xs = static_cast<uint8_t*>(workspace), *const wq = xs + x.bytes, *const part = wq + w.bytes;
  QuantJobs js = {};
  js.n = 2;
  js.job[0] = quant_job(X, xsr, xsc, M, K, x.form(xs), xt.form(XT), false);
  js.job[0].masked = 1;
  js.job[1] = quant_job(W, wsr, wsc, N, K, w.form(wq), wt.form(WT), true);
  const int64_t mb = ceil_div(M, bs), kb = ceil_div(K, bs);
  js.mask = MaskSrc{mask, msr, msc, (int32_t)(bs / kFp8Block), 1, (int32_t)mb, (int32_t)kb, (uint32_t)seed, (uint32_t)(seed >> 32),
                    (uint32_t)offset, (uint32_t)(offset >> 32), (float)p, mask ? nullptr : rng_state};
  js.mask_out = mask ? nullptr : mask_out;
  if (int rc = launch_quantize(js, dtype, (hipStream_t)stream)) return rc;
  Fp8Gemm g = product(x, xs, w, wq, Y, ysr, ysc, M, N, K, (float)(1.0 / (1.0 - p)), part, fp8_gemm_scratch(M, N, K, kFp8Dsd));
  g.mask = mask ? mask : mask_out;
  g.msr = mask ? msr : kb;
  g.msc = mask ? msc : 1;
  g.split = (int32_t)(bs / kFp8Block);
  return launch_fp8_gemm(g, kFp8Dsd, dtype, (hipStream_t)stream);
}

int sd_fp8_dropout_matmul_backward(const void* dY, int64_t dysr, int64_t dysc, const uint8_t* mask, int64_t msr, int64_t msc, void* XT,
                                   void* WT, void* dX, int64_t dxsr, int64_t dxsc, void* dW, int64_t dwsr, int64_t dwsc, int64_t M,
                                   int64_t N, int64_t K, int64_t bs, double p, int dtype, void* workspace, int64_t workspace_bytes,
                                   void* stream) {
  const char* fn = "fp8_dropout_matmul_backward";
  if (int rc = check_dropout(fn, M, N, K, bs, p, dtype)) return rc;
  SD_REQUIRE(N > 0, "%s: no outputs", fn);
  SD_REQUIRE(dX != nullptr || dW != nullptr, "%s: neither gradient is asked for", fn);
  SD_REQUIRE(mask != nullptr && msr >= 1 && msc >= 1, "%s: the mask is required", fn);
  if (int rc = check_matrix(fn, "dY", dY, dysr, dysc, M, N)) return rc;
  if (dX) {
    if (int rc = check_matrix(fn, "dX", dX, dxsr, dxsc, M, K)) return rc;
    SD_REQUIRE(WT != nullptr && aligned16(WT), "%s: dX needs WT, on 16 bytes", fn);
  }
  if (dW) {
    if (int rc = check_matrix(fn, "dW", dW, dwsr, dwsc, N, K)) return rc;
    SD_REQUIRE(XT != nullptr && aligned16(XT), "%s: dW needs XT, on 16 bytes", fn);
  }
  if (int rc = check_workspace(fn, workspace, workspace_bytes, sd_fp8_dropout_matmul_workspace_bytes(M, N, K, 1))) return rc;
  const Packed dy(M, N, false), dyt(N, M, false), xt(K, M, false), wt(K, N, true);
  uint8_t *const dyq = static_cast<uint8_t*>(workspace), *const dytq = dyq + dy.bytes, *const part = dytq + dyt.bytes;
  QuantJobs js = {};
  js.n = 1;
  js.job[0] = quant_job(dY, dysr, dysc, M, N, dX ? dy.form(dyq) : Fp8Form{}, dW ? dyt.form(dytq) : Fp8Form{}, false);
  if (int rc = launch_quantize(js, dtype, (hipStream_t)stream)) return rc;
  const float scale = (float)(1.0 / (1.0 - p));
  // dX[m, k] = sum over n of dY[m, n] W[n, k], kept blocks
  Fp8Gemm gx = product(dy, dyq, wt, WT, dX, dxsr, dxsc, M, K, N, scale, nullptr, 0);
  gx.mask = mask;
  gx.msr = msr;
  gx.msc = msc;
  // dW^T[k, n] = sum over m of X[m, k] dY[m, n], kept blocks of X
  Fp8Gemm gw = product(xt, XT, dyt, dytq, dW, dwsc, dwsr, K, N, M, scale, part, fp8_gemm_scratch(K, N, M, kFp8Dsd));
  gw.mask = mask;
  gw.msr = msc;
  gw.msc = msr;
  gx.split = gw.split = (int32_t)(bs / kFp8Block);
  gx.keep = gw.keep = (float)(1.0 - p);
  if (dX && dW) return launch_fp8_backward(gx, gw, dtype, (hipStream_t)stream);
  return dX ? launch_fp8_gemm(gx, kFp8Sdd, dtype, (hipStream_t)stream) : launch_fp8_gemm(gw, kFp8Dsd, dtype, (hipStream_t)stream);
}

int sd_adamw_step_scaled(int count, void* const* params, const void* const* grads, void* const* exp_avgs, void* const* exp_avg_sqs,
                         uint8_t* const* exp_avg_scales, uint8_t* const* exp_avg_sq_scales, const int64_t* numels, int64_t* step,
                         const float* lr_at, double lr, double beta1, double beta2, double eps, double weight_decay, int dtype, int state_bits,
                         int advance, const float* grad_scale, void* stream) {
  SD_REQUIRE(count >= 0, "adamw_step: negative count");
  SD_REQUIRE(dtype == SD_F16 || dtype == SD_BF16 || dtype == SD_F32, "adamw_step: dtype must be SD_F16, SD_BF16 or SD_F32 (got %d)", dtype);
  SD_REQUIRE(state_bits == 8 || state_bits == 32, "adamw_step: averages are held in 8 or in 32 bits (got %d)", state_bits);
  SD_REQUIRE(step != nullptr && reinterpret_cast<uintptr_t>(step) % 8 == 0, "adamw_step: step must be an aligned device pointer");
  SD_REQUIRE(lr_at != nullptr || (lr >= 0.0 && lr <= DBL_MAX), "adamw_step: lr must not be negative (got %g)", lr);
  SD_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "adamw_step: betas must be in [0, 1) (got %g, %g)", beta1, beta2);
  SD_REQUIRE(eps == 0.0 || (eps >= 0x1p-126 && eps <= 0x1p120), "adamw_step: eps must be 0 or from 2^-126 to 2^120 (got %g)", eps);
  SD_REQUIRE(weight_decay >= 0.0, "adamw_step: weight_decay must not be negative (got %g)", weight_decay);
  SD_REQUIRE(count == 0 || (params && grads && exp_avgs && exp_avg_sqs && numels), "adamw_step: null array");
  for (int i = 0; i < count; ++i) {
    SD_REQUIRE(numels[i] >= 0, "adamw_step: tensor %d: negative size", i);
    if (numels[i] == 0) continue;
    SD_REQUIRE(params[i] && grads[i] && exp_avgs[i] && exp_avg_sqs[i], "adamw_step: tensor %d: null pointer", i);
    SD_REQUIRE(state_bits == 32 || (exp_avg_scales && exp_avg_sq_scales && exp_avg_scales[i] && exp_avg_sq_scales[i]), "adamw_step: tensor %d: averages in 8 bits need their scales", i);
  }
  return launch_adamw(count, params, grads, exp_avgs, exp_avg_sqs, state_bits == 8 ? exp_avg_scales : nullptr, state_bits == 8 ? exp_avg_sq_scales : nullptr,
                      numels, step, lr_at, lr, beta1, beta2, eps, weight_decay, dtype, state_bits, advance != 0, grad_scale, (hipStream_t)stream);
}

int sd_adamw_step(int count, void* const* params, const void* const* grads, void* const* exp_avgs, void* const* exp_avg_sqs,
                  uint8_t* const* exp_avg_scales, uint8_t* const* exp_avg_sq_scales, const int64_t* numels, int64_t* step,
                  const float* lr_at, double lr, double beta1, double beta2, double eps, double weight_decay, int dtype, int state_bits,
                  int advance, void* stream) {
  return sd_adamw_step_scaled(count, params, grads, exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales, numels, step, lr_at, lr, beta1, beta2,
                              eps, weight_decay, dtype, state_bits, advance, nullptr, stream);
}

int sd_adamw_state_values(int count, const uint8_t* const* codes, const uint8_t* const* scales, float* const* values, const int64_t* numels,
                          const int32_t* second, void* stream) {
  SD_REQUIRE(count >= 0, "adamw_state_values: negative count");
  SD_REQUIRE(count == 0 || (codes && scales && values && numels && second), "adamw_state_values: null array");
  for (int i = 0; i < count; ++i) {
    SD_REQUIRE(numels[i] >= 0, "adamw_state_values: tensor %d: negative size", i);
    SD_REQUIRE(numels[i] == 0 || (codes[i] && scales[i] && values[i]), "adamw_state_values: tensor %d: null pointer", i);
  }
  return launch_state_values(count, codes, scales, values, numels, second, (hipStream_t)stream);
}

}  // extern "C"
