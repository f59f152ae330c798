// y = x . W^T for at most 16 rows of x in 16 bits and weights in 8 bits (fp8.h): the product of serving a few tokens.
//
// Bound by reading the weights, a byte each: nothing else is as large.  So they go from memory straight into the matrix instruction's
// registers, every byte once, and x, which a launch before would have to bring into 8 bits, is quantized by each workgroup as it reads
// it (16 rows of x are a few KB out of the L2 for every 128 columns, and the arithmetic hides behind the loads).  A workgroup owns 16
// outputs and its waves share out the 128-blocks of the reduction, wave w every 128-block w + waves * n, and meet once in LDS.
#include "fp8.h"

namespace sd {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

template <typename T, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void fp8_few_kernel(Fp8Few g) {
  __shared__ float sums[WAVES][16][17];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, r = lane & 15, q = lane >> 4;
  const int n0 = (int)blockIdx.x * 16, nk = (g.K + kFp8Block - 1) / kFp8Block;
  const bool has_w = n0 + r < g.N, has_x = r < g.M;
  const uint8_t* const w = g.w + (int64_t)(has_w ? n0 + r : 0) * g.ldw;
  const uint16_t* const x = g.x + (int64_t)(has_x ? r : 0) * g.ldx;
  const uint8_t* const sw = g.sw + (int64_t)(n0 / kFp8Block) * g.sw_r;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
  for (int k = wave; k < nk; k += WAVES) {
    u32x4 wl = {0u, 0u, 0u, 0u}, wh = wl;
    if (has_w) {
      wl = *reinterpret_cast<const u32x4*>(w + (int64_t)k * kFp8Block + 16 * q);
      wh = *reinterpret_cast<const u32x4*>(w + (int64_t)k * kFp8Block + 64 + 16 * q);
    }
    const int ws = sw[(int64_t)k * g.sw_k];
    // this lane's 32 elements of row r, two to a word: 16 q .. + 15 and 64 + 16 q .. + 15 of the block
    uint32_t v[16], size[16], most = 0u;
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const int c = k * kFp8Block + (h >> 1) * 64 + 16 * q + (h & 1) * 8, left = has_x ? g.K - c : 0;
      if (left >= 8) {
        const u32x4 e = *reinterpret_cast<const u32x4_any*>(x + c);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[4 * h + i] = e[i];
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          v[4 * h + i] = (2 * i < left ? x[c + 2 * i] : 0u) | (2 * i + 1 < left ? (uint32_t)x[c + 2 * i + 1] << 16 : 0u);
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      size[i] = v[i] & 0x7fff7fffu;
      most = pk_max(most, size[i]);
    }
    most = max(most & 0xffffu, most >> 16);
    if (most >= kInfinite<T>) {
      most = 0u;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t lo = size[i] & 0xffffu, hi = size[i] >> 16;
        most = max(most, max(lo < kInfinite<T> ? lo : 0u, hi < kInfinite<T> ? hi : 0u));
      }
    }
    most = max(most, (uint32_t)__shfl_xor((int)most, 16));
    most = max(most, (uint32_t)__shfl_xor((int)most, 32));
    const uint32_t xs = fp8_scale_of(size_bits<T>(most));
    i32x8 a, b;
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = (int)codes_of<T, true>(codes_of<T, false>(0u, v[2 * i], xs), v[2 * i + 1], xs);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      b[i] = (int)wl[i];
      b[4 + i] = (int)wh[i];
    }
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 0, 0, 0, (int)xs, 0, ws);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) sums[wave][4 * q + i][r] = acc[i];
  __syncthreads();
  if (t < 256) {
    const int m = t >> 4, n = t & 15;
    if (m < g.M && n0 + n < g.N) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < WAVES; ++i) sum += sums[i][m][n];
      g.y[(int64_t)m * g.ldy + n0 + n] = T::from_float(sum);
    }
  }
}

}  // namespace

int launch_fp8_few(const Fp8Few& g, int dtype, hipStream_t stream) {
  if (g.M == 0 || g.N == 0) return SD_OK;
  const int nk = (int)ceil_div(g.K, kFp8Block);
  const bool wide = nk > 16;
  auto* kernel = dtype == SD_BF16 ? (wide ? &fp8_few_kernel<BF16, 16> : &fp8_few_kernel<BF16, 4>)
                                  : (wide ? &fp8_few_kernel<F16, 16> : &fp8_few_kernel<F16, 4>);
  hipLaunchKernelGGL(kernel, dim3((unsigned)ceil_div(g.N, 16)), dim3(wide ? 1024 : 256), 0, stream, g);
  note_kernel("fp8:few waves=%d", wide ? 16 : 4);
  return check_launch("fp8_few");
}

}  // namespace sd
