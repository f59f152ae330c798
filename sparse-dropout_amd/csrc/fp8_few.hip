// y = x . W^T for few rows of x in 16 bits and weights in 8 bits (fp8.h): the product of serving a few tokens.
//
// Bound by reading the weights, a byte each, as long as there are few rows.  So they go from memory straight into the matrix
// instruction's registers, every byte once, and x, which a launch before would have to bring into 8 bits, is quantized by each workgroup as
// it reads it out of the L2.  A workgroup owns 16 or 32 outputs and its waves share out the 128-blocks of the reduction, wave w every 128-block
// w + waves * n, a few of them on their way at a time, and meet once in LDS.  Rows come in groups of 16, up to four; what a row behind the
// last or an output behind the last holds is never stored, so their lanes read another's.  One token through 4096 to 1024 5.7 us, most of it a
// memory latency and the launch; through 8192 to 8192 18.3, 3.7 TB/s.
#include "fp8.h"

namespace sd {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

// This lane's 32 elements of a row in one 128-block, two to a word: 32 q .. + 31.  (Each load of a wave touches whole lines then.)
struct RowPart {
  uint32_t v[16];
  __device__ inline void load(const uint16_t* at) {  // the block's first element plus 32 q
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const u32x4 e = *reinterpret_cast<const u32x4_any*>(at + 8 * h);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[4 * h + i] = e[i];
    }
  }
  __device__ inline void load_some(const uint16_t* at, int left) {  // of the block, `left` elements behind `at` are there
#pragma unroll
    for (int h = 0; h < 4; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = 8 * h + 2 * i;
        v[4 * h + i] = (c < left ? at[c] : 0u) | (c + 1 < left ? (uint32_t)at[c + 1] << 16 : 0u);
      }
  }
  // as codes, with the scale's byte
  template <typename T>
  __device__ inline i32x8 codes(int& byte) const {
    uint32_t most = 0u;
#pragma unroll
    for (int i = 0; i < 16; ++i) most = pk_max(most, v[i] & 0x7fff7fffu);
    most = max(most & 0xffffu, most >> 16);
    if (most >= kInfinite<T>) {
      most = 0u;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t lo = v[i] & 0x7fffu, hi = v[i] >> 16 & 0x7fffu;
        most = max(most, max(lo < kInfinite<T> ? lo : 0u, hi < kInfinite<T> ? hi : 0u));
      }
    }
    most = max(most, (uint32_t)__shfl_xor((int)most, 16));
    most = max(most, (uint32_t)__shfl_xor((int)most, 32));
    const uint32_t s = fp8_scale_of(size_bits<T>(most));
    byte = (int)s;
    i32x8 a;
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = (int)codes_of<T, true>(codes_of<T, false>(0u, v[2 * i], s), v[2 * i + 1], s);
    return a;
  }
};

__device__ inline i32x8 load_weights(const uint8_t* at) {  // the block's first code plus 32 q
  const u32x4 lo = *reinterpret_cast<const u32x4*>(at), hi = *reinterpret_cast<const u32x4*>(at + 16);
  i32x8 b;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    b[i] = (int)lo[i];
    b[4 + i] = (int)hi[i];
  }
  return b;
}

// COLS: of 16 outputs; AHEAD: 128-blocks of a wave on their way together
template <typename T, int WAVES, int GROUPS, int COLS, int AHEAD>
__global__ __launch_bounds__(WAVES * 64, WAVES / 4) void fp8_few_kernel(Fp8Few g) {
  __shared__ float sums[WAVES][16][17];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), r = lane & 15, q = lane >> 4;
  const int n0 = (int)blockIdx.x * 16 * COLS, whole = g.K / kFp8Block, left = g.K - whole * kFp8Block;
  const uint8_t* w[COLS];
#pragma unroll
  for (int j = 0; j < COLS; ++j) w[j] = g.w + (int64_t)min(n0 + 16 * j + r, g.N - 1) * g.ldw + 32 * q;
  const uint8_t* const sw = g.sw + (int64_t)(n0 / kFp8Block) * g.sw_r;
  const uint16_t* x[GROUPS];
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) x[i] = g.x + (int64_t)min(16 * i + r, g.M - 1) * g.ldx + 32 * q;
  f32x4 acc[GROUPS][COLS] = {};
  auto multiply = [&](const RowPart (&p)[GROUPS], const i32x8 (&b)[COLS], int ws) {
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) {
      int xs;
      const i32x8 a = p[i].template codes<T>(xs);
#pragma unroll
      for (int j = 0; j < COLS; ++j) acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b[j], acc[i][j], 0, 0, 0, xs, 0, ws);
    }
  };
  for (int k0 = wave; k0 < whole; k0 += WAVES * AHEAD) {
    RowPart p[AHEAD][GROUPS];
    i32x8 b[AHEAD][COLS];
    int ws[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int64_t k = k0 + u * WAVES;
      if (k < whole) {
#pragma unroll
        for (int j = 0; j < COLS; ++j) b[u][j] = load_weights(w[j] + k * kFp8Block);
        ws[u] = sw[k * g.sw_k];
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) p[u][i].load(x[i] + k * kFp8Block);
      }
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (k0 + u * WAVES < whole) multiply(p[u], b[u], ws[u]);
  }
  if (left && wave == whole % WAVES) {
    RowPart p[GROUPS];
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) p[i].load_some(x[i] + (int64_t)whole * kFp8Block, left - 32 * q);
    i32x8 b[COLS];
#pragma unroll
    for (int j = 0; j < COLS; ++j) b[j] = load_weights(w[j] + (int64_t)whole * kFp8Block);
    multiply(p, b, sw[(int64_t)whole * g.sw_k]);
  }
#pragma unroll
  for (int i = 0; i < GROUPS; ++i)
#pragma unroll
    for (int j = 0; j < COLS; ++j) {
      if (i || j) __syncthreads();
#pragma unroll
      for (int e = 0; e < 4; ++e) sums[wave][4 * q + e][r] = acc[i][j][e];
      __syncthreads();
      if (t < 256) {
        const int row = t >> 4, n = n0 + 16 * j + (t & 15), m = 16 * i + row;
        if (m < g.M && n < g.N) {
          float sum = 0.f;
#pragma unroll
          for (int o = 0; o < WAVES; ++o) sum += sums[o][row][t & 15];
          g.y[(int64_t)m * g.ldy + n] = T::from_float(sum);
        }
      }
    }
}

struct FewPlan {
  int groups;  // of 16 rows
  bool wide;   // sixteen waves instead of four
  bool many;   // more workgroups than CUs: of 32 outputs each, x is read and quantized half as often
  double us;
};
// Sixteen waves a workgroup where the reduction is long (one row, sixteen and four: 4096 to 4096 6.0 and 8.4 us, 4096 to 1024 5.6 and 6.8; 1500 to 10000
// 10.3 and 7.5).  The time, from 7 layers between 512^2 and 8192^2 at 1 to 64 rows: 5 us, and for each 128-block of a wave and group of rows 2.1
// with sixteen waves (32 rows through 4096^2 12.1 us, 64 19.9), 1 with four (64 rows of 2048 to 8192 19.8).  It leaves out what 32 outputs a
// workgroup save (2048 to 8192: 32 rows 9.1 us).  More workgroups than CUs: 32 outputs each instead of 16 (16 rows of 2048 to 8192 6.8 us and 8.5, of
// 8192 to 8192 19.9 and 26.0, of 1000 to 5000 5.5 and 6.1; one row of 8192 to 8192 18.3 and 17.1); with a workgroup or less a CU they would
// leave CUs idle (16 rows of 4096 to 4096 10.1 and 8.3).
FewPlan few_plan(int64_t M, int64_t N, int64_t K) {
  FewPlan p;
  const int64_t nk = ceil_div(K, kFp8Block), wgs = ceil_div(N, 16);
  p.groups = M <= 16 ? 1 : M <= 32 ? 2 : 4;
  p.wide = nk > 16;
  p.many = wgs > 256;
  const int waves = p.wide ? 16 : 4;
  const double rounds = (double)(wgs * waves) / 4096.0;
  p.us = 5.0 + (p.wide ? 2.1 : 1.0) * p.groups * (double)ceil_div(nk, waves) * (rounds > 1.0 ? rounds : 1.0);
  return p;
}

template <typename T>
void launch_few(const Fp8Few& g, const FewPlan& p, hipStream_t stream) {
  const bool two = p.many && (p.groups == 1 || (p.groups == 2 && !p.wide));
  const dim3 grid((unsigned)ceil_div(g.N, two ? 32 : 16)), block(p.wide ? 1024 : 256);
  if (p.groups == 1) {
    auto* kernel = !p.wide ? p.many ? &fp8_few_kernel<T, 4, 1, 2, 2> : &fp8_few_kernel<T, 4, 1, 1, 4> : p.many ? &fp8_few_kernel<T, 16, 1, 2, 2> : &fp8_few_kernel<T, 16, 1, 1, 2>;
    hipLaunchKernelGGL(kernel, grid, block, 0, stream, g);
  } else if (p.groups == 2) {
    auto* kernel = p.wide ? &fp8_few_kernel<T, 16, 2, 1, 2> : p.many ? &fp8_few_kernel<T, 4, 2, 2, 2> : &fp8_few_kernel<T, 4, 2, 1, 2>;
    hipLaunchKernelGGL(kernel, grid, block, 0, stream, g);
  } else {  // (a long reduction of that many rows goes through the tiles)
    hipLaunchKernelGGL((&fp8_few_kernel<T, 4, 4, 1, 1>), grid, dim3(256), 0, stream, g);
  }
}

}  // namespace

// Whether the kernel takes the product: up to 16 rows always; up to 64 where it is expected to take less than quantizing x and 128 x 128
// tiles do, 10 to 18 us at such sizes.  us here and on the tiles, features to outputs at 17, 32, 33 and 64 rows:
//   1024 to 4096  5.5, 12.6   5.8, 12.6    7.4, 12.6   8.2, 11.8     2048 to 8192  8.3, 15.1   9.1, 15.8   15.5, 15.7   19.8, 16.4
//   4096 to 1024  9.5, 15.2  12.0, 16.1   18.2, 15.9  19.7, 14.8     8192 to 2048  17.0, 17.2  22.1, 18.4  32.7, 18.0   35.2, 18.4
//   1000 to 5000  7.5, 12.8   8.2, 12.8   13.5, 12.8  14.8, 12.4 (the one here that the rule gets wrong, from 33 rows on)
bool fp8_few_takes(int64_t M, int64_t N, int64_t K) { return M <= 16 || (M <= kFp8FewRows && few_plan(M, N, K).us <= 15.0); }

int launch_fp8_few(const Fp8Few& g, int dtype, hipStream_t stream) {
  if (g.M == 0 || g.N == 0) return SD_OK;
  const FewPlan p = few_plan(g.M, g.N, g.K);
  if (dtype == SD_BF16) launch_few<BF16>(g, p, stream);
  else launch_few<F16>(g, p, stream);
  note_kernel("fp8:few waves=%d groups=%d", p.wide ? 16 : 4, p.groups);
  return check_launch("fp8_few");
}

}  // namespace sd
