// Matrices in 16 or 32 bits -> e4m3 codes with a power of two for each block of 1 x 128 or 128 x 128 (fp8.h), and back.
//
// A training step needs its activations and output gradients twice: with blocks along their rows for the products that sum over
// features, and with blocks along their columns, transposed, for the weight gradient, which sums over tokens.  Both come out of one
// read: a workgroup holds a 128 x 128 tile in registers, 8 x 8 elements a thread, takes the largest magnitude along both directions
// and writes the codes both ways.  Bound by its reads and writes: 2 bytes in and 1 or 2 out per element.
#include "fp8.h"

#include <type_traits>

namespace sd {
namespace {

constexpr int kThreads = 256;

struct F32 {
  static constexpr int id = kF32;
};

// eight consecutive elements, zeros where `left` ends
template <typename T>
__device__ inline void load_eight(const void* src, int64_t at, int left, float (&v)[8]) {
  if constexpr (T::id == kF32) {
    typedef f32x4 __attribute__((aligned(4))) f32x4_any;
    const float* s = static_cast<const float*>(src) + at;
    if (left >= 8) {
      const f32x4 a = *reinterpret_cast<const f32x4_any*>(s), b = *reinterpret_cast<const f32x4_any*>(s + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = a[i];
        v[4 + i] = b[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i < left ? s[i] : 0.f;
    }
  } else {
    const uint16_t* s = static_cast<const uint16_t*>(src) + at;
    if (left >= 8) {
      const u32x4 w = *reinterpret_cast<const u32x4_any*>(s);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = T::to_float((uint16_t)(i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i < left ? T::to_float(s[i]) : 0.f;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void quantize_kernel(QuantJobs js) {
  __shared__ uint32_t most_of[4][kFp8Block];  // [wave][column], or [wave][0] of a square block
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int which = js.n > 1 && blockIdx.x >= js.job[1].first_block ? 1 : 0;
  const QuantJob& p = js.job[which];
  const uint32_t tile = blockIdx.x - p.first_block;
  const int tr = (int)(tile / p.tiles_c), tc = (int)(tile - (uint32_t)tr * p.tiles_c);
  bool dropped = false;
  if (p.masked) {
    MaskSrc src = js.mask;
    src.resolve();
    const int i = p.mask_t ? tc : tr, j = p.mask_t ? tr : tc, si = i / src.split, sj = j / src.split;
    dropped = src.dropped_entry(si, sj);
    if (js.mask_out && t == 0 && si * src.split == i && sj * src.split == j) js.mask_out[(int64_t)si * src.kb + sj] = dropped ? 1 : 0;
  }
  if (!dropped) {  // (uniform)
    const int r0 = tr * kFp8Block + (t >> 4) * 8, c0 = tc * kFp8Block + (t & 15) * 8;
    float v[8][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int left = r0 + i < p.rows ? p.cols - c0 : 0;
      load_eight<T>(p.src, (int64_t)(r0 + i) * p.ld + c0, left, v[i]);
    }
    uint32_t row_most[8], col_most[8] = {};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      row_most[i] = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t a = finite_magnitude(v[i][j]);
        row_most[i] = max(row_most[i], a);
        col_most[j] = max(col_most[j], a);
      }
    }
    uint32_t row_scale[8], col_scale[8];
    if (p.square) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, row_most[i]);
#pragma unroll
      for (int d = 1; d < 64; d *= 2) m = max(m, (uint32_t)__shfl_xor((int)m, d));
      if (lane == 0) most_of[wave][0] = m;
      __syncthreads();
      m = max(max(most_of[0][0], most_of[1][0]), max(most_of[2][0], most_of[3][0]));
      const uint32_t s = fp8_scale_of(m);
#pragma unroll
      for (int i = 0; i < 8; ++i) row_scale[i] = col_scale[i] = s;
    } else {
      if (p.along.data) {
#pragma unroll
        for (int i = 0; i < 8; ++i) row_scale[i] = fp8_scale_of(max_of_row16(row_most[i]));
      }
      if (p.across.data) {  // (uniform)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint32_t m = col_most[j];
          m = max(m, (uint32_t)__shfl_xor((int)m, 16));
          m = max(m, (uint32_t)__shfl_xor((int)m, 32));
          if (lane < 16) most_of[wave][(t & 15) * 8 + j] = m;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int c = (t & 15) * 8 + j;
          col_scale[j] = fp8_scale_of(max(max(most_of[0][c], most_of[1][c]), max(most_of[2][c], most_of[3][c])));
        }
      }
    }
    if (p.along.data) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (r0 + i >= p.rows) continue;
        const float s = fp8_inverse(row_scale[i]);
        const u32x2 q = {pack_fp8(v[i][0] * s, v[i][1] * s, v[i][2] * s, v[i][3] * s),
                         pack_fp8(v[i][4] * s, v[i][5] * s, v[i][6] * s, v[i][7] * s)};
        *reinterpret_cast<u32x2*>(p.along.data + (int64_t)(r0 + i) * p.along.ld + c0) = q;
        if ((t & 15) == 0 && !p.square) p.along.scales[(int64_t)(r0 + i) * p.along.s_r + (int64_t)tc * p.along.s_k] = (uint8_t)row_scale[i];
      }
      if (p.square && t == 0) p.along.scales[(int64_t)tr * p.along.s_r + (int64_t)tc * p.along.s_k] = (uint8_t)row_scale[0];
    }
    if (p.across.data) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (c0 + j >= p.cols) continue;
        const float s = fp8_inverse(col_scale[j]);
        const u32x2 q = {pack_fp8(v[0][j] * s, v[1][j] * s, v[2][j] * s, v[3][j] * s),
                         pack_fp8(v[4][j] * s, v[5][j] * s, v[6][j] * s, v[7][j] * s)};
        *reinterpret_cast<u32x2*>(p.across.data + (int64_t)(c0 + j) * p.across.ld + r0) = q;
        if (t < 16 && !p.square) p.across.scales[(int64_t)(c0 + j) * p.across.s_r + (int64_t)tr * p.across.s_k] = (uint8_t)col_scale[j];
      }
      if (p.square && t == 0) p.across.scales[(int64_t)tc * p.across.s_r + (int64_t)tr * p.across.s_k] = (uint8_t)col_scale[0];
    }
  }
  report_in(const_cast<uint64_t*>(js.mask.state), gridDim.x);
}

// codes and scales -> values, four to a thread.  Bound by what it writes.
template <typename T>
__global__ __launch_bounds__(kThreads) void dequantize_kernel(const uint8_t* data, int64_t ld, const uint8_t* scales, int64_t s_r, int64_t s_k,
                                                              int square, int64_t rows, int64_t cols, uint32_t quads, void* out, int64_t out_ld) {
  const int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x, r = at / quads, c = (at - r * quads) * 4;
  if (r >= rows) return;
  const uint32_t q = *reinterpret_cast<const uint32_t*>(data + r * ld + c);
  const float s = fp8_power(scales[(square ? r / kFp8Block : r) * s_r + c / kFp8Block * s_k]);
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)q, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)q, true);
  const float v[4] = {lo[0] * s, lo[1] * s, hi[0] * s, hi[1] * s};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (c + i >= cols) break;
    if constexpr (T::id == kF32) static_cast<float*>(out)[r * out_ld + c + i] = v[i];
    else static_cast<uint16_t*>(out)[r * out_ld + c + i] = T::from_float(v[i]);
  }
}

}  // namespace

int launch_quantize(QuantJobs& js, int dtype, hipStream_t stream) {
  js.blocks = 0;
  for (int i = 0; i < js.n; ++i) {
    QuantJob& p = js.job[i];
    p.tiles_c = (uint32_t)ceil_div(p.cols, kFp8Block);
    p.first_block = js.blocks;
    js.blocks += (uint32_t)(ceil_div(p.rows, kFp8Block) * p.tiles_c);
  }
  if (js.blocks == 0) return SD_OK;
  auto* kernel = dtype == kF32 ? &quantize_kernel<F32> : dtype == SD_BF16 ? &quantize_kernel<BF16> : &quantize_kernel<F16>;
  hipLaunchKernelGGL(kernel, dim3(js.blocks), dim3(kThreads), 0, stream, js);
  return check_launch("fp8_quantize");
}

int launch_dequantize(const uint8_t* data, int64_t ld, const uint8_t* scales, int64_t s_r, int64_t s_k, int square, int64_t rows,
                      int64_t cols, void* out, int64_t out_ld, int dtype, hipStream_t stream) {
  const int64_t quads = ceil_div(cols, 4), blocks = ceil_div(rows * quads, kThreads);
  if (blocks == 0) return SD_OK;
  if (blocks >= (1LL << 31)) return fail(SD_ERR_UNSUPPORTED, "fp8_dequantize: %lld x %lld is too large for one launch", (long long)rows, (long long)cols);
  auto* kernel = dtype == kF32 ? &dequantize_kernel<F32> : dtype == SD_BF16 ? &dequantize_kernel<BF16> : &dequantize_kernel<F16>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kThreads), 0, stream, data, ld, scales, s_r, s_k, square, rows, cols, (uint32_t)quads, out, out_ld);
  return check_launch("fp8_dequantize");
}

}  // namespace sd
