// Matrices in 16 or 32 bits -> e4m3 codes with a power of two for each block of 1 x 128 or 128 x 128 (fp8.h), and back.
//
// A training step needs its activations and output gradients twice: with blocks along their rows for the products that sum over
// features, and with blocks along their columns, transposed, for the weight gradient, which sums over tokens.  Both come out of one
// read: a workgroup holds a 128 x 128 tile in registers, 4 rows x 8 columns a thread, takes the largest magnitude along both directions
// and writes the codes both ways, those across turned through LDS so that both are stored in whole 128-byte lines.
// Bound by its reads and writes, 2 bytes in and 1 or 2 out per element, as long as the arithmetic stays out of the way: magnitudes of
// 16-bit elements are compared two at a time as whole numbers, and the conversion takes two of them and the scale in one
// instruction (its results are those of multiplying in fp32 and converting, for every 16-bit number within the range).
// 8192^2 in 128 x 128 blocks 38 us, 5.3 TB/s; an output gradient of that size both ways 60 us, X with half of its blocks dropped and W both ways 74.
#include "fp8.h"

#include <type_traits>

namespace sd {
namespace {

constexpr int kThreads = 512;
constexpr uint32_t kDrawingBlocks = 256;  // workgroups up to which they draw the mask themselves (launch_quantize)
constexpr int kRows = 4;           // of a thread, by eight columns
constexpr int kTurnPitch = 132;    // bytes of a column's codes in LDS: 33 words, so that a wave's words meet a bank twice at most

struct F32 {
  static constexpr int id = kF32;
};

// Eight elements of a row and what is done with them.  w: two to a word; magnitudes are 15-bit whole numbers, of which the larger
// stands for the larger number.
template <typename T>
struct Eight {
  uint32_t w[4];
  __device__ inline void load(const void* src, int64_t at, int left) {
    const uint16_t* s = static_cast<const uint16_t*>(src) + at;
    if (left >= 8) {
      const u32x4 v = *reinterpret_cast<const u32x4_any*>(s);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = v[i];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = (2 * i < left ? s[2 * i] : 0u) | (2 * i + 1 < left ? (uint32_t)s[2 * i + 1] << 16 : 0u);
    }
  }
  __device__ inline void sizes(uint32_t (&a)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = w[i] & 0x7fff7fffu;
  }
};
// A thread's 4 x 8 elements.
template <typename T>
struct Patch {
  Eight<T> e[kRows];
  __device__ inline void load(const void* src, int64_t ld, int r0, int c0, int rows, int cols) {
#pragma unroll
    for (int i = 0; i < kRows; ++i) e[i].load(src, (int64_t)(r0 + i) * ld + c0, r0 + i < rows ? cols - c0 : 0);
  }
  // the largest finite magnitude of each row, and of the columns two to a word
  __device__ inline void most(uint32_t (&row)[kRows], uint32_t (&col)[4]) const {
    uint32_t a[kRows][4], all = 0u;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      e[i].sizes(a[i]);
      all = pk_max(all, pk_max(pk_max(a[i][0], a[i][1]), pk_max(a[i][2], a[i][3])));
    }
    if (max(all & 0xffffu, all >> 16) >= kInfinite<T>) {
#pragma unroll
      for (int i = 0; i < kRows; ++i)
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          if ((a[i][d] & 0xffffu) >= kInfinite<T>) a[i][d] &= 0xffff0000u;
          if (a[i][d] >> 16 >= kInfinite<T>) a[i][d] &= 0xffffu;
        }
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const uint32_t m = pk_max(pk_max(a[i][0], a[i][1]), pk_max(a[i][2], a[i][3]));
      row[i] = max(m & 0xffffu, m >> 16);
    }
#pragma unroll
    for (int d = 0; d < 4; ++d) col[d] = pk_max(pk_max(a[0][d], a[1][d]), pk_max(a[2][d], a[3][d]));
  }
  static constexpr int kColWords = 4;
  __device__ static inline uint32_t merge(uint32_t a, uint32_t b) { return pk_max(a, b); }
  __device__ static inline uint32_t bits(uint32_t m) { return size_bits<T>(m); }
  __device__ static inline uint32_t col_bits(const uint32_t (&col)[4], int j) { return size_bits<T>(j & 1 ? col[j / 2] >> 16 : col[j / 2] & 0xffffu); }
  __device__ inline u32x2 row_codes(int i, uint32_t byte) const {
    u32x2 q;
#pragma unroll
    for (int h = 0; h < 2; ++h) q[h] = codes_of<T, true>(codes_of<T, false>(0u, e[i].w[2 * h], byte), e[i].w[2 * h + 1], byte);
    return q;
  }
  __device__ inline uint32_t col_codes(int j, uint32_t byte) const {  // of the four rows
    const uint32_t pick = j & 1 ? 0x07060302u : 0x05040100u;
    const int d = j / 2;
    const uint32_t lo = __builtin_amdgcn_perm(e[1].w[d], e[0].w[d], pick), hi = __builtin_amdgcn_perm(e[3].w[d], e[2].w[d], pick);
    return codes_of<T, true>(codes_of<T, false>(0u, lo, byte), hi, byte);
  }
};
template <>
struct Patch<F32> {
  float v[kRows][8];
  __device__ inline void load(const void* src, int64_t ld, int r0, int c0, int rows, int cols) {
    typedef f32x4 __attribute__((aligned(4))) f32x4_any;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const float* s = static_cast<const float*>(src) + (int64_t)(r0 + i) * ld + c0;
      const int left = r0 + i < rows ? cols - c0 : 0;
      if (left >= 8) {
        const f32x4 a = *reinterpret_cast<const f32x4_any*>(s), b = *reinterpret_cast<const f32x4_any*>(s + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[i][j] = a[j];
          v[i][4 + j] = b[j];
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = j < left ? s[j] : 0.f;
      }
    }
  }
  static constexpr int kColWords = 8;
  __device__ inline void most(uint32_t (&row)[kRows], uint32_t (&col)[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) col[j] = 0u;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      row[i] = 0u;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t a = finite_magnitude(v[i][j]);
        row[i] = max(row[i], a);
        col[j] = max(col[j], a);
      }
    }
  }
  __device__ static inline uint32_t merge(uint32_t a, uint32_t b) { return max(a, b); }
  __device__ static inline uint32_t bits(uint32_t m) { return m; }
  __device__ static inline uint32_t col_bits(const uint32_t (&col)[8], int j) { return col[j]; }
  __device__ inline u32x2 row_codes(int i, uint32_t byte) const {
    const float s = fp8_inverse(byte);
    return u32x2{pack_fp8(v[i][0] * s, v[i][1] * s, v[i][2] * s, v[i][3] * s), pack_fp8(v[i][4] * s, v[i][5] * s, v[i][6] * s, v[i][7] * s)};
  }
  __device__ inline uint32_t col_codes(int j, uint32_t byte) const {
    const float s = fp8_inverse(byte);
    return pack_fp8(v[0][j] * s, v[1][j] * s, v[2][j] * s, v[3][j] * s);
  }
};

template <typename T>
__global__ __launch_bounds__(kThreads) void quantize_kernel(QuantJobs js) {
  constexpr int W = Patch<T>::kColWords;
  __shared__ __attribute__((aligned(16))) uint32_t most_of[kThreads / 64][16 * W];  // [wave][the columns' words], or [wave][0] of a square block
  __shared__ uint32_t turned[kFp8Block * kTurnPitch / 4];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int which = js.n > 1 && blockIdx.x >= js.job[1].first_block ? 1 : 0;
  const QuantJob& p = js.job[which];
  const uint32_t tile = blockIdx.x - p.first_block;
  const int tr = (int)(tile / p.tiles_c), tc = (int)(tile - (uint32_t)tr * p.tiles_c);
  const int r0 = tr * kFp8Block + (t >> 4) * kRows, c0 = tc * kFp8Block + (t & 15) * 8;
  bool dropped = false;
  if (p.masked) {
    MaskSrc src = js.mask;
    src.resolve();
    const int i = p.mask_t ? tc : tr, j = p.mask_t ? tr : tc, si = i / src.split, sj = j / src.split;
    dropped = src.dropped_entry(si, sj);
    if (js.mask_out && t == 0 && si * src.split == i && sj * src.split == j) js.mask_out[(int64_t)si * src.kb + sj] = dropped ? 1 : 0;
  }
  if (!dropped) {  // (uniform)
    Patch<T> v;
    v.load(p.src, p.ld, r0, c0, p.rows, p.cols);
    uint32_t row_scale[kRows], col_scale[8], row_most[kRows], col_most[W];
    v.most(row_most, col_most);
    if (p.square) {
      uint32_t m = max(max(row_most[0], row_most[1]), max(row_most[2], row_most[3]));
      m = max_of_row16(m);
      m = max(m, (uint32_t)__shfl_xor((int)m, 16));
      m = max(m, (uint32_t)__shfl_xor((int)m, 32));
      if (lane == 0) most_of[wave][0] = m;
      __syncthreads();
      m = most_of[0][0];
#pragma unroll
      for (int i = 1; i < kThreads / 64; ++i) m = max(m, most_of[i][0]);
      const uint32_t s = fp8_scale_of(Patch<T>::bits(m));
#pragma unroll
      for (int i = 0; i < kRows; ++i) row_scale[i] = s;
#pragma unroll
      for (int j = 0; j < 8; ++j) col_scale[j] = s;
    } else {
      if (p.along.data) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) row_scale[i] = fp8_scale_of(Patch<T>::bits(max_of_row16(row_most[i])));
      }
      if (p.across.data) {  // (uniform)
#pragma unroll
        for (int d = 0; d < W; ++d) {
          col_most[d] = Patch<T>::merge(col_most[d], (uint32_t)__shfl_xor((int)col_most[d], 16));
          col_most[d] = Patch<T>::merge(col_most[d], (uint32_t)__shfl_xor((int)col_most[d], 32));
          if (lane < 16) most_of[wave][lane * W + d] = col_most[d];
        }
        __syncthreads();
#pragma unroll
        for (int d = 0; d < W; ++d) {
#pragma unroll
          for (int i = 0; i < kThreads / 64; ++i) col_most[d] = Patch<T>::merge(col_most[d], most_of[i][(t & 15) * W + d]);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) col_scale[j] = fp8_scale_of(Patch<T>::col_bits(col_most, j));
      }
    }
    if (p.along.data) {
#pragma unroll
      for (int i = 0; i < kRows; ++i)
        if (r0 + i < p.rows) *reinterpret_cast<u32x2*>(p.along.data + (int64_t)(r0 + i) * p.along.ld + c0) = v.row_codes(i, row_scale[i]);
      if (p.square) {
        if (t == 0) p.along.scales[(int64_t)tr * p.along.s_r + (int64_t)tc * p.along.s_k] = (uint8_t)row_scale[0];
      } else if ((t & 15) == 0) {
#pragma unroll
        for (int i = 0; i < kRows; ++i)
          if (r0 + i < p.rows) p.along.scales[(int64_t)(r0 + i) * p.along.s_r + (int64_t)tc * p.along.s_k] = (uint8_t)row_scale[i];
      }
    }
    if (p.across.data) {
#pragma unroll
      for (int j = 0; j < 8; ++j) turned[((t & 15) * 8 + j) * (kTurnPitch / 4) + (t >> 4)] = v.col_codes(j, col_scale[j]);
      if (p.square) {
        if (t == 0) p.across.scales[(int64_t)tc * p.across.s_r + (int64_t)tr * p.across.s_k] = (uint8_t)col_scale[0];
      } else if (t < 16) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c0 + j < p.cols) p.across.scales[(int64_t)(c0 + j) * p.across.s_r + (int64_t)tr * p.across.s_k] = (uint8_t)col_scale[j];
      }
      __syncthreads();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = h * 64 + (t >> 3), at = (t & 7) * 4;
        if (tc * kFp8Block + c >= p.cols) continue;
        const uint32_t* w = turned + c * (kTurnPitch / 4) + at;
        *reinterpret_cast<u32x4*>(p.across.data + (int64_t)(tc * kFp8Block + c) * p.across.ld + tr * kFp8Block + at * 4) = u32x4{w[0], w[1], w[2], w[3]};
      }
    }
  }
  report_in(const_cast<uint64_t*>(js.mask.state), gridDim.x);
}

// A mask drawn by a launch of its own, four entries a thread.
constexpr int kDrawThreads = 256;
__global__ __launch_bounds__(kDrawThreads) void draw_mask_kernel(MaskSrc src, int64_t rows, uint8_t* out) {
  src.resolve();
  write_mask(src, rows, out, (int64_t)blockIdx.x * kDrawThreads + threadIdx.x, (int64_t)gridDim.x * kDrawThreads);
  report_in(const_cast<uint64_t*>(src.state), gridDim.x);
}

// codes and scales -> values, four to a thread at a time.  Bound by what it writes.
constexpr int kOutThreads = 256;
constexpr int64_t kOutBlocks = 1 << 20;
template <typename T>
__global__ __launch_bounds__(kOutThreads) void dequantize_kernel(const uint8_t* data, int64_t ld, const uint8_t* scales, int64_t s_r, int64_t s_k,
                                                              int square, int64_t rows, int64_t cols, uint32_t quads, void* out, int64_t out_ld) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  for (int64_t at = (int64_t)blockIdx.x * kOutThreads + threadIdx.x; at < rows * quads; at += (int64_t)gridDim.x * kOutThreads) {
    const int64_t r = at / quads, c = (at - r * quads) * 4;
    const uint32_t q = *reinterpret_cast<const uint32_t*>(data + r * ld + c);
    const float s = fp8_power(scales[(square ? r / kFp8Block : r) * s_r + c / kFp8Block * s_k]);
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)q, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)q, true);
    const float v[4] = {lo[0] * s, lo[1] * s, hi[0] * s, hi[1] * s};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (c + i >= cols) break;
      if constexpr (T::id == kF32) static_cast<float*>(out)[r * out_ld + c + i] = v[i];
      else static_cast<uint16_t*>(out)[r * out_ld + c + i] = T::from_float(v[i]);
    }
  }
}

}  // namespace

int launch_quantize(QuantJobs& js, int dtype, hipStream_t stream) {
  int64_t blocks = 0;
  for (int i = 0; i < js.n; ++i) {
    QuantJob& p = js.job[i];
    p.tiles_c = (uint32_t)ceil_div(p.cols, kFp8Block);
    p.first_block = (uint32_t)blocks;
    blocks += ceil_div(p.rows, kFp8Block) * p.tiles_c;
    if (blocks * kThreads >= (1LL << 32)) return fail(SD_ERR_UNSUPPORTED, "fp8_quantize: a %d x %d matrix is too large for one launch", p.rows, p.cols);
  }
  js.blocks = (uint32_t)blocks;
  if (js.blocks == 0) return SD_OK;
  // Workgroups that draw from the generator's state report one at a time, 10 ns each, so that the last can move it on: beyond some
  // hundreds of them a launch that draws the mask before takes less.  Forward passes of 512 outputs, drawn by the workgroups and by a launch: 32
  // workgroups 11.1 and 12.8 us, 192 17.4 and 18.8, 320 19.7 and 20.0, 576 24.0 and 22.3, 1152 37 and 30, 4352 85 and 52.
  if (js.mask_out && js.mask.state && js.blocks > kDrawingBlocks) {
    const int64_t groups = ceil_div((int64_t)js.mask.mb * js.mask.kb, 4 * kDrawThreads);
    hipLaunchKernelGGL(&draw_mask_kernel, dim3((unsigned)(groups < 64 ? groups : 64)), dim3(kDrawThreads), 0, stream, js.mask, (int64_t)js.mask.mb, js.mask_out);
    if (int rc = check_launch("fp8_draw")) return rc;
    js.mask.mask = js.mask_out;
    js.mask.st_row = js.mask.kb;
    js.mask.st_col = 1;
    js.mask.state = nullptr;
    js.mask_out = nullptr;
  }
  auto* kernel = dtype == kF32 ? &quantize_kernel<F32> : dtype == SD_BF16 ? &quantize_kernel<BF16> : &quantize_kernel<F16>;
  hipLaunchKernelGGL(kernel, dim3(js.blocks), dim3(kThreads), 0, stream, js);
  return check_launch("fp8_quantize");
}

int launch_dequantize(const uint8_t* data, int64_t ld, const uint8_t* scales, int64_t s_r, int64_t s_k, int square, int64_t rows,
                      int64_t cols, void* out, int64_t out_ld, int dtype, hipStream_t stream) {
  const int64_t quads = ceil_div(cols, 4), all = ceil_div(rows * quads, kOutThreads), blocks = all < kOutBlocks ? all : kOutBlocks;
  if (blocks == 0) return SD_OK;
  auto* kernel = dtype == kF32 ? &dequantize_kernel<F32> : dtype == SD_BF16 ? &dequantize_kernel<BF16> : &dequantize_kernel<F16>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kOutThreads), 0, stream, data, ld, scales, s_r, s_k, square, rows, cols, (uint32_t)quads, out, out_ld);
  return check_launch("fp8_dequantize");
}

}  // namespace sd
