// Matrices in 8-bit floating point and what the kernels that make and multiply them are told.
//
// A matrix [rows, cols] in 8 bits is e4m3 codes, row-major, a row's pitch a multiple of 16 bytes and its columns filled up with zeros
// to a multiple of 128, and a power of two for each block of 1 x 128 or 128 x 128: a byte, the exponent plus 127 (e8m0).  The scale
// is the least one with which the block's largest magnitude stays within 448.  Being a power of two it divides without rounding, so a
// value is rounded once, to e4m3 (by half of 2^-3 relative at most, and half of 2^-9 * scale below 2^-6 * scale), and the matrix
// instruction takes the exponent as an operand: scales cost the products no arithmetic.
#pragma once
#include "common.h"
#include "mask_source.h"

#include <type_traits>

namespace sd {

constexpr int kFp8Block = 128;
constexpr int kF32 = SD_F32;

// One matrix to be brought into 8 bits, row-major (a column-major one is the transpose of a row-major one: the caller swaps
// `along` and `across`).
struct Fp8Form {
  uint8_t* data;  // null: not wanted
  int64_t ld;     // bytes
  uint8_t* scales;
  int64_t s_r, s_k;  // scales[i * s_r + k * s_k]: row (square: 128 rows) i of the form, its 128-block k
};
struct QuantJob {
  const void* src;
  int64_t ld;  // elements
  int32_t rows, cols;
  Fp8Form along;   // codes [rows][cols], blocks along a row
  Fp8Form across;  // codes [cols][rows], blocks along a column
  int32_t square;  // blocks of 128 x 128, one scale for both forms
  int32_t masked, mask_t;  // leaves dropped blocks out; mask_t: the mask's rows run along the matrix's columns
  uint32_t tiles_c, first_block;
};
struct QuantJobs {
  QuantJob job[2];
  int n;
  uint32_t blocks;
  MaskSrc mask;       // of the one masked job; split: 128-blocks to a mask entry
  uint8_t* mask_out;  // where a drawn mask is stored, mask.kb bytes a row
};
int launch_quantize(QuantJobs& js, int dtype, hipStream_t stream);  // fills first_block, tiles_c and blocks

// C[m, n] = scale * sum over k of A[m, k] * B[n, k]
struct Fp8Gemm {
  const uint8_t *a, *b;
  int64_t lda, ldb;
  const uint8_t* sa;  // sa[k * sa_ld + m]: scale of row m's 128-block k
  int64_t sa_ld;
  const uint8_t* sb;  // square: sb[(n / 128) * sb_r + k * sb_k], else sb[k * sb_k + n]
  int64_t sb_r, sb_k;
  int32_t sb_square;
  uint16_t* c;
  int64_t c_sr, c_sc;
  int64_t M, N, K;
  float scale;
  const uint8_t* mask;  // null: nothing is dropped; else bytes, one to `split` x `split` blocks of 128
  int64_t msr, msc;
  int32_t split;
  float keep;        // expected fraction of blocks kept: picks the kernel
  float* part;       // fp32 scratch for a split reduction: [splits][M][N] in C's element order
  int64_t part_bytes;
};
enum Fp8Mode { kFp8Dense = 0, kFp8Dsd = 1, kFp8Sdd = 2 };  // the mask is over A's blocks [m, k], or over C's [m, n]
int launch_fp8_gemm(const Fp8Gemm& g, int mode, int dtype, hipStream_t stream);
// dX (SDD, B square) and dW (DSD) of a layer, in one launch where neither fills the chip
int launch_fp8_backward(const Fp8Gemm& gx, const Fp8Gemm& gw, int dtype, hipStream_t stream);
// scratch that a split reduction wants, 0 for none
int64_t fp8_gemm_scratch(int64_t M, int64_t N, int64_t K, int mode);

// y[m, n] for at most kFp8FewRows rows of x in 16 bits against weights in 8: x is quantized as it is read
constexpr int kFp8FewRows = 64;
bool fp8_few_takes(int64_t M, int64_t N, int64_t K);
struct Fp8Few {
  const uint16_t* x;
  int64_t ldx;
  const uint8_t* w;
  int64_t ldw;
  const uint8_t* sw;
  int64_t sw_r, sw_k;
  uint16_t* y;
  int64_t ldy;
  int32_t M, N, K;
};
int launch_fp8_few(const Fp8Few& g, int dtype, hipStream_t stream);

// the scale's byte of a block from the bits of its largest finite magnitude
__device__ inline uint32_t fp8_scale_of(uint32_t most) {
  const int e = (int)(most >> 23) - 8 + ((most & 0x7fffffu) > 0x600000u ? 1 : 0);  // 448 = 1.75 * 2^8
  return most == 0u ? 127u : (uint32_t)(e < 0 ? 0 : e);
}
// 2^(127 - byte), for bytes that fp8_scale_of gives (up to 247)
__device__ inline float fp8_inverse(uint32_t byte) { return __builtin_bit_cast(float, (254u - byte) << 23); }
// 2^(byte - 127); of 255 NaN, as the matrix instruction has it
__device__ inline float fp8_power(uint32_t byte) {
  const uint32_t bits = byte << 23;
  return __builtin_bit_cast(float, byte == 0u ? 0x400000u : byte == 255u ? 0x7fc00000u : bits);
}
__device__ inline uint32_t finite_magnitude(float x) {
  const uint32_t a = __builtin_bit_cast(uint32_t, x) & 0x7fffffffu;
  return a < 0x7f800000u ? a : 0u;
}
__device__ inline uint32_t pack_fp8(float a, float b, float c, float d) {
  int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
}

// 16-bit elements, two to a word.  Their magnitudes are 15-bit whole numbers, of which the larger stands for the larger number;
// from kInfinite on they are not finite.
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

__device__ inline uint32_t pk_max(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
template <typename T>
constexpr uint32_t kInfinite = T::id == SD_BF16 ? 0x7f80u : 0x7c00u;
// the bits in fp32 of a magnitude
template <typename T>
__device__ inline uint32_t size_bits(uint32_t m) {
  return T::id == SD_BF16 ? m << 16 : __builtin_bit_cast(uint32_t, F16::to_float((uint16_t)m));
}
// Two elements over 2^(byte - 127) as codes, in the lower or upper half of a word: the codes that multiplying in fp32 and converting
// give, for every 16-bit number and scale.  (The instruction looks at the scale's exponent alone, so byte 0 needs no other form.)
template <typename T, bool HI>
__device__ inline uint32_t codes_of(uint32_t old, uint32_t pair, uint32_t byte) {
  const float scale = __builtin_bit_cast(float, byte << 23);
  s16x2 r;
  if constexpr (T::id == SD_BF16) r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(__builtin_bit_cast(s16x2, old), __builtin_bit_cast(bf16x2, pair), scale, HI);
  else r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(__builtin_bit_cast(s16x2, old), __builtin_bit_cast(f16x2, pair), scale, HI);
  return __builtin_bit_cast(uint32_t, r);
}

// the largest of a value over the 16 lanes of a row, in all of them
__device__ inline uint32_t max_of_row16(uint32_t v) {
  auto turned = [](uint32_t x, auto n) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x120 + decltype(n)::value, 0xf, 0xf, false); };
  v = max(v, turned(v, std::integral_constant<int, 8>()));
  v = max(v, turned(v, std::integral_constant<int, 4>()));
  v = max(v, turned(v, std::integral_constant<int, 2>()));
  return max(v, turned(v, std::integral_constant<int, 1>()));
}

}  // namespace sd
