// C = scale * A . B^T of matrices in 8 bits with a scale for each block of 128 (fp8.h), dense, over the kept blocks of A (DSD) or for
// the kept blocks of C (SDD).
//
// The matrix instruction v_mfma_scale_f32_16x16x128_f8f6f4 takes one 128-block of 16 rows of either operand and the exponents of both
// blocks' scales, and adds to fp32 sums: a step of the loops below is one 128-block of the reduction.  Its operands come in any order
// of the block's elements as long as both have the same: a lane holds bytes 16 g .. + 15 and 64 + 16 g .. + 15 of a row, g = lane / 16.
//
// Sums.  The matrix cores add eight consecutive products of a row and a column at a time, each cut to a multiple of 2^-13 of the power of
// two that the largest of the eight (by the sum of two exponents) stands for, and then to the sums in fp32.  The codes themselves are off by up to
// 2^-4 each, so a product by 2^-3: what is cut off is 2^-10 of that, and there is no way to the cores' rate around it.
//
// Row order.  A tile's 64 rows lie in LDS as four groups of 16, group i the rows 4 r + i: the four scale bytes of rows 4 r .. + 3
// are then one word of the row order, in the lane that needs them, and the instruction picks its byte of it.  The sums come out in
// patches of four rows by four columns a lane, so C is stored from registers in whole 128-byte lines along either index.
#include "fp8.h"
#include "fp8_scales.h"
#include "gemm_device.h"
#include "tile_map.h"

#include <atomic>
#include <cmath>

namespace sd {
namespace {

constexpr int kB = kFp8Block;
constexpr int kBlockBytes = kB * kB;  // of one 128 x 128 block of codes
constexpr int kLdsLimit = 160 * 1024;
constexpr int kCus = 256;
// Workgroups of both gradients up to which they share a launch (layer steps, together and apart: 1024^3 34 and 41 us, 2048^3 50 and 60, 16384 x 512 over 512
// 58 and 62; behind it 3000^3 106 and 116, 3840^3 144 and 163, 7000 x 2000 over 1500 undropped 136 and 133).
constexpr int64_t kPairBlocks = 1024;
constexpr int kMaxList = 4096;        // 128-blocks that a workgroup's list can hold

typedef int i32x8 __attribute__((ext_vector_type(8)));

__device__ inline f32x4 mfma(const i32x8& a, const i32x8& b, const f32x4& c, int sa, int i, int sb, int j) {
  // (the byte selectors are immediates; the loops around are unrolled)
#define SD_J(I)                                                                                          \
  switch (j) {                                                                                           \
    case 0: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, I, sa, 0, sb);        \
    case 1: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, I, sa, 1, sb);        \
    case 2: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, I, sa, 2, sb);        \
    default: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, I, sa, 3, sb);       \
  }
  switch (i) {
    case 0: SD_J(0)
    case 1: SD_J(1)
    case 2: SD_J(2)
    default: SD_J(3)
  }
#undef SD_J
}

// raw buffer over `bytes` behind `base` (both wave-uniform): what a lane asks for behind them arrives as zeros
__device__ inline u32x4 buffer_over(const void* base, int64_t bytes) {
  const uint64_t b = (uint64_t)(uintptr_t)base;
  const uint32_t n = bytes <= 0 ? 0u : bytes > 0x7fffffff ? 0x7fffffffu : (uint32_t)bytes;
  return u32x4{uniform((uint32_t)b), uniform((uint32_t)(b >> 32)) & 0xffffu, uniform(n), 0x00027000u};
}
__device__ inline void buffer4_to_lds(u32x4 buffer, uint32_t lane_off, uint32_t lds_dst) {  // 4 bytes a lane
  const uint32_t a = uniform(lds_dst);
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds" ::"v"(lane_off), "s"(buffer), "s"(a) : "memory");
}
__device__ inline void buffer1_to_lds(u32x4 buffer, uint32_t lane_off, uint32_t lds_dst) {  // a byte a lane, to words
  const uint32_t a = uniform(lds_dst);
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_ubyte %0, %1, 0 offen lds" ::"v"(lane_off), "s"(buffer), "s"(a) : "memory");
}
__device__ inline void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ inline void wait_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
__device__ inline void barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// raw buffer over an operand's block of up to 128 rows
__device__ inline u32x4 block_buffer(const uint8_t* first_row, int64_t ld, int64_t rows) {
  return buffer_over(first_row, (rows < kB ? rows : kB) * ld);
}
// One 128-row block of an operand on its way into LDS, 1 KB (8 LDS rows) an instruction, 16 in all.  LDS row s = 8 q + lane / 8 of a
// group of 64 holds row 4 (s % 16) + s / 16; the 16-byte chunks of an LDS row are turned by (s / 2) % 8, so that the 16 rows of a
// fragment read meet no bank twice.
struct BlockRows {
  uint32_t even, odd;  // a lane's offset in instructions 2 n and 2 n + 1 of a group of eight
  uint32_t ld;
  __device__ inline BlockRows(int64_t ld_, int lane) {
    ld = (uint32_t)ld_;
    const uint32_t r = (uint32_t)lane / 8, p = (uint32_t)lane % 8;
    even = 4 * r * ld + ((p ^ (r / 2)) << 4);
    odd = (4 * r + 32) * ld + ((p ^ (4 + r / 2)) << 4);
  }
  // instruction q (0 .. 15; wave-uniform) of 128-block k
  __device__ inline void load(u32x4 buffer, int q, int k, uint32_t lds_block) const {
    const uint32_t on = (uint32_t)(64 * (q / 8) + q % 8 / 2) * ld + (uint32_t)k * kB;
    buffer16_to_lds(buffer, (q & 1 ? odd : even) + on, lds_block + (uint32_t)q * 1024);
  }
};

// fragment of 16 rows: group i of the 64 rows at `base`
__device__ inline i32x8 read_fragment(const char* base, int i, int lane) {
  const int r = lane & 15, g = lane >> 4;
  const char* row = base + (16 * i + r) * kB;
  const u32x4 lo = *reinterpret_cast<const u32x4*>(row + ((g ^ (r >> 1)) & 7) * 16);
  const u32x4 hi = *reinterpret_cast<const u32x4*>(row + (((g + 4) ^ (r >> 1)) & 7) * 16);
  i32x8 f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    f[e] = (int)lo[e];
    f[4 + e] = (int)hi[e];
  }
  return f;
}

struct Args {
  Fp8Gemm g;
  int32_t nk, per_split;  // 128-blocks of the reduction, of one part of it
  int32_t tiles_m, tiles_n, splits;
  bool big, duo;  // tiles of 256 x 256, of 128 x 256 (SDD) instead of 128 x 128
};

__device__ inline bool dropped(const Fp8Gemm& g, int i, int j) {
  if (g.split > 1) {
    i /= g.split;
    j /= g.split;
  }
  return g.mask[i * g.msr + j * g.msc] != 0;
}

// N neighbouring elements of C, or of a part's sums, of which `left` are there.
template <typename T, int N>
__device__ inline void store_run(const Fp8Gemm& g, float* part, int64_t at, const float (&x)[N], int left) {
  typedef f32x4 __attribute__((aligned(4))) f32x4_any;
  typedef u32x2 __attribute__((aligned(2))) u32x2_any;
  if (left < N) {
#pragma unroll
    for (int e = 0; e < N - 1; ++e) {
      if (e >= left) break;
      if (part) part[at + e] = x[e];
      else g.c[at + e] = T::from_float(x[e] * g.scale);
    }
  } else if (part) {
#pragma unroll
    for (int e = 0; e < N; e += 4) *reinterpret_cast<f32x4_any*>(part + at + e) = f32x4{x[e], x[e + 1], x[e + 2], x[e + 3]};
  } else {
    uint32_t w[N / 2];
#pragma unroll
    for (int e = 0; e < N; e += 2) w[e / 2] = T::pack2(x[e] * g.scale, x[e + 1] * g.scale);
    if constexpr (N == 4) *reinterpret_cast<u32x2_any*>(g.c + at) = u32x2{w[0], w[1]};
    else *reinterpret_cast<u32x4_any*>(g.c + at) = u32x4{w[0], w[1], w[2], w[3]};
  }
}
// The patch of 64 rows (from m0) x 64 columns (from n0) of a wave: sums of row group i and column group j in acc[i][j], scaled and
// rounded to C, or as they are to a part of a split reduction.  Four or eight elements a lane at a time, by straight code where the patch
// is whole.  (Element by element at C's edge 200 rows take 3 us longer than 256 through 2048 to 8192.)
template <typename T, bool WHOLE>
__device__ inline void store_patch_rows(const Fp8Gemm& g, int64_t m0, int64_t n0, const f32x4 (&acc)[4][4], float* part, int lane) {
  const int r = lane & 15, q = lane >> 4;
  const bool along_n = g.c_sc == 1;
  const int64_t ld = part ? (along_n ? g.N : g.M) : (along_n ? g.c_sr : g.c_sc);
  const int rows = WHOLE ? 64 : (int)(g.M - m0 < 64 ? g.M - m0 : 64) - 16 * q, cols = WHOLE ? 64 : (int)(g.N - n0 < 64 ? g.N - n0 : 64) - 4 * r;
  if (along_n) {
    const int64_t at = (m0 + 16 * q) * ld + n0 + 4 * r;
#pragma unroll
    for (int v = 0; v < 4; ++v)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x[4] = {acc[i][0][v], acc[i][1][v], acc[i][2][v], acc[i][3][v]};
        if (WHOLE || 4 * v + i < rows) store_run<T>(g, part, at + (4 * v + i) * ld, x, WHOLE ? 4 : cols);
      }
  } else {  // sixteen rows a lane and column
    const int64_t at = (n0 + 4 * r) * ld + m0 + 16 * q;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = acc[e & 3][j][2 * h + e / 4];
        if (WHOLE || j < cols) store_run<T>(g, part, at + j * ld + 8 * h, x, WHOLE ? 8 : rows - 8 * h);
      }
  }
}
template <typename T>
__device__ inline void store_patch(const Fp8Gemm& g, int64_t m0, int64_t n0, const f32x4 (&acc)[4][4], float* part, int lane) {
  if (m0 >= g.M || n0 >= g.N) return;
  if (m0 + 64 <= g.M && n0 + 64 <= g.N) store_patch_rows<T, true>(g, m0, n0, acc, part, lane);
  else store_patch_rows<T, false>(g, m0, n0, acc, part, lane);
}

// Entries 128-block | flags << 16 of blocks [lo, hi): in front, in their order, those with any flag set, whose number is
// returned; ALL: the others from behind.  flag(k): bits of what of block k is kept.  scratch: hi - lo bytes.
template <int THREADS, bool ALL, typename Flag>
__device__ inline int make_list(int lo, int hi, uint32_t* list, uint8_t* scratch, int* count, Flag flag) {
  const int t = threadIdx.x, n = hi - lo;
  for (int k = t; k < n; k += THREADS) scratch[k] = (uint8_t)flag(lo + k);
  __syncthreads();
  if (t < 64) {
    int done = 0, none = 0;
    for (int k0 = 0; k0 < n; k0 += 64) {
      const bool in = k0 + t < n;
      const uint32_t f = in ? scratch[k0 + t] : 0u;
      const uint64_t some = __ballot(f != 0u), below = (1ull << t) - 1;
      if (f) list[done + __popcll(some & below)] = (uint32_t)(lo + k0 + t) | f << 16;
      done += __popcll(some);
      if (ALL) {
        const uint64_t empty = __ballot(in && f == 0u);
        if (in && f == 0u) list[n - 1 - none - __popcll(empty & below)] = (uint32_t)(lo + k0 + t);
        none += __popcll(empty);
      }
    }
    if (t == 0) *count = done;
  }
  __syncthreads();
  return *count;
}

// ---- 128 x 128 tiles ------------------------------------------------------------------------------------------------------
// Waves of 64 x 64.  One group of four, two stages and two workgroups to a CU: while one waits at its barrier the other's matrix instructions
// run; bound by the LDS, 32 KB in and 64 KB out a step for 512 clocks of matrix instructions.  Where there are no more of them than CUs, two
// groups of four that take the steps in turn: a phase is a step, in which one group reads its step's fragments into registers and the
// other's matrix instructions run from theirs; each has two of four stages, and loads the step after its next into the one that it has just
// read.  At the end either group gives the other two of its four patches' sums through LDS and stores the other two.
constexpr int kMidStage = 2 * kBlockBytes + 2 * 512;  // A block, B block, words of scales of either
constexpr int mid_lds(int groups, int list) { return 2 * groups * kMidStage + list * 5 + 16; }
static_assert(mid_lds(2, kMaxList) <= kLdsLimit, "LDS");

template <typename T, int MODE, bool SQUARE, int GROUPS>
__device__ __forceinline__ void mid_tile(const Args& p, int block, char* smem) {
  constexpr int STAGES = 2 * GROUPS;
  const Fp8Gemm& g = p.g;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), grp = GROUPS == 1 ? 0 : wave >> 2, c = wave & 3;
  int tm, tn, part;
  tile_of_split_block<DSD_GROUP_M>(block, p.tiles_m, p.tiles_n, p.splits, tm, tn, part);
  const int64_t m0 = (int64_t)tm * kB, n0 = (int64_t)tn * kB;
  const int lo = part * p.per_split, hi = min(p.nk, lo + p.per_split);
  float* const out_part = p.splits > 1 ? g.part + (int64_t)part * g.M * g.N : nullptr;
  uint32_t* const list = reinterpret_cast<uint32_t*>(smem + STAGES * kMidStage);
  int steps = hi - lo;
  if constexpr (MODE == kFp8Dsd) {
    uint8_t* const scratch = reinterpret_cast<uint8_t*>(list + p.per_split);
    int* const count = reinterpret_cast<int*>(smem);
    steps = make_list<GROUPS * 256, false>(lo, hi, list, scratch, count, [&](int k) { return dropped(g, tm, k) ? 0 : 1; });
    __syncthreads();  // (count lies where the first stage goes)
  }
  if constexpr (MODE == kFp8Sdd) {
    if (dropped(g, tm, tn)) steps = 0;
  }
  steps = __builtin_amdgcn_readfirstlane(steps);
  const int wm = c >> 1, wn = c & 1;
  const BlockRows rows_a(g.lda, lane), rows_b(g.ldb, lane);
  const u32x4 of_a = block_buffer(g.a + m0 * g.lda, g.lda, g.M - m0), of_b = block_buffer(g.b + n0 * g.ldb, g.ldb, g.N - n0);
  const u32x4 ba = buffer_over(g.sa + m0, row_scales_left(p.nk, g.sa_ld, g.M, m0));
  const u32x4 bb = SQUARE ? buffer_over(g.sb + tn * g.sb_r, (int64_t)(p.nk - 1) * g.sb_k + 1) : buffer_over(g.sb + n0, row_scales_left(p.nk, g.sb_k, g.N, n0));
  const uint32_t lds = lds_address(smem);
  const int per_step = c < 2 ? 9 : 8;  // loads of this wave
  auto step_block = [&](int s) { return MODE == kFp8Dsd ? __builtin_amdgcn_readfirstlane((int)(list[s] & 0xffffu)) : lo + s; };
  auto load = [&](int s) {
    const int k = step_block(s);
    const uint32_t at = lds + (uint32_t)(s % STAGES) * kMidStage;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      rows_a.load(of_a, c * 4 + q, k, at);
      rows_b.load(of_b, c * 4 + q, k, at + kBlockBytes);
    }
    if (c == 0) buffer4_to_lds(ba, (uint32_t)((int64_t)k * g.sa_ld) + (lane & 31) * 4, at + 2 * kBlockBytes);
    if (c == 1) {
      if (SQUARE) buffer1_to_lds(bb, (uint32_t)((int64_t)k * g.sb_k), at + 2 * kBlockBytes + 512);
      else buffer4_to_lds(bb, (uint32_t)((int64_t)k * g.sb_k) + (lane & 31) * 4, at + 2 * kBlockBytes + 512);
    }
  };
  f32x4 acc[4][4] = {};
  i32x8 fa[4], fb[4];
  int sa, sb;
  auto read = [&](int s) {
    const char* st = smem + (s % STAGES) * kMidStage;
    const char* scales = st + 2 * kBlockBytes;
    sa = *reinterpret_cast<const int*>(scales + 64 * wm + 4 * (lane & 15));
    sb = *reinterpret_cast<const int*>(scales + 512 + (SQUARE ? 0 : 64 * wn + 4 * (lane & 15)));
    if (SQUARE) sb *= 0x01010101;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      fa[i] = read_fragment(st + wm * 64 * kB, i, lane);
      fb[i] = read_fragment(st + kBlockBytes + wn * 64 * kB, i, lane);
    }
  };
  auto multiply = [&] {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = mfma(fa[i], fb[j], acc[i][j], sa, i, sb, j);
  };
  if constexpr (GROUPS == 1) {
    if (steps > 0) load(0);
    for (int s = 0; s < steps; ++s) {
      wait_loads();
      barrier();
      if (s + 1 < steps) load(s + 1);  // (into the stage of step s - 1, which every wave is done with)
      read(s);
      multiply();
      wait_reads();  // (before the stage that was read is loaded over, behind the next barrier)
    }
  } else if (steps > 0) {
    if (grp < steps) load(grp);
    if (grp + 2 < steps) load(grp + 2);
    wait_loads_all_but(grp + 2 < steps ? per_step : 0);
    barrier();
    if (grp == 1) barrier();
    for (int s = grp; s < steps; s += 2) {
      read(s);
      wait_reads();
      barrier();  // (the group is done with the stage)
      if (s + 4 < steps) load(s + 4);
      __builtin_amdgcn_s_setprio(1);
      multiply();
      __builtin_amdgcn_s_setprio(0);
      wait_loads_all_but(s + 4 < steps ? per_step : 0);  // (step s + 2 is there)
      if (s + 1 < steps) barrier();
    }
    barrier();
    f32x4* const sums = reinterpret_cast<f32x4*>(smem) + c * 16 * 64;
    const bool stores = (c < 2) == (grp == 0);
    if (!stores) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sums[(4 * i + j) * 64 + lane] = acc[i][j];
    }
    __syncthreads();
    if (!stores) return;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] += sums[(4 * i + j) * 64 + lane];
  } else if ((c < 2) != (grp == 0)) {
    return;
  }
  store_patch<T>(g, m0 + 64 * wm, n0 + 64 * wn, acc, out_part, lane);
}

template <typename T, int MODE, bool SQUARE, int GROUPS>
__global__ __launch_bounds__(GROUPS * 256, 2) void fp8_mid_kernel(Args p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  mid_tile<T, MODE, SQUARE, GROUPS>(p, (int)blockIdx.x, smem);
}

// Both gradients of a layer in one launch, the weight gradient's workgroups behind the input gradient's.
template <typename T, int GROUPS>
__global__ __launch_bounds__(GROUPS * 256, 2) void fp8_pair_kernel(Args x, Args w, int first_w) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  if ((int)blockIdx.x < first_w) mid_tile<T, kFp8Sdd, true, GROUPS>(x, (int)blockIdx.x, smem);
  else mid_tile<T, kFp8Dsd, false, GROUPS>(w, (int)blockIdx.x - first_w, smem);
}

// ---- 256 x 256 tiles ------------------------------------------------------------------------------------------------------
// Eight waves of 128 x 64 in two groups of four, one for each of the tile's two row blocks; waves w and w + 4 share a SIMD.  A step of a
// wave is a memory phase (its share of the coming blocks on its way, then all of the step's fragments into registers) and a compute phase of
// 32 matrix instructions and nothing else.  A barrier ends each phase, and the second group runs one phase behind the first, so
// that of each SIMD's two waves one computes while the other reads.  Two stages of 64 KB: reading step s, group 0 loads B of step
// s + 1 into the other stage, group 1 the second row block of A of step s + 1 there and the first one of step s + 2 into the stage
// it reads, whose first block group 0 is done with.  A wave waits for its own loads at the end of the compute phase behind.
//
// DSD walks the 128-blocks that either row block keeps; a group whose row block drops one skips its phases' work, and the block is not
// loaded.  SDD takes two of the column blocks that either row of the pair keeps, in their order (behind them those that neither
// keeps, whose blocks of C come out as zeros); a wave whose block of C is dropped skips its work.
// 8192^3: 377 us, 2920 TFLOP/s, at the clock that the power limit leaves (the library's, with one scale for all, 337; the first 150 launches after
// a pause, while the clock settles, take 400 to 545).  Half of the blocks dropped: 255 us (DSD; in a run of 20, 285, the loads alone took 192 and reads
// and products alone 242: phases of a row block that drops its 128-block idle).
constexpr int kBigStage = 4 * kBlockBytes;        // A's two blocks, B's two
constexpr int kBigScales = 2 * kBigStage;         // then 256 bytes of A's scales and 256 of B's for each stage
constexpr int kBigList = kBigScales + 2 * 512;
constexpr int big_lds(int list) { return kBigList + list * 5 + 16; }

template <typename T, int MODE, bool SQUARE>
__global__ __launch_bounds__(512, 2) void fp8_big_kernel(Args p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const Fp8Gemm& g = p.g;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), grp = wave >> 2, c = wave & 3;
  int tm, tn, part;
  tile_of_split_block<DSD_GROUP_M>((int)blockIdx.x, p.tiles_m, p.tiles_n, p.splits, tm, tn, part);
  const int lo = part * p.per_split, hi = min(p.nk, lo + p.per_split);
  float* const out_part = p.splits > 1 ? g.part + (int64_t)part * g.M * g.N : nullptr;
  uint32_t* const list = reinterpret_cast<uint32_t*>(smem + kBigList);
  int* const count = reinterpret_cast<int*>(smem + kBigScales);
  const int row_blocks = (int)((g.M + kB - 1) / kB), col_blocks = (int)((g.N + kB - 1) / kB);
  auto kept_rows = [&](int j) {  // of column j (SDD) or 128-block j (DSD)
    return (dropped(g, 2 * tm, j) ? 0u : 1u) | (2 * tm + 1 < row_blocks && !dropped(g, 2 * tm + 1, j) ? 2u : 0u);
  };
  int steps = hi - lo, cols[2] = {2 * tn, 2 * tn + 1};
  uint32_t tiles = 0xfu;  // SDD: bit 2 b + g of row block g, column block b
  if constexpr (MODE == kFp8Dsd) {
    steps = make_list<512, false>(lo, hi, list, reinterpret_cast<uint8_t*>(list + p.per_split), count, kept_rows);
    __syncthreads();  // (count lies where the first scales go)
  }
  if constexpr (MODE == kFp8Sdd) {
    make_list<512, true>(0, col_blocks, list, reinterpret_cast<uint8_t*>(list + col_blocks), count, kept_rows);
    const uint32_t e0 = list[2 * tn], e1 = 2 * tn + 1 < col_blocks ? list[2 * tn + 1] : (uint32_t)col_blocks;
    cols[0] = (int)(e0 & 0xffffu);
    cols[1] = (int)(e1 & 0xffffu);
    tiles = uniform(e0 >> 16 | e1 >> 16 << 2);
    if (tiles == 0u) steps = 0;
    __syncthreads();
  }
  steps = __builtin_amdgcn_readfirstlane(steps);
  const int64_t m0 = (int64_t)tm * 2 * kB, c0 = (int64_t)__builtin_amdgcn_readfirstlane(cols[0]) * kB, c1 = (int64_t)__builtin_amdgcn_readfirstlane(cols[1]) * kB;
  // group 0 loads B, a column block to two waves; group 1 loads A
  const int64_t n_mine = c < 2 ? c0 : c1;
  const BlockRows rows(grp == 0 ? g.ldb : g.lda, lane);
  const u32x4 of_b = block_buffer(g.b + n_mine * g.ldb, g.ldb, g.N - n_mine);
  const u32x4 of_a0 = block_buffer(g.a + m0 * g.lda, g.lda, g.M - m0), of_a1 = block_buffer(g.a + (m0 + kB) * g.lda, g.lda, g.M - m0 - kB);
  const u32x4 ba = buffer_over(g.sa + m0, row_scales_left(p.nk, g.sa_ld, g.M, m0));
  const u32x4 bb = SQUARE ? buffer_over(g.sb, (int64_t)(col_blocks - 1) * g.sb_r + (int64_t)(p.nk - 1) * g.sb_k + 1)
                          : buffer_over(g.sb + c0, row_scales_left(p.nk, g.sb_k, g.N, c0));
  const uint32_t square_at = SQUARE ? (uint32_t)((lane < 32 ? c0 : c1) / kB * g.sb_r) : 0u;
  const uint32_t lds = lds_address(smem);
  auto load_b = [&](int s, int k) {
    const uint32_t at = lds + (uint32_t)(s & 1) * kBigStage + (2 + c / 2) * kBlockBytes, scales = lds + kBigScales + (uint32_t)(s & 1) * 512;
    if (MODE != kFp8Sdd || (tiles >> (2 * (c / 2)) & 3u)) {
#pragma unroll
      for (int q = 0; q < 8; ++q) rows.load(of_b, 8 * (c & 1) + q, k, at);
    }
    if (c == 0) buffer4_to_lds(ba, (uint32_t)((int64_t)k * g.sa_ld) + lane * 4, scales);
    if (c == 1) {
      if (SQUARE) buffer1_to_lds(bb, square_at + (uint32_t)((int64_t)k * g.sb_k), scales + 256);
      else buffer4_to_lds(bb, (uint32_t)((int64_t)k * g.sb_k) + lane * 4, scales + 256);
    }
  };
  auto load_a = [&](int row, int s, int k) {
    const uint32_t at = lds + (uint32_t)(s & 1) * kBigStage + row * kBlockBytes;
    if (row) {
#pragma unroll
      for (int q = 0; q < 4; ++q) rows.load(of_a1, 4 * c + q, k, at);
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) rows.load(of_a0, 4 * c + q, k, at);
    }
  };
  auto entry = [&](int s) -> uint32_t {
    if (MODE == kFp8Dsd) return s < steps ? list[s] : 0u;
    return (uint32_t)(lo + s) | (MODE == kFp8Sdd ? ((tiles | tiles >> 2) & 3u) : 3u) << 16;
  };
  auto flag = [](uint32_t e, int row) { return (e >> 16 >> row & 1u) != 0u; };
  auto block = [](uint32_t e) { return (int)(e & 0xffffu); };

  f32x4 acc[2][4][4] = {};
  if (steps > 0) {
    uint32_t e0 = uniform(entry(0)), e1 = uniform(entry(1)), e2 = uniform(entry(2));
    const bool works = MODE != kFp8Sdd || (tiles >> (2 * (c / 2) + grp) & 1u);
    if (grp == 0) {
      load_b(0, block(e0));
    } else {
      if (flag(e0, 0)) load_a(0, 0, block(e0));
      if (flag(e0, 1)) load_a(1, 0, block(e0));
      if (steps > 1 && flag(e1, 0)) load_a(0, 1, block(e1));
    }
    wait_loads();
    barrier();
    if (grp == 1) barrier();
    for (int s = 0; s < steps; ++s) {
      // memory phase
      if (grp == 0) {
        if (s + 1 < steps) load_b(s + 1, block(e1));
      } else {
        if (s + 1 < steps && flag(e1, 1)) load_a(1, s + 1, block(e1));
        if (s + 2 < steps && flag(e2, 0)) load_a(0, s + 2, block(e2));
      }
      const bool on = works && flag(e0, grp);
      i32x8 fa[8], fb[4];
      int sa[2], sb;
      if (on) {
        const char* st = smem + (s & 1) * kBigStage;
        const char* scales = smem + kBigScales + (s & 1) * 512;
        sa[0] = *reinterpret_cast<const int*>(scales + 128 * grp + 4 * (lane & 15));
        sa[1] = *reinterpret_cast<const int*>(scales + 128 * grp + 64 + 4 * (lane & 15));
        sb = *reinterpret_cast<const int*>(scales + 256 + (SQUARE ? 128 * (c / 2) : 64 * c + 4 * (lane & 15)));
        if (SQUARE) sb *= 0x01010101;
#pragma unroll
        for (int j = 0; j < 4; ++j) fb[j] = read_fragment(st + (2 + c / 2) * kBlockBytes + (c & 1) * 64 * kB, j, lane);
#pragma unroll
        for (int i = 0; i < 8; ++i) fa[i] = read_fragment(st + grp * kBlockBytes + (i / 4) * 64 * kB, i & 3, lane);
      }
      wait_reads();
      barrier();
      // compute phase
      const uint32_t e3 = entry(s + 3);
      if (on) {
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[h][i][j] = mfma(fa[4 * h + i], fb[j], acc[h][i][j], sa[h], i, sb, j);
        __builtin_amdgcn_s_setprio(0);
      }
      e0 = e1;
      e1 = e2;
      e2 = uniform(e3);
      wait_loads();
      if (grp == 0 || s + 1 < steps) barrier();
    }
  }
  const int64_t n_out = n_mine + (c & 1) * 64;
#pragma unroll
  for (int h = 0; h < 2; ++h) store_patch<T>(g, m0 + grp * kB + h * 64, n_out, acc[h], out_part, lane);
}

// ---- 128 x 256 tiles of C's kept blocks ------------------------------------------------------------------------------------------
// SDD where much is dropped: a workgroup takes two kept column blocks of one row block, so none of its work is for blocks that
// are dropped.  Eight waves of 128 x 64 in two groups of four that take the steps in turn, so that each has half of the reduction; waves w
// and w + 4, one of either group, share a SIMD.  A phase is a step: while one group reads the step's fragments into registers (and
// puts the blocks of the step after next on their way into the third stage), the other's matrix instructions run from theirs.  At the end the
// groups swap halves of their sums through LDS, add and store a half each.
// dX of 8192^3 at p = 0.5: 293 us, 307 on 256 x 256 tiles (duo_pays has both at other sizes); it loads 48 KB for two blocks of C a step, those 64 for up to four.
// (DSD in this shape, whose row blocks walk the reduction apart from each other and meet in the L2 less: 431 us when 256 x 256 took 310.)
constexpr int kDuoStage = 3 * kBlockBytes;        // A's block, B's two
constexpr int kDuoScales = 3 * kDuoStage;         // then 256 bytes of A's scales and 256 of B's for each stage
constexpr int kDuoList = kDuoScales + 3 * 512;
constexpr int kDuoMaxList = 2048;
constexpr int duo_lds(int list) { return kDuoList + list * 5 + 16; }
static_assert(duo_lds(kDuoMaxList) <= kLdsLimit && 8 * 16 * 1024 <= kDuoScales, "LDS");

template <typename T>
__global__ __launch_bounds__(512, 2) void fp8_duo_kernel(Args p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const Fp8Gemm& g = p.g;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), grp = wave >> 2, c = wave & 3;
  int tm, tn;
  tile_of_block<DSD_GROUP_M>((int)blockIdx.x, p.tiles_m, p.tiles_n, tm, tn);
  uint32_t* const list = reinterpret_cast<uint32_t*>(smem + kDuoList);
  const int col_blocks = (int)((g.N + kB - 1) / kB), steps_all = p.nk;
  make_list<512, true>(0, col_blocks, list, reinterpret_cast<uint8_t*>(list + col_blocks), reinterpret_cast<int*>(smem), [&](int j) { return dropped(g, tm, j) ? 0u : 1u; });
  const uint32_t e0 = list[2 * tn], e1 = 2 * tn + 1 < col_blocks ? list[2 * tn + 1] : (uint32_t)col_blocks;
  const uint32_t tiles = uniform(e0 >> 16 | e1 >> 16 << 1);  // which of the two are kept
  const int steps = tiles ? steps_all : 0;
  const int64_t m0 = (int64_t)tm * kB, c0 = (int64_t)uniform(e0 & 0xffffu) * kB, c1 = (int64_t)uniform(e1 & 0xffffu) * kB;
  const int64_t n_mine = c < 2 ? c0 : c1;
  __syncthreads();  // (the count lies where the first stage goes)
  // a wave loads a quarter of A's block and half of its column block
  const BlockRows rows_a(g.lda, lane), rows_b(g.ldb, lane);
  const u32x4 of_a = block_buffer(g.a + m0 * g.lda, g.lda, g.M - m0), of_b = block_buffer(g.b + n_mine * g.ldb, g.ldb, g.N - n_mine);
  const u32x4 ba = buffer_over(g.sa + m0, row_scales_left(p.nk, g.sa_ld, g.M, m0));
  const u32x4 bb = buffer_over(g.sb, (int64_t)(col_blocks - 1) * g.sb_r + (int64_t)(p.nk - 1) * g.sb_k + 1);
  const uint32_t square_at = (uint32_t)((lane < 32 ? c0 : c1) / kB * g.sb_r);
  const uint32_t lds = lds_address(smem);
  const bool works = (tiles >> (c / 2) & 1u) != 0u;
  auto load = [&](int k, int stage) {
    const uint32_t at = lds + (uint32_t)stage * kDuoStage, scales = lds + kDuoScales + (uint32_t)stage * 512;
    if (works) {
#pragma unroll
      for (int q = 0; q < 8; ++q) rows_b.load(of_b, 8 * (c & 1) + q, k, at + (1 + c / 2) * kBlockBytes);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) rows_a.load(of_a, 4 * c + q, k, at);
    if (c == 0) buffer4_to_lds(ba, (uint32_t)((int64_t)k * g.sa_ld) + (lane & 31) * 4, scales);
    if (c == 1) buffer1_to_lds(bb, square_at + (uint32_t)((int64_t)k * g.sb_k), scales + 256);
  };

  f32x4 acc[2][4][4] = {};
  if (steps > 0) {
    if (grp < steps) load(grp, grp);
    wait_loads();
    barrier();
    if (grp == 1) barrier();
    int stage = grp;
    for (int s = grp; s < steps; s += 2) {
      // memory phase; the stage after next, which is the one before this, is free
      const int to = stage == 0 ? 2 : stage - 1;
      if (s + 2 < steps) load(s + 2, to);
      i32x8 fa[8], fb[4];
      int sa[2], sb;
      const char* st = smem + stage * kDuoStage;
      const char* scales = smem + kDuoScales + stage * 512;
      sa[0] = *reinterpret_cast<const int*>(scales + 4 * (lane & 15));
      sa[1] = *reinterpret_cast<const int*>(scales + 64 + 4 * (lane & 15));
      sb = *reinterpret_cast<const int*>(scales + 256 + 128 * (c / 2)) * 0x01010101;
      if (works) {
#pragma unroll
        for (int j = 0; j < 4; ++j) fb[j] = read_fragment(st + (1 + c / 2) * kBlockBytes + (c & 1) * 64 * kB, j, lane);
#pragma unroll
        for (int i = 0; i < 8; ++i) fa[i] = read_fragment(st + (i / 4) * 64 * kB, i & 3, lane);
      }
      wait_reads();
      barrier();
      // compute phase
      if (works) {
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[h][i][j] = mfma(fa[4 * h + i], fb[j], acc[h][i][j], sa[h], i, sb, j);
        __builtin_amdgcn_s_setprio(0);
      }
      stage = to;
      wait_loads();
      if (s + 1 < steps) barrier();
    }
    // group 0 gives away the sums of the second 64 rows, group 1 those of the first
    barrier();
    f32x4* const mine = reinterpret_cast<f32x4*>(smem) + wave * 16 * 64;
    const f32x4* const other = reinterpret_cast<const f32x4*>(smem) + (wave ^ 4) * 16 * 64;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) mine[(4 * i + j) * 64 + lane] = grp ? acc[0][i][j] : acc[1][i][j];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[0][i][j] = (grp ? acc[1][i][j] : acc[0][i][j]) + other[(4 * i + j) * 64 + lane];
  }
  store_patch<T>(g, m0 + grp * 64, n_mine + (c & 1) * 64, acc[0], nullptr, lane);
}

// C = scale * sum of the parts, in their order
template <typename T>
__global__ __launch_bounds__(256) void fp8_sum_kernel(Fp8Gemm g, int splits) {
  const bool along_n = g.c_sc == 1;
  const int64_t width = along_n ? g.N : g.M, total = g.M * g.N, ld = along_n ? g.c_sr : g.c_sc;
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= total) return;
  if (total % 4 == 0 && width % 4 == 0) {
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < splits; ++s) sum += *reinterpret_cast<const f32x4*>(g.part + s * total + at);
    sum *= g.scale;
    typedef u32x2 __attribute__((aligned(2))) u32x2_any;
    const int64_t r = at / width;
    *reinterpret_cast<u32x2_any*>(g.c + r * ld + (at - r * width)) = u32x2{T::pack2(sum[0], sum[1]), T::pack2(sum[2], sum[3])};
    return;
  }
  for (int64_t e = at; e < at + 4 && e < total; ++e) {
    float sum = 0.f;
    for (int s = 0; s < splits; ++s) sum += g.part[s * total + e];
    const int64_t r = e / width;
    g.c[r * ld + (e - r * width)] = T::from_float(sum * g.scale);
  }
}

// Lets a kernel have more than 64 KB of LDS, once per device.
int configure(const void* kernel, std::atomic<bool>* done) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 16)
    return fail(SD_ERR_RUNTIME, "hipGetDevice failed or device index out of range");
  if (done[dev].load(std::memory_order_acquire)) return SD_OK;
  const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, kLdsLimit);
  if (e != hipSuccess) return fail(SD_ERR_RUNTIME, "hipFuncSetAttribute: %s", hipGetErrorString(e));
  done[dev].store(true, std::memory_order_release);
  return SD_OK;
}

// How a product is cut up.  256 x 256 tiles where they fill the chip; else 128 x 128 ones, and where there are few of them and the
// reduction is long, that is cut into parts.  A part costs its fp32 sums, written and read once, and one more launch; what it saves are
// steps, a microsecond each with two workgroups on a CU and 0.55 with one (128 x 32768 at 512, 1024, 2048: 8, 11, 16 us).
struct Plan {
  bool big;
  int splits, per_split;
};
Plan plan(int64_t M, int64_t N, int64_t K, int mode) {
  const int64_t nk = ceil_div(K, kB), tiles = ceil_div(M, kB) * ceil_div(N, kB), big_tiles = ceil_div(M, 2 * kB) * ceil_div(N, 2 * kB);
  const bool big = big_tiles >= kCus;
  int64_t splits = 1;
  if (mode != kFp8Sdd && !big) {
    double least = 1e30;
    for (int64_t s = 1; s <= 16 && (s == 1 || nk / s >= 2); ++s) {
      const int64_t steps = ceil_div(nk, s), wgs = tiles * ceil_div(nk, steps);
      const double us = wgs <= kCus ? 0.55 * steps : (double)ceil_div(wgs, 2 * kCus) * (1.0 * steps + 3.0);
      const double sum = s == 1 ? 0.0 : 4.0 + 8e-6 / 4.0 * (double)(ceil_div(nk, steps) * M * N);
      if (us + sum < least) {
        least = us + sum;
        splits = s;
      }
    }
  }
  if (mode == kFp8Dsd && ceil_div(nk, splits) > kMaxList) splits = ceil_div(nk, kMaxList);
  const int64_t per = ceil_div(nk, splits > 0 ? splits : 1);
  return {big, (int)ceil_div(nk, per), (int)per};
}

int64_t blocks_of(const Args& p) { return (int64_t)p.tiles_m * p.tiles_n * p.splits; }

template <typename T>
int launch_sum(const Args& p, hipStream_t stream) {
  if (p.splits <= 1) return SD_OK;
  hipLaunchKernelGGL(&fp8_sum_kernel<T>, dim3((unsigned)ceil_div(p.g.M * p.g.N, 1024)), dim3(256), 0, stream, p.g, p.splits);
  return check_launch("fp8_sum");
}

template <typename T, int MODE, int GROUPS>
int launch_mid(const Args& p, hipStream_t stream) {
  auto* kernel = p.g.sb_square ? &fp8_mid_kernel<T, MODE, true, GROUPS> : &fp8_mid_kernel<T, MODE, false, GROUPS>;
  static std::atomic<bool> configured[2][16] = {};
  if (int rc = configure(reinterpret_cast<const void*>(kernel), configured[p.g.sb_square])) return rc;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks_of(p)), dim3(GROUPS * 256), mid_lds(GROUPS, MODE == kFp8Dsd ? p.per_split : 0), stream, p);
  note_kernel("fp8:mid groups=%d splits=%d", GROUPS, p.splits);
  return check_launch("fp8_gemm");
}

// Two groups of waves where every workgroup has a CU to itself and more than eight steps.  One group and two: 1024^2 over 512 6.0 and 7.4 us, 1024 8.4 and
// 9.2, 1152 9.2 and 9.9, 1536 11.5 and 11.5, 2048 13.1 and 13.1; 2048^2 over 2048 15.0 and 14.5, over 4096 23.9 and 22.3, 512 x 4096 over 4096 22.6 and 20.8
// (with few steps the exchange of sums at the end, about 1 us, counts); more tiles than CUs: 2176 x 2048 over 2048 16.0 and 25.2.
bool deep(int64_t blocks, const Args& p) { return blocks <= kCus && p.per_split > 8; }

template <typename T, int MODE>
int launch_big(const Args& p, hipStream_t stream) {
  auto* kernel = p.g.sb_square ? &fp8_big_kernel<T, MODE, true> : &fp8_big_kernel<T, MODE, false>;
  static std::atomic<bool> configured[2][16] = {};
  if (int rc = configure(reinterpret_cast<const void*>(kernel), configured[p.g.sb_square])) return rc;
  const int list = MODE == kFp8Dsd ? p.per_split : MODE == kFp8Sdd ? (int)ceil_div(p.g.N, kB) : 0;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks_of(p)), dim3(512), big_lds(list), stream, p);
  note_kernel("fp8:big splits=%d", p.splits);
  return check_launch("fp8_gemm");
}

template <typename T>
int launch_duo(const Args& p, hipStream_t stream) {
  auto* kernel = &fp8_duo_kernel<T>;
  static std::atomic<bool> configured[16] = {};
  if (int rc = configure(reinterpret_cast<const void*>(kernel), configured)) return rc;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks_of(p)), dim3(512), duo_lds((int)ceil_div(p.g.N, kB)), stream, p);
  note_kernel("fp8:duo");
  return check_launch("fp8_gemm");
}

template <typename T, int MODE>
int launch(const Args& p, hipStream_t stream) {
  if (p.duo) return launch_duo<T>(p, stream);
  if (p.big) {
    if (int rc = launch_big<T, MODE>(p, stream)) return rc;
    return launch_sum<T>(p, stream);
  }
  if (blocks_of(p) >= (1LL << 31)) return fail(SD_ERR_UNSUPPORTED, "fp8 product: %lld tiles are too many for one launch", (long long)blocks_of(p));
  if (int rc = deep(blocks_of(p), p) ? launch_mid<T, MODE, 2>(p, stream) : launch_mid<T, MODE, 1>(p, stream)) return rc;
  return launch_sum<T>(p, stream);
}

template <typename T, int GROUPS>
int launch_pair(const Args& x, const Args& w, hipStream_t stream) {
  auto* kernel = &fp8_pair_kernel<T, GROUPS>;
  static std::atomic<bool> configured[16] = {};
  if (int rc = configure(reinterpret_cast<const void*>(kernel), configured)) return rc;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(blocks_of(x) + blocks_of(w))), dim3(GROUPS * 256), mid_lds(GROUPS, w.per_split), stream, x, w, (int)blocks_of(x));
  note_kernel("fp8:pair groups=%d splits=%d", GROUPS, w.splits);
  if (int rc = check_launch("fp8_pair")) return rc;
  return launch_sum<T>(w, stream);
}

// Rounds of the busiest XCD's 32 CUs through the workgroups that have work, of `rows` x `cols` of them of which each row's first `full` do: an
// XCD gets one run of an order that walks DSD_GROUP_M rows column by column, and half of the XCDs may get the empty ends of rows.
int64_t busiest_rounds(int64_t rows, int64_t cols, double full) {
  const int64_t run = ceil_div(rows * cols, 8), group = DSD_GROUP_M * cols;
  const double in_group = DSD_GROUP_M * (full < (double)cols ? full : (double)cols), rest = (double)(run % group);
  const int64_t work = (int64_t)ceil((double)(run / group) * in_group + (rest < in_group ? rest : in_group));
  return work > 32 ? ceil_div(work, 32) : 1;
}
// SDD on tiles of 128 x 256 of a row block's kept blocks instead of 256 x 256 of those that either row block of a pair keeps: where their
// rounds are expected to take less.  Microseconds, with nk = N / 128 steps, a round 0.9 nk + 10 and 1.25 nk + 5.  Input gradients with their quantizing,
// 128 x 256 and 256 x 256: 8192^3, p = 0.4 378 and 362 us, 0.5 329 and 343, 0.75 218 and 345; 4096^3, 0.5 74 and 58, 0.75 72 and 56;
// 4096 x 8192 over 8192, 0.5 248 and 185 (the full ends of 32 row blocks go to four XCDs), 8192 x 8192 over 4096, 0.75 123 and 173.
// Over 152 products of 4096 to 18000 rows, p from 0.2 to 0.9 and blocks of 128 to 384 the choice takes 0.7 % longer than the faster of both (17 % at
// most), by the drop rate alone (from 0.45 on) 8 % (50 %), 256 x 256 tiles always 3.3 % (76 %).
bool duo_pays(const Fp8Gemm& g) {
  const double cols = (double)ceil_div(g.N, kB), keep = g.keep;
  // a pair of row blocks shares its mask where the mask's blocks are a multiple of 256, else one of two keeps more; an odd number of kept
  // blocks, every other row, leaves half a workgroup
  const bool even = g.split % 2 == 0;
  const double either = even ? keep : 1.0 - (1.0 - keep) * (1.0 - keep), odd = even ? 0.0 : 0.25;
  const int64_t pairs = ceil_div(g.N, 2 * kB), nk = ceil_div(g.K, kB);
  const double duo = (double)busiest_rounds(ceil_div(g.M, kB), pairs, cols * keep / 2 + odd) * (0.9 * nk + 10.0);
  const double big = (double)busiest_rounds(ceil_div(g.M, 2 * kB), pairs, cols * either / 2 + odd) * (1.25 * nk + 5.0) + 5.0;
  return duo < big;
}

int make_args(const Fp8Gemm& g, int mode, Args& p) {
  p.g = g;
  const Plan q = plan(g.M, g.N, g.K, mode);
  p.nk = (int)ceil_div(g.K, kB);
  p.splits = q.splits;
  p.per_split = q.per_split;
  if (q.splits > 1 && (g.part == nullptr || g.part_bytes < (int64_t)p.splits * g.M * g.N * 4)) {
    if (mode == kFp8Dsd && p.nk > kMaxList) return fail(SD_ERR_INVALID, "fp8 product: a reduction of %d blocks needs its scratch", p.nk);
    p.splits = 1;
    p.per_split = p.nk;
  }
  // (SDD on large tiles lists a row pair's column blocks)
  p.big = q.big && !(mode == kFp8Sdd && (!g.sb_square || ceil_div(g.N, kB) > kMaxList));
  p.duo = p.big && mode == kFp8Sdd && ceil_div(g.N, kB) <= kDuoMaxList && duo_pays(g);
  if (p.duo) p.big = false;
  p.tiles_m = (int)ceil_div(g.M, p.big ? 2 * kB : kB);
  p.tiles_n = (int)ceil_div(g.N, p.big || p.duo ? 2 * kB : kB);
  return SD_OK;
}

}  // namespace

int64_t fp8_gemm_scratch(int64_t M, int64_t N, int64_t K, int mode) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const Plan q = plan(M, N, K, mode);
  return q.splits > 1 ? (int64_t)q.splits * M * N * 4 : 0;
}

int launch_fp8_gemm(const Fp8Gemm& g, int mode, int dtype, hipStream_t stream) {
  if (g.M == 0 || g.N == 0) return SD_OK;
  Args p;
  if (int rc = make_args(g, mode, p)) return rc;
  if (dtype == SD_BF16) {
    if (mode == kFp8Dense) return launch<BF16, kFp8Dense>(p, stream);
    return mode == kFp8Dsd ? launch<BF16, kFp8Dsd>(p, stream) : launch<BF16, kFp8Sdd>(p, stream);
  }
  if (mode == kFp8Dense) return launch<F16, kFp8Dense>(p, stream);
  return mode == kFp8Dsd ? launch<F16, kFp8Dsd>(p, stream) : launch<F16, kFp8Sdd>(p, stream);
}

int launch_fp8_backward(const Fp8Gemm& gx, const Fp8Gemm& gw, int dtype, hipStream_t stream) {
  Args x, w;
  if (int rc = make_args(gx, kFp8Sdd, x)) return rc;
  if (int rc = make_args(gw, kFp8Dsd, w)) return rc;
  const int64_t blocks = blocks_of(x) + blocks_of(w);
  if (!gx.sb_square || gw.sb_square || x.big || w.big || x.duo || w.duo || blocks > kPairBlocks) {
    if (int rc = launch_fp8_gemm(gx, kFp8Sdd, dtype, stream)) return rc;
    return launch_fp8_gemm(gw, kFp8Dsd, dtype, stream);
  }
  const bool two = deep(blocks, x) || deep(blocks, w);
  if (dtype == SD_BF16) return two ? launch_pair<BF16, 2>(x, w, stream) : launch_pair<BF16, 1>(x, w, stream);
  return two ? launch_pair<F16, 2>(x, w, stream) : launch_pair<F16, 1>(x, w, stream);
}

}  // namespace sd
