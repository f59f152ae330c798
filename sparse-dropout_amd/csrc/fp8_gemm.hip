// C = scale * A . B^T of matrices in 8 bits with a scale for each block of 128 (fp8.h), dense, over the kept blocks of A (DSD) or for
// the kept blocks of C (SDD).
//
// The matrix instruction v_mfma_scale_f32_16x16x128_f8f6f4 takes one 128-block of 16 rows of either operand and the exponents of both
// blocks' scales, and adds to fp32 sums: a step of the loops below is one 128-block of the reduction.  Its operands come in any order
// of the block's elements as long as both have the same: a lane holds bytes 16 g .. + 15 and 64 + 16 g .. + 15 of a row, g = lane / 16.
//
// Row order.  A tile's 64 rows lie in LDS as four groups of 16, group i the rows 4 r + i: the four scale bytes of rows 4 r .. + 3
// are then one word of the row order, in the lane that needs them, and the instruction picks its byte of it.  The sums come out in
// patches of four rows by four columns a lane, so C is stored from registers in whole 128-byte lines along either index.
#include "fp8.h"
#include "gemm_device.h"
#include "tile_map.h"

#include <atomic>

namespace sd {
namespace {

constexpr int kB = kFp8Block;
constexpr int kBlockBytes = kB * kB;  // of one 128 x 128 block of codes
constexpr int kLdsLimit = 160 * 1024;
constexpr int kCus = 256;
constexpr int64_t kPairBlocks = 1024;  // workgroups of both gradients up to which they share a launch
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

// One 128-row block of an operand on its way into LDS, 1 KB (8 LDS rows) an instruction, 16 in all.
struct BlockLoader {
  u32x4 buffer;       // from the block's first row
  uint32_t even, odd; // a lane's offset in instructions 2 n and 2 n + 1 of a group of eight (see offset())
  uint32_t ld;
  // LDS row s = 8 q + lane / 8 of a group of 64 holds row 4 (s % 16) + s / 16; the 16-byte chunks of an LDS row are turned by
  // (s / 2) % 8, so that the 16 rows of a fragment read meet no bank twice
  __device__ inline void init(const uint8_t* base, int64_t ld_, int64_t rows, int lane) {
    buffer = buffer_over(base, (rows < kB ? rows : kB) * ld_);
    ld = (uint32_t)ld_;
    const uint32_t r = (uint32_t)lane / 8, p = (uint32_t)lane % 8;
    even = 4 * r * ld + ((p ^ (r / 2)) << 4);
    odd = (4 * r + 32) * ld + ((p ^ (4 + r / 2)) << 4);
  }
  // instruction q (0 .. 15; wave-uniform) of 128-block k
  __device__ inline void load(int q, int k, uint32_t lds_block) const {
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
};

__device__ inline bool dropped(const Fp8Gemm& g, int i, int j) {
  if (g.split > 1) {
    i /= g.split;
    j /= g.split;
  }
  return g.mask[i * g.msr + j * g.msc] != 0;
}

// The patch of 64 rows (from m0) x 64 columns (from n0) of a wave: sums of row group i and column group j in acc[i][j].
template <typename T>
__device__ inline void store_patch(const Fp8Gemm& g, int64_t m0, int64_t n0, const f32x4 (&acc)[4][4], float* part, int lane) {
  const int r = lane & 15, q = lane >> 4;
  const bool along_n = g.c_sc == 1;
  const float scale = part ? 1.f : g.scale;
  const int64_t ld = part ? (along_n ? g.N : g.M) : (along_n ? g.c_sr : g.c_sc);
  if (along_n) {
    const int64_t n = n0 + 4 * r;
    if (n >= g.N) return;
    const bool whole = n + 4 <= g.N;
#pragma unroll
    for (int v = 0; v < 4; ++v)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t m = m0 + 16 * q + 4 * v + i;
        if (m >= g.M) continue;
        const float x[4] = {acc[i][0][v] * scale, acc[i][1][v] * scale, acc[i][2][v] * scale, acc[i][3][v] * scale};
        if (part) {
          float* dst = part + m * ld + n;
          if (whole && g.N % 4 == 0) *reinterpret_cast<f32x4*>(dst) = f32x4{x[0], x[1], x[2], x[3]};
          else
            for (int j = 0; j < 4; ++j)
              if (n + j < g.N) dst[j] = x[j];
        } else {
          uint16_t* dst = g.c + m * ld + n;
          typedef u32x2 __attribute__((aligned(2))) u32x2_any;
          if (whole) *reinterpret_cast<u32x2_any*>(dst) = u32x2{T::pack2(x[0], x[1]), T::pack2(x[2], x[3])};
          else
            for (int j = 0; j < 4; ++j)
              if (n + j < g.N) dst[j] = T::from_float(x[j]);
        }
      }
    return;
  }
  const int64_t m = m0 + 16 * q;  // sixteen rows a lane and column
  if (m >= g.M) return;
  const bool whole = m + 16 <= g.M;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t n = n0 + 4 * r + j;
    if (n >= g.N) continue;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = acc[e & 3][j][2 * h + e / 4] * scale;
      if (part) {
        float* dst = part + n * ld + m + 8 * h;
        if (whole && g.M % 4 == 0) {
          *reinterpret_cast<f32x4*>(dst) = f32x4{x[0], x[1], x[2], x[3]};
          *reinterpret_cast<f32x4*>(dst + 4) = f32x4{x[4], x[5], x[6], x[7]};
        } else {
          for (int e = 0; e < 8; ++e)
            if (m + 8 * h + e < g.M) dst[e] = x[e];
        }
      } else {
        uint16_t* dst = g.c + n * ld + m + 8 * h;
        if (whole) *reinterpret_cast<u32x4_any*>(dst) = u32x4{T::pack2(x[0], x[1]), T::pack2(x[2], x[3]), T::pack2(x[4], x[5]), T::pack2(x[6], x[7])};
        else
          for (int e = 0; e < 8; ++e)
            if (m + 8 * h + e < g.M) dst[e] = T::from_float(x[e]);
      }
    }
  }
}

// The steps of a workgroup: list[s] = 128-block | flags << 16 of the blocks with any flag set, in order; returns how many.
// flag(k): bits of what of block k is kept, for k in [lo, hi).  smem: (hi - lo) bytes of scratch.
template <int THREADS, typename Flag>
__device__ inline int make_list(int lo, int hi, uint32_t* list, uint8_t* scratch, int* count, Flag flag) {
  const int t = threadIdx.x, n = hi - lo;
  for (int k = t; k < n; k += THREADS) scratch[k] = (uint8_t)flag(lo + k);
  __syncthreads();
  if (t < 64) {
    int done = 0;
    for (int k0 = 0; k0 < n; k0 += 64) {
      const uint32_t f = k0 + t < n ? scratch[k0 + t] : 0u;
      const uint64_t some = __ballot(f != 0u);
      if (f) list[done + __popcll(some & ((1ull << t) - 1))] = (uint32_t)(lo + k0 + t) | f << 16;
      done += __popcll(some);
    }
    if (t == 0) *count = done;
  }
  __syncthreads();
  return *count;
}

// ---- 128 x 128 tiles ------------------------------------------------------------------------------------------------------
// Four waves of 64 x 64.  Two stages and two workgroups to a CU: while one waits at its barrier the other's matrix instructions run; bound
// by the LDS, 32 KB in and 64 KB out a step for 512 clocks of matrix instructions.  Four stages, a workgroup to a CU, where
// there are no more of them than CUs: then a step costs what is left of a load's latency, of which three steps are on their way.
constexpr int kMidStage = 2 * kBlockBytes + 2 * 512;  // A block, B block, words of scales of either
constexpr int mid_lds(int stages, int list) { return stages * kMidStage + list * 5 + 16; }

template <typename T, int MODE, bool SQUARE, int STAGES>
__device__ __forceinline__ void mid_tile(const Args& p, int block, char* smem) {
  const Fp8Gemm& g = p.g;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
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
    steps = make_list<256>(lo, hi, list, scratch, count, [&](int k) { return dropped(g, tm, k) ? 0 : 1; });
    __syncthreads();  // (count lies where the first stage goes)
  }
  if constexpr (MODE == kFp8Sdd) {
    if (dropped(g, tm, tn)) steps = 0;
  }
  steps = __builtin_amdgcn_readfirstlane(steps);
  const int wm = wave >> 1, wn = wave & 1;
  BlockLoader la, lb;
  la.init(g.a + m0 * g.lda, g.lda, g.M - m0, lane);
  lb.init(g.b + n0 * g.ldb, g.ldb, g.N - n0, lane);
  const u32x4 ba = buffer_over(g.sa + m0, (int64_t)p.nk * g.sa_ld - m0);
  const u32x4 bb = SQUARE ? buffer_over(g.sb + tn * g.sb_r, (int64_t)(p.nk - 1) * g.sb_k + 1) : buffer_over(g.sb + n0, (int64_t)p.nk * g.sb_k - n0);
  const uint32_t lds = lds_address(smem);
  const int per_step = wave < 2 ? 9 : 8;  // loads of this wave
  auto step_block = [&](int s) { return MODE == kFp8Dsd ? __builtin_amdgcn_readfirstlane((int)(list[s] & 0xffffu)) : lo + s; };
  auto load = [&](int s) {
    const int k = step_block(s);
    const uint32_t at = lds + (uint32_t)(s % STAGES) * kMidStage;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      la.load(wave * 4 + q, k, at);
      lb.load(wave * 4 + q, k, at + kBlockBytes);
    }
    if (wave == 0) buffer4_to_lds(ba, (uint32_t)((int64_t)k * g.sa_ld) + (lane & 31) * 4, at + 2 * kBlockBytes);
    if (wave == 1) {
      if (SQUARE) buffer1_to_lds(bb, (uint32_t)((int64_t)k * g.sb_k), at + 2 * kBlockBytes + 512);
      else buffer4_to_lds(bb, (uint32_t)((int64_t)k * g.sb_k) + (lane & 31) * 4, at + 2 * kBlockBytes + 512);
    }
  };
  f32x4 acc[4][4] = {};
  for (int s = 0; s < STAGES - 1 && s < steps; ++s) load(s);
  for (int s = 0; s < steps; ++s) {
    wait_loads_all_but(per_step * min(STAGES - 2, steps - 1 - s));
    barrier();
    if (s + STAGES - 1 < steps) load(s + STAGES - 1);  // (into the stage of step s - 1, which every wave is done with)
    const char* st = smem + (s % STAGES) * kMidStage;
    const char* scales = st + 2 * kBlockBytes;
    const int sa = *reinterpret_cast<const int*>(scales + 64 * wm + 4 * (lane & 15));
    int sb = *reinterpret_cast<const int*>(scales + 512 + (SQUARE ? 0 : 64 * wn + 4 * (lane & 15)));
    if (SQUARE) sb *= 0x01010101;
    i32x8 fa[4], fb[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      fa[i] = read_fragment(st + wm * 64 * kB, i, lane);
      fb[i] = read_fragment(st + kBlockBytes + wn * 64 * kB, i, lane);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = mfma(fa[i], fb[j], acc[i][j], sa, i, sb, j);
    wait_reads();  // (before the stage that was read is loaded over, behind the next barrier)
  }
  store_patch<T>(g, m0 + 64 * wm, n0 + 64 * wn, acc, out_part, lane);
}

template <typename T, int MODE, bool SQUARE, int STAGES>
__global__ __launch_bounds__(256, STAGES == 2 ? 2 : 1) void fp8_mid_kernel(Args p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  mid_tile<T, MODE, SQUARE, STAGES>(p, (int)blockIdx.x, smem);
}

// Both gradients of a layer in one launch, the weight gradient's workgroups behind the input gradient's.
template <typename T, int STAGES>
__global__ __launch_bounds__(256, STAGES == 2 ? 2 : 1) void fp8_pair_kernel(Args x, Args w, int first_w) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  if ((int)blockIdx.x < first_w) mid_tile<T, kFp8Sdd, true, STAGES>(x, (int)blockIdx.x, smem);
  else mid_tile<T, kFp8Dsd, false, STAGES>(w, (int)blockIdx.x - first_w, smem);
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

struct Plan {
  int splits, per_split;
};
Plan plan(int64_t M, int64_t N, int64_t K, int mode) {
  const int64_t nk = ceil_div(K, kB), tiles = ceil_div(M, kB) * ceil_div(N, kB);
  int64_t splits = 1;
  if (mode != kFp8Sdd) {
    while (tiles * splits < 256 && nk / (splits * 2) >= 4) splits *= 2;
  }
  if (mode == kFp8Dsd && ceil_div(nk, splits) > kMaxList) splits = ceil_div(nk, kMaxList);
  const int64_t per = ceil_div(nk, splits > 0 ? splits : 1);
  return {(int)ceil_div(nk, per), (int)per};
}

int64_t blocks_of(const Args& p) { return (int64_t)p.tiles_m * p.tiles_n * p.splits; }

template <typename T>
int launch_sum(const Args& p, hipStream_t stream) {
  if (p.splits <= 1) return SD_OK;
  hipLaunchKernelGGL(&fp8_sum_kernel<T>, dim3((unsigned)ceil_div(p.g.M * p.g.N, 1024)), dim3(256), 0, stream, p.g, p.splits);
  return check_launch("fp8_sum");
}

template <typename T, int MODE, int STAGES>
int launch_mid(const Args& p, hipStream_t stream) {
  auto* kernel = p.g.sb_square ? &fp8_mid_kernel<T, MODE, true, STAGES> : &fp8_mid_kernel<T, MODE, false, STAGES>;
  static std::atomic<bool> configured[2][16] = {};
  if (int rc = configure(reinterpret_cast<const void*>(kernel), configured[p.g.sb_square])) return rc;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks_of(p)), dim3(256), mid_lds(STAGES, MODE == kFp8Dsd ? p.per_split : 0), stream, p);
  note_kernel("fp8:mid stages=%d splits=%d", STAGES, p.splits);
  return check_launch("fp8_gemm");
}

// Four stages where every workgroup has a CU to itself and more than two steps
bool deep(int64_t blocks, const Args& p) { return blocks <= kCus && p.per_split > 2; }

template <typename T, int MODE>
int launch(const Args& p, hipStream_t stream) {
  if (blocks_of(p) >= (1LL << 31)) return fail(SD_ERR_UNSUPPORTED, "fp8 product: %lld tiles are too many for one launch", (long long)blocks_of(p));
  if (int rc = deep(blocks_of(p), p) ? launch_mid<T, MODE, 4>(p, stream) : launch_mid<T, MODE, 2>(p, stream)) return rc;
  return launch_sum<T>(p, stream);
}

template <typename T, int STAGES>
int launch_pair(const Args& x, const Args& w, hipStream_t stream) {
  auto* kernel = &fp8_pair_kernel<T, STAGES>;
  static std::atomic<bool> configured[16] = {};
  if (int rc = configure(reinterpret_cast<const void*>(kernel), configured)) return rc;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(blocks_of(x) + blocks_of(w))), dim3(256), mid_lds(STAGES, w.per_split), stream, x, w, (int)blocks_of(x));
  note_kernel("fp8:pair stages=%d splits=%d", STAGES, w.splits);
  if (int rc = check_launch("fp8_pair")) return rc;
  return launch_sum<T>(w, stream);
}

int make_args(const Fp8Gemm& g, int mode, Args& p) {
  p.g = g;
  const Plan q = plan(g.M, g.N, g.K, mode);
  p.nk = (int)ceil_div(g.K, kB);
  p.splits = q.splits;
  p.per_split = q.per_split;
  if (p.splits > 1 && (g.part == nullptr || g.part_bytes < (int64_t)p.splits * g.M * g.N * 4)) {
    if (mode == kFp8Dsd && p.nk > kMaxList) return fail(SD_ERR_INVALID, "fp8 product: a reduction of %d blocks needs its scratch", p.nk);
    p.splits = 1;
    p.per_split = p.nk;
  }
  p.tiles_m = (int)ceil_div(g.M, kB);
  p.tiles_n = (int)ceil_div(g.N, kB);
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
  if (!gx.sb_square || gw.sb_square || blocks > kPairBlocks) {
    if (int rc = launch_fp8_gemm(gx, kFp8Sdd, dtype, stream)) return rc;
    return launch_fp8_gemm(gw, kFp8Dsd, dtype, stream);
  }
  const bool four = deep(blocks, x) || deep(blocks, w);
  if (dtype == SD_BF16) return four ? launch_pair<BF16, 4>(x, w, stream) : launch_pair<BF16, 2>(x, w, stream);
  return four ? launch_pair<F16, 4>(x, w, stream) : launch_pair<F16, 2>(x, w, stream);
}

}  // namespace sd
