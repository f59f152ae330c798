// AdamW over many tensors in few launches, the two averages held in 32 or in 8 bits.
//
//   m = beta1 m + (1 - beta1) g        v = beta2 v + (1 - beta2) g^2
//   p = p (1 - lr decay) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
//
// Bound by the bytes of parameters, gradients and averages: 28 an element in 32 bits throughout, 16 with averages in 8.  Tensors of any
// number go by tables of kTensors in the launch's arguments, a workgroup takes runs of elements off the whole of them.
//
// Averages in 8 bits have a power of two for each block of 128 elements.  The first is e4m3; the second, which has no sign, has five
// bits of exponent and three of mantissa, so that 2^34 lies between its least and its largest number: a second average that is small
// in its block must not come out as zero, for its element would then move by m / eps.  An average moves by (1 - beta) of the way a
// step, a thousandth for the second, which is less than half of the 2^-3 between two numbers: rounded to nearest it would never move.
// So it is rounded at random, up with the probability that its place between the two numbers says, and stays right on average.  The random
// bits are a function of step and element alone: equal runs have equal states.  The averages are computed in 64 bits before that,
// since whether a value lies below or above its random border must not depend on how the compiler orders 32-bit arithmetic.
#include "fp8.h"

#include <cfloat>

namespace sd {
namespace {

constexpr int kThreads = 256, kWide = 1024;  // of a workgroup, few and many
constexpr int kTensors = 56;
constexpr int kPer = 8;                    // elements of a thread at a time
constexpr int kChunk = kThreads * kPer;    // what the tables count in: whole 128-blocks

struct AdamTensor {
  void* p;
  const void* g;
  void *m, *v;
  uint8_t *ms, *vs;
  int64_t n;
};
struct AdamTable {
  AdamTensor tensor[kTensors];
  uint32_t first[kTensors + 1];  // chunk of the launch that a tensor begins at
  int32_t n;
  int64_t* step;
  int32_t last;  // of the call's launches: moves the step on
  const float* lr_at;
  double lr, beta1, beta2, eps, decay;
};
static_assert(sizeof(AdamTable) <= 4096, "a launch's arguments");

struct F32 {
  typedef float elem;
  static constexpr int id = kF32;
  __device__ static inline float to_float(float v) { return v; }
  __device__ static inline float from_float(float v) { return v; }
};

template <typename T>
struct Elem {
  typedef uint16_t type;
};
template <>
struct Elem<F32> {
  typedef float type;
};

// base^t by squaring; its relative error grows with t as t * 2^-53
__device__ inline double power(double base, uint32_t t) {
  double r = 1.0;
  for (; t; t >>= 1) {
    if (t & 1) r *= base;
    base *= base;
  }
  return r;
}

// a wa + b wb, each product and the sum rounded by itself, as elementary operations round them (see encode_border)
__device__ inline double weighted(double a, double wa, double b, double wb) {
#pragma clang fp contract(off)
  const double x = a * wa, y = b * wb;
  return x + y;
}

// M. O'Neill's permuted congruential generator, 32 bits, output function RXS-M-XS, one step behind x
__device__ inline uint32_t mixed(uint32_t x) {
  const uint32_t s = x * 747796405u + 2891336453u;
  const uint32_t w = ((s >> ((s >> 28) + 4)) ^ s) * 277803737u;
  return (w >> 22) ^ w;
}

template <typename E>
__device__ inline void load_run(const E* src, int left, float (&out)[kPer]);
template <>
__device__ inline void load_run<float>(const float* src, int left, float (&out)[kPer]) {
  typedef f32x4 __attribute__((aligned(4))) f32x4_any;
  if (left >= kPer) {
    const f32x4 a = *reinterpret_cast<const f32x4_any*>(src), b = *reinterpret_cast<const f32x4_any*>(src + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      out[i] = a[i];
      out[4 + i] = b[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) out[i] = i < left ? src[i] : 0.f;
  }
}
template <typename T>
__device__ inline void load_typed(const void* src, int64_t at, int left, float (&out)[kPer]) {
  if constexpr (T::id == kF32) {
    load_run<float>(static_cast<const float*>(src) + at, left, out);
  } else {
    const uint16_t* s = static_cast<const uint16_t*>(src) + at;
    if (left >= kPer) {
      const u32x4 w = *reinterpret_cast<const u32x4_any*>(s);
#pragma unroll
      for (int i = 0; i < kPer; ++i) out[i] = T::to_float((uint16_t)(i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu));
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i) out[i] = i < left ? T::to_float(s[i]) : 0.f;
    }
  }
}
template <typename T>
__device__ inline void store_typed(void* dst, int64_t at, int left, const float (&v)[kPer]) {
  if constexpr (T::id == kF32) {
    typedef f32x4 __attribute__((aligned(4))) f32x4_any;
    float* d = static_cast<float*>(dst) + at;
    if (left >= kPer) {
      *reinterpret_cast<f32x4_any*>(d) = f32x4{v[0], v[1], v[2], v[3]};
      *reinterpret_cast<f32x4_any*>(d + 4) = f32x4{v[4], v[5], v[6], v[7]};
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (i < left) d[i] = v[i];
    }
  } else {
    uint16_t* d = static_cast<uint16_t*>(dst) + at;
    if (left >= kPer) {
      *reinterpret_cast<u32x4_any*>(d) = u32x4{T::pack2(v[0], v[1]), T::pack2(v[2], v[3]), T::pack2(v[4], v[5]), T::pack2(v[6], v[7])};
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (i < left) d[i] = T::from_float(v[i]);
    }
  }
}
// eight codes
typedef u32x2 __attribute__((aligned(1))) u32x2_any;
__device__ inline u32x2 load_codes(const uint8_t* src, int left) {
  if (left >= kPer) return *reinterpret_cast<const u32x2_any*>(src);
  u32x2 w = {0u, 0u};
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (i < left) w[i / 4] |= (uint32_t)src[i] << (8 * (i % 4));
  return w;
}
__device__ inline void store_codes(uint8_t* dst, int left, u32x2 w) {
  if (left >= kPer) {
    *reinterpret_cast<u32x2_any*>(dst) = w;
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (i < left) dst[i] = (uint8_t)(w[i / 4] >> (8 * (i % 4)));
  }
}

// ---- the two formats ------------------------------------------------------------------------------------------------------
// 8 bits of a magnitude: exponent behind the bias, three bits of mantissa.  LIMIT20: the upper 20 bits of the largest number's mantissa,
// TOP its exponent.
struct First {
  static constexpr int bias = 7, least = -6, top = 8;
  static constexpr uint32_t limit20 = 0xC0000u;  // 448 = 1.75 * 2^8
  static constexpr uint32_t infinite = 0x7f, nan = 0x7f;  // (e4m3 has no infinity)
  __device__ static inline float decode(u32x2 w, int i) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const int word = (int)w[i / 4];
    const f32x2 pair = i & 2 ? __builtin_amdgcn_cvt_pk_f32_fp8(word, true) : __builtin_amdgcn_cvt_pk_f32_fp8(word, false);
    return pair[i & 1];
  }
};
struct Second {
  static constexpr int bias = 15, least = -14, top = 15;
  static constexpr uint32_t limit20 = 0xE0000u;  // 61440 = 1.875 * 2^15
  static constexpr uint32_t infinite = 0xf8, nan = 0xff;
  __device__ static inline float decode(u32x2 w, int i) {  // an fp16 without its sign and its last seven bits
    return F16::to_float((uint16_t)(((w[i / 4] >> (8 * (i % 4))) & 0xffu) << 7));
  }
};

// What decides a block's scale, as a number that grows with the magnitude: the upper half of its 64 bits, with the lower half's
// being other than zero in the last.  0 for what is not finite in 32 bits.
__device__ inline uint32_t magnitude_word(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x) & 0x7fffffffffffffffull;
  const uint32_t hi = (uint32_t)(b >> 32), w = hi | ((uint32_t)b != 0u ? 1u : 0u);
  return w < ((1023u + 128u) << 20) ? w : 0u;
}
// the byte of the least power of two with which `word` stays within the largest number
template <typename Format>
__device__ inline uint32_t scale_byte(uint32_t word) {
  const int e = (int)(word >> 20) - 1023 - Format::top + ((word & 0xfffffu) > Format::limit20 ? 1 : 0) + 127;
  return word == 0u ? 127u : (uint32_t)(e < 0 ? 0 : e);
}
// Where |x| and the random bits make a border but for the last few of 64 bits, the code is what the formula gives in torch, step by step:
// torch.ldexp multiplies by pow(2, k), which for some k is an ulp below 2^k on this hardware.  (Weights like 0.9 and 0.1 make such sums of
// one element in 10^7, where 9 m + g is a multiple of ten of its last places; equal formulas have equal states with this.)
template <typename Format>
__device__ inline uint32_t encode_border(double x, uint32_t byte, uint32_t random, const double* powers) {
#pragma clang fp contract(off)
  const double y = fabs(x) * powers[254u - byte];
  const int exponent = (int)((uint32_t)(__builtin_bit_cast(uint64_t, y) >> 52) & 0x7ffu) - 1023, at = max(exponent, Format::least);
  const double steps = y * powers[127 + 3 - at], up = (double)random * 0x1p-16;
  return (uint32_t)(steps + up) + (at > Format::least ? (uint32_t)(at + Format::bias - 1) * 8u : 0u);
}
// |x| / 2^(byte - 127) rounded down after random / 2^16 of the distance to the next number was added: whole numbers without a branch.  In
// 2^16 parts of a step the number is `parts` and `rest` / 2^32.  rare: it is next to a border, or not finite (encode_rare).
template <typename Format>
__device__ inline uint32_t encode(double x, uint32_t byte, uint32_t random, bool& rare) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint32_t hi = (uint32_t)(b >> 32) & 0x7fffffffu, lo = (uint32_t)b;
  const int exponent = (int)(hi >> 20) - 1023 - ((int)byte - 127), above = exponent - Format::least;
  const uint32_t shift = (uint32_t)min(1 - min(above, 0), 31), mantissa = (hi & 0xfffffu) | 0x100000u;
  const uint32_t parts = (mantissa >> shift) + random, rest = (mantissa << (32u - shift)) | (lo >> shift);
  rare = (rest + 4u < 8u && ((parts + (rest >> 31)) & 0xffffu) == 0u) || hi >= (1023u + 128u) << 20;
  return ((parts >> 16) + (uint32_t)max(above, 0) * 8u) & 0xffu;  // (of a rare one anything)
}
template <typename Format>
__device__ inline uint32_t encode_rare(double x, uint32_t byte, uint32_t random, const double* powers) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x) & 0x7fffffffffffffffull;
  if (b > 0x7ff0000000000000ull) return Format::nan;
  if (b >= (uint64_t)(1023u + 128u) << 52) return Format::infinite;
  return encode_border<Format>(x, byte, random, powers);
}

// m / (sqrt(v) root + eps), of 32 bits' roundings six off at most: the hardware's root and reciprocal are one unit of the last place off
// (2 roundings each, of numbers that are not subnormal: such v are scaled by 2^24 before it; eps is 0 or from 2^-126 to 2^120, sqrt(v) root
// ends below 2^96).  The exact root and division take 27 instructions instead of 8,
// 694 us instead of 645 for 168 M fp32 parameters.
__device__ inline float moved(float m, float v, float root, float eps) {
  const bool tiny = v < 0x1p-126f;
  return m * __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(v * (tiny ? 0x1p24f : 1.f)) * (tiny ? root * 0x1p-12f : root) + eps);
}

template <typename T, int BITS, int THREADS>
__global__ __launch_bounds__(THREADS) void adamw_kernel(AdamTable a) {
  constexpr int PART = THREADS / kThreads;  // chunks that a workgroup takes at a time
  const int part = PART == 1 ? 0 : __builtin_amdgcn_readfirstlane((int)threadIdx.x / kThreads), lane = (int)threadIdx.x % kThreads;
  __shared__ double powers[BITS == 8 ? 256 : 1];
  if constexpr (BITS == 8) {
    if (threadIdx.x < 256) powers[threadIdx.x] = pow(2.0, (double)((int)threadIdx.x - 127));
    __syncthreads();
  }
  float by = 0.f, root = 0.f, keep = 0.f;
  const float eps = (float)a.eps;
  bool known = false;
  uint32_t t = 0u, key = 0u;
  const uint32_t chunks = a.first[a.n];
  int which = 0;
  // (with no elements at all one workgroup runs, to move the step on: through an empty piece of an empty tensor)
  for (uint32_t chunk = blockIdx.x * PART + part; chunk < chunks || !known; chunk += gridDim.x * PART) {
    while (chunk >= a.first[which + 1] && which + 1 < a.n) ++which;
    const AdamTensor& x = a.tensor[which];
    const int64_t at = (int64_t)(chunk - a.first[which]) * kChunk + lane * kPer;
    const int64_t rest = x.n - at;
    const int left = rest < 0 ? 0 : rest > kPer ? kPer : (int)rest;
    float p[kPer], g[kPer];
    load_typed<T>(x.p, at, left, p);
    load_typed<T>(x.g, at, left, g);
    // the step's factors, worked out while the first loads are on their way
    auto factors = [&] {
      if (known) return;
      t = (uint32_t)__builtin_amdgcn_readfirstlane((int)*reinterpret_cast<const volatile uint32_t*>(a.step)) + 1u;
      const double lr = a.lr_at ? (double)*a.lr_at : a.lr;
      by = (float)(lr / (1.0 - power(a.beta1, t)));
      root = (float)(1.0 / sqrt(1.0 - power(a.beta2, t)));
      keep = (float)(1.0 - lr * a.decay);
      key = t * 0x9E3779B1u;
      known = true;
    };
    if constexpr (BITS == 32) {
      float m[kPer], v[kPer];
      load_run<float>(static_cast<const float*>(x.m) + at, left, m);
      load_run<float>(static_cast<const float*>(x.v) + at, left, v);
      factors();
      const float b1 = (float)a.beta1, c1 = (float)(1.0 - a.beta1), b2 = (float)a.beta2, c2 = (float)(1.0 - a.beta2);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        m[i] = m[i] * b1 + g[i] * c1;
        v[i] = v[i] * b2 + (g[i] * g[i]) * c2;
        p[i] = p[i] * keep - by * (m[i] / (sqrtf(v[i]) * root + eps));
      }
      store_typed<F32>(x.m, at, left, m);
      store_typed<F32>(x.v, at, left, v);
      store_typed<T>(x.p, at, left, p);
    } else {
      const int64_t block = at / 128;
      uint8_t *const mc = static_cast<uint8_t*>(x.m) + at, *const vc = static_cast<uint8_t*>(x.v) + at;
      u32x2 mw = load_codes(mc, left), vw = load_codes(vc, left);
      const float ms = fp8_power(left ? x.ms[block] : 127u), vs = fp8_power(left ? x.vs[block] : 127u);
      factors();
      double m[kPer], v[kPer];
      uint32_t m_most = 0, v_most = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const double gd = (double)g[i];
        m[i] = weighted((double)(First::decode(mw, i) * ms), a.beta1, gd, 1.0 - a.beta1);
        v[i] = weighted((double)(Second::decode(vw, i) * vs), a.beta2, gd * gd, 1.0 - a.beta2);
        m_most = max(m_most, magnitude_word(m[i]));
        v_most = max(v_most, magnitude_word(v[i]));
        p[i] = p[i] * keep - by * moved((float)m[i], (float)v[i], root, eps);
        __builtin_amdgcn_sched_barrier(0);
      }
      store_typed<T>(x.p, at, left, p);
      // sixteen lanes hold a block (those behind the tensor's end hold zeros)
      const uint32_t mb = scale_byte<First>(max_of_row16(m_most)), vb = scale_byte<Second>(max_of_row16(v_most));
      mw = u32x2{0u, 0u};
      vw = u32x2{0u, 0u};
      uint32_t rare = 0u;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const uint32_t random = mixed(key + (uint32_t)at + i);
        const uint32_t sign = (uint32_t)(__builtin_bit_cast(uint64_t, m[i]) >> 56) & 0x80u;
        bool rare_m, rare_v;
        const uint32_t mq = encode<First>(m[i], mb, random >> 16, rare_m) | sign, vq = encode<Second>(v[i], vb, random & 0xffffu, rare_v);
        mw[i / 4] |= mq << (8 * (i % 4));
        vw[i / 4] |= vq << (8 * (i % 4));
        rare |= (rare_m ? 1u : 0u) << i | (rare_v ? 256u : 0u) << i;
        __builtin_amdgcn_sched_barrier(0);  // (interleaved, the eight take more registers than four waves a SIMD have)
      }
      while (rare) {  // (one at a time: written out eight times it takes twice the registers)
        const int bit = __builtin_ctz(rare), i = bit & 7;
        rare &= rare - 1u;
        double z = bit < 8 ? m[0] : v[0];
#pragma unroll
        for (int j = 1; j < kPer; ++j) z = bit == j ? m[j] : bit == 8 + j ? v[j] : z;
        const uint32_t random = mixed(key + (uint32_t)at + i), sign = (uint32_t)(__builtin_bit_cast(uint64_t, z) >> 56) & 0x80u;
        const uint32_t q = bit < 8 ? encode_rare<First>(z, mb, random >> 16, powers) | sign : encode_rare<Second>(z, vb, random & 0xffffu, powers);
        const uint32_t hole = ~(0xffu << (8 * (i % 4))), piece = q << (8 * (i % 4));
        if (bit < 4) mw[0] = (mw[0] & hole) | piece;
        else if (bit < 8) mw[1] = (mw[1] & hole) | piece;
        else if (bit < 12) vw[0] = (vw[0] & hole) | piece;
        else vw[1] = (vw[1] & hole) | piece;
      }
      store_codes(mc, left, mw);
      store_codes(vc, left, vw);
      if ((threadIdx.x & 15) == 0 && left) {
        x.ms[block] = (uint8_t)mb;
        x.vs[block] = (uint8_t)vb;
      }
    }
  }
  // The step moves on when every workgroup is done with it: the last to report writes it.  Its upper half counts the reports meanwhile, one
  // at a time, 10 ns each where they are few; 2048 take 126 us more than 512 (launch_table).  (Made at the start they hold up the others' reads of the step: 58 us for 1.9 M parameters, at the end 19.
  // A launch that moves the step on takes 4 us.)
  if (a.last) {
    __syncthreads();
    if (threadIdx.x == 0 && atomicAdd(reinterpret_cast<uint32_t*>(a.step) + 1, 1u) == gridDim.x - 1) {
      *(reinterpret_cast<uint32_t*>(a.step) + 1) = 0u;
      *reinterpret_cast<uint32_t*>(a.step) = t;
    }
  }
}

struct ValueTensor {
  const uint8_t *codes, *scales;
  float* out;
  int64_t n;
  int32_t second;
};
struct ValueTable {
  ValueTensor tensor[kTensors];
  uint32_t first[kTensors + 1];
  int32_t n;
};
static_assert(sizeof(ValueTable) <= 4096, "a launch's arguments");

// averages in 8 bits -> their values in 32, four a thread at a time so that a wave's stores are whole lines.  Bound by what it writes.
__global__ __launch_bounds__(kThreads) void state_values_kernel(ValueTable a) {
  const uint32_t chunks = a.first[a.n];
  int which = 0;
  for (uint32_t chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    while (chunk >= a.first[which + 1]) ++which;
    const ValueTensor& x = a.tensor[which];
#pragma unroll
    for (int h = 0; h < kPer / 4; ++h) {
      const int64_t at = (int64_t)(chunk - a.first[which]) * kChunk + (h * kThreads + threadIdx.x) * 4, rest = x.n - at;
      if (rest <= 0) continue;
      const float s = fp8_power(x.scales[at / 128]);
      u32x2 w = {0u, 0u};
      if (rest >= 4) {
        typedef uint32_t __attribute__((aligned(1))) u32_any;
        w[0] = *reinterpret_cast<const u32_any*>(x.codes + at);
      } else {
        for (int i = 0; i < rest; ++i) w[0] |= (uint32_t)x.codes[at + i] << (8 * i);
      }
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = (x.second ? Second::decode(w, i) : First::decode(w, i)) * s;
      if (rest >= 4) {
        typedef f32x4 __attribute__((aligned(4))) f32x4_any;
        *reinterpret_cast<f32x4_any*>(x.out + at) = f32x4{v[0], v[1], v[2], v[3]};
      } else {
#pragma unroll
        for (int i = 0; i < 3; ++i)
          if (i < rest) x.out[at + i] = v[i];
      }
    }
  }
}

// workgroups: as many as are resident, each through several chunks
unsigned grid_of(uint32_t chunks) { return chunks < 2048 ? chunks : 2048; }

// Workgroups of 1024 threads where their number matters, for they report one after the other, and not where everything is done at once (too few
// of them for all CUs).  With averages in 8 bits, whose arithmetic is what takes the time in the end, not for long tables either.  us with 256 threads
// and with 1024, by runs of 2048 elements:
//   32 bits, fp32   100: 5.6, 6.6   200: 7.3, 7.1   300: 9.0, 7.7   2048: 170, 44   8192: 207, 101   32768: 406, 375   81920: 925, 927
//   32 bits, bf16   100: 6.3, 7.0   200: 7.7, 7.6   300: 9.0, 8.0   2048: 148, 26   8192: 138, 77    32768: 309, 300   81920: 733, 728
//   8 bits, fp32    256: 10.4, 12.3   512: 13.8, 13.8   700: 16.7, 15.2   8192: 130, 77   16384: 158, 139   24576: 199, 199   65536: 477, 490
//   8 bits, bf16    256: 10.0, 12.3   512: 13.7, 13.5   700: 15.8, 13.9   8192: 93, 68    16384: 125, 124   24576: 178, 193   65536: 458, 489
template <typename T>
void launch_table(const AdamTable& a, int bits, uint32_t chunks, hipStream_t stream) {
  const bool wide = bits == 8 ? chunks > 512 && chunks <= 16384 : chunks >= 256;
  const dim3 grid(wide ? (chunks + 3) / 4 < 512 ? (chunks + 3) / 4 : 512 : chunks ? grid_of(chunks) : 1), block(wide ? kWide : kThreads);
  if (bits == 8) hipLaunchKernelGGL((wide ? &adamw_kernel<T, 8, kWide> : &adamw_kernel<T, 8, kThreads>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((wide ? &adamw_kernel<T, 32, kWide> : &adamw_kernel<T, 32, kThreads>), grid, block, 0, stream, a);
}

}  // namespace

int launch_adamw(int count, void* const* p, const void* const* g, void* const* m, void* const* v, uint8_t* const* ms, uint8_t* const* vs,
                 const int64_t* n, int64_t* step, const float* lr_at, double lr, double beta1, double beta2, double eps, double decay,
                 int dtype, int bits, bool moves_on, hipStream_t stream) {
  AdamTable a = {};
  a.step = step;
  a.lr_at = lr_at;
  a.lr = lr;
  a.beta1 = beta1;
  a.beta2 = beta2;
  a.eps = eps;
  a.decay = decay;
  for (int i = 0; i < count || (i == 0 && moves_on);) {
    a.n = 0;
    a.first[0] = 0;
    int64_t chunks = 0;
    for (; i < count && a.n < kTensors; ++i) {
      const int64_t more = ceil_div(n[i], kChunk);
      if (chunks + more >= (1LL << 31)) break;
      if (more == 0) continue;
      a.tensor[a.n] = AdamTensor{p[i], g[i], m[i], v[i], ms ? ms[i] : nullptr, vs ? vs[i] : nullptr, n[i]};
      chunks += more;
      a.first[++a.n] = (uint32_t)chunks;
    }
    if (i < count && a.n == 0) return fail(SD_ERR_UNSUPPORTED, "adamw_step: a tensor of %lld elements is too large", (long long)n[i]);
    a.last = moves_on && i == count ? 1 : 0;
    if (chunks == 0 && !a.last) break;
    if (chunks == 0) a.tensor[0] = AdamTensor{};
    if (dtype == kF32) launch_table<F32>(a, bits, (uint32_t)chunks, stream);
    else if (dtype == SD_BF16) launch_table<BF16>(a, bits, (uint32_t)chunks, stream);
    else launch_table<F16>(a, bits, (uint32_t)chunks, stream);
    if (int rc = check_launch("adamw_step")) return rc;
    if (i == count) break;
  }
  return SD_OK;
}

int launch_state_values(int count, const uint8_t* const* codes, const uint8_t* const* scales, float* const* out, const int64_t* n,
                        const int32_t* second, hipStream_t stream) {
  ValueTable a = {};
  for (int i = 0; i < count;) {
    a.n = 0;
    a.first[0] = 0;
    int64_t chunks = 0;
    for (; i < count && a.n < kTensors; ++i) {
      const int64_t more = ceil_div(n[i], kChunk);
      if (chunks + more >= (1LL << 31)) break;
      if (more == 0) continue;
      a.tensor[a.n] = ValueTensor{codes[i], scales[i], out[i], n[i], second[i]};
      chunks += more;
      a.first[++a.n] = (uint32_t)chunks;
    }
    if (i < count && a.n == 0) return fail(SD_ERR_UNSUPPORTED, "adamw_state_values: a tensor of %lld elements is too large", (long long)n[i]);
    if (chunks == 0) break;
    hipLaunchKernelGGL(&state_values_kernel, dim3(grid_of((uint32_t)chunks)), dim3(kThreads), 0, stream, a);
    if (int rc = check_launch("adamw_state_values")) return rc;
  }
  return SD_OK;
}

}  // namespace sd
