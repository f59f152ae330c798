// A gate's arithmetic, h = act(g) u and its gradients, and the stores of the products that carry it.
//
// Forward.  Both projections are one product with W_in [2 F, K], whose columns a workgroup takes 16 of the gate and the same 16 of the other
// projection at a time: 16-column tile 2 q of its output is g, tile 2 q + 1 is u of the hidden columns 16 q .. + 15.  Either tile of a pair is
// in the same registers of the same lanes, so H needs nothing from another wave, and where nothing will be differentiated G and U never leave the
// registers: 3 of the 4 bytes a passing gate would move.  gated_hidden, gated_up: which row of W_in column n of a tile is.
//   8192 x 2048 to 8192 bf16: 408 us, 447 with G and U; the product alone, which writes both, 419 to 425, and a gate's pass 73 more (with the clock
//   settled; 415 to 437 in a block, card by card)
//   4096 x 1024 to 4096 fp16:  66 us,  69;              66 and 16            1024 x 512 to 2048: 10.8, 12.7; 10.8 and 3.6
// Bound by the matrix cores and the loads into LDS as the ungated product is; at the largest the store of 2 or 6 bytes an element adds to that (360 us
// without one).  Workgroups of the first round started up to 13 us apart, so that no two CUs' stores meet, take the same: it is not that they come together.
//
// Backward.  dH = (dY W_out) . keep is a product whose store reads g and u of its place and writes dg and du instead of dh.
//   8192 x 8192 from 2048 bf16: 336 us, the product and a pass 233 and 120; half dropped 235, 163 and 121 (243 in a block)
//   4096 x 4096 from 1024 fp16: 55 us, 37 and 26           1024 x 2048 from 512: 9.3, 7.3 and 4.9
// Bound by the product and behind it by the 8 bytes read and written for each of its results: the gate saves dH's way to memory and back and a
// launch.  (With nontemporal loads or stores, in either direction, a block's 372 us were 373 to 395, another's 1432 1421 to 1442.)
#pragma once
#include "common.h"

namespace sd {

// act(g).  SILU: g / (1 + exp(-g)), one exponential and one reciprocal.  Within 2^-19 of itself where |g| < 16: what rounds g / ln 2, by up to 2^-20 there,
// moves the exponential by 0.7 times that, the constant by |g| 2^-26, and each of the other steps by 2^-24 or 2^-23; beyond it grows with -g.  An exponential
// of 2^126 and more gives 0 for a value under 2^-119.  NaN stays NaN in every gate (ReLU's comparison is the one that it fails).
__device__ inline float gate_value(int act, float g) {
  if (act == SD_ACT_SILU) return g * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(g * -1.4426950408889634f));
  if (act == SD_ACT_RELU) return g <= 0.f ? 0.f : g;
  return act_apply(act, g);
}
// act(g) and act'(g) together: they share what is dear.  GELU: Phi(g) from the root of its tail, phi(g) one exponential more.  ReLU': 0 or 1, or NaN.
// A G that was beyond its type has been kept as an infinity: there they are their limits, 0 and 0 below, infinite and 1 above.
__device__ inline void gate_slope(int act, float g, float& value, float& slope) {
  if (act == SD_ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(g * -1.4426950408889634f)), rest = 1.f - s;
    value = s != 0.f ? g * s : 0.f;
    slope = rest != 0.f ? __builtin_fmaf(value, rest, s) : s;
  } else if (act == SD_ACT_GELU) {
    const float root = normal_tail_root(fabsf(g)), below = g >= 0.f ? __builtin_fmaf(-root, root, 1.f) : root * root;
    const float bell = __builtin_amdgcn_exp2f((g * -0.72134752044448170f) * g);
    value = below != 0.f ? g * below : 0.f;
    slope = bell != 0.f ? __builtin_fmaf(g * 0.39894228040143268f, bell, below) : below;
  } else {
    value = gate_value(act, g);
    slope = g > 0.f ? 1.f : value;
  }
}
// dG = d U act'(G) and dU = d act(G) in the places of G and U; d: of H.  A U that was beyond its type is an infinity too, and nothing behind a slope of 0.
// Where d is 0 so are both: what was dropped has no gradient, whatever stands there.
__device__ inline void gate_gradient(int act, float d, float& gate, float& up) {
  float value, slope;
  gate_slope(act, gate, value, slope);
  const float u = slope == 0.f && __builtin_isinf(up) ? 0.f : up;
  gate = d != 0.f ? d * u * slope : 0.f;
  up = d != 0.f ? d * value : 0.f;
}

// columns of the product's output as its tiles see them
__host__ __device__ inline int64_t gated_columns(int64_t F) { return (F + 15) / 16 * 32; }
// hidden column of column n, from the first of a tile, and whether it is the other projection's
__device__ inline int gated_hidden(int n) { return n / 32 * 16 + n % 16; }
__device__ inline bool gated_up(int n) { return (n & 16) != 0; }

template <typename T>
__device__ inline u32x4 pack_eight(const float (&v)[8]) {
  return u32x4{T::pack2(v[0], v[1]), T::pack2(v[2], v[3]), T::pack2(v[4], v[5]), T::pack2(v[6], v[7])};
}
template <typename T>
__device__ inline void unpack_eight(u32x4 w, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = T::to_float((uint16_t)(i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu));
}

// N hidden columns from column c of row m on, unscaled fp32 accumulators of both projections
template <typename T, int N>
__device__ inline void store_gate(const GemmArgs& g, int64_t m, int64_t c, float (&gate)[N], float (&up)[N]) {
  if (m >= g.M || c >= g.c_cols) return;
  const int valid = g.gate - c < N ? (int)(g.gate - c) : N;
  uint16_t* h = g.c + m * g.c_sr + c;
  if (valid < N)  // zeros behind the last column
    for (int i = valid > 0 ? valid : 0; i < N && c + i < g.c_cols; ++i) h[i] = 0;
  if (valid <= 0) return;
  float out[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    gate[i] *= g.scale;
    up[i] *= g.scale;
  }
  auto apply = [&](int act) {
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = gate_value(act, gate[i]) * up[i];
  };
  if (g.act == SD_ACT_SILU) apply(SD_ACT_SILU);
  else if (g.act == SD_ACT_GELU) apply(SD_ACT_GELU);
  else apply(SD_ACT_RELU);
  auto put = [&](uint16_t* at, const float (&v)[N]) {
    if (valid < N) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < valid) at[i] = T::from_float(v[i]);
    } else if constexpr (N == 8) {
      *reinterpret_cast<u32x4_any*>(at) = pack_eight<T>(v);
    } else {
      static_assert(N == 4, "8 or 16 bytes");
      typedef u32x2 __attribute__((aligned(2))) u32x2_any;
      *reinterpret_cast<u32x2_any*>(at) = u32x2{T::pack2(v[0], v[1]), T::pack2(v[2], v[3])};
    }
  };
  if (g.aux) {
    uint16_t* a = g.aux + m * g.aux_sr + c;
    put(a, gate);
    put(a + g.aux_up, up);
  }
  put(h, out);
}

// A wave's tile [64 rows][32 gate and 32 other columns, 16 by 16] of accumulators staged in LDS with a pitch of 68 floats; c0: its first
// hidden column.
template <typename T>
__device__ inline void store_staged_gate(const GemmArgs& g, const float* stg, int lane, int64_t m0, int64_t c0) {
  constexpr int PITCH = 68;
#pragma unroll
  for (int pass = 0; pass < 4; ++pass) {
    const int row = pass * 16 + lane / 4, ch = lane % 4;
    const float* at = stg + row * PITCH + ch / 2 * 32 + ch % 2 * 8;
    float gate[8], up[8];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(at + 4 * i), b = *reinterpret_cast<const f32x4*>(at + 16 + 4 * i);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        gate[4 * i + e] = a[e];
        up[4 * i + e] = b[e];
      }
    }
    store_gate<T, 8>(g, m0 + row, c0 + ch * 8, gate, up);
  }
}

// What the gradient's store reads of a position, on its way ahead of the stores in front (see aux_eight); nothing where it does not take eight.
struct GateAt {
  u32x4 gate, up;
  __device__ inline void load(const GemmArgs& g, int64_t m, int64_t c) {
    gate = up = u32x4{0u, 0u, 0u, 0u};
    if (m >= g.M || c + 8 > g.gate) return;
    const uint16_t* at = g.aux + m * g.aux_sr + c;
    gate = *reinterpret_cast<const u32x4_any*>(at);
    up = *reinterpret_cast<const u32x4_any*>(at + g.aux_up);
  }
};
// zeros behind both gradients of row m (where F is no multiple of 8)
__device__ inline void fill_gradient(const GemmArgs& g, int64_t m) {
  for (int64_t i = 2 * g.gate; i < g.c_cols; ++i) g.c[m * g.c_sr + i] = 0;
}
// eight of dh, unscaled fp32 accumulators
template <typename T>
__device__ inline void store_gate_gradient(const GemmArgs& g, int64_t m, int64_t c, float (&dh)[8], const GateAt& pre) {
  if (m >= g.M || c >= g.gate) return;
  const int valid = g.gate - c < 8 ? (int)(g.gate - c) : 8;
  uint16_t* out = g.c + m * g.c_sr + c;
  float gate[8], up[8];
  if (valid == 8) {
    unpack_eight<T>(pre.gate, gate);
    unpack_eight<T>(pre.up, up);
  } else {
    const uint16_t* at = g.aux + m * g.aux_sr + c;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      gate[i] = i < valid ? T::to_float(at[i]) : 0.f;
      up[i] = i < valid ? T::to_float(at[g.aux_up + i]) : 0.f;
    }
  }
  auto apply = [&](int act) {
#pragma unroll
    for (int i = 0; i < 8; ++i) gate_gradient(act, dh[i] * g.scale, gate[i], up[i]);
  };
  if (g.act == SD_ACT_SILU) apply(SD_ACT_SILU);
  else if (g.act == SD_ACT_GELU) apply(SD_ACT_GELU);
  else apply(SD_ACT_RELU);
  if (valid == 8) {
    *reinterpret_cast<u32x4_any*>(out) = pack_eight<T>(gate);
    *reinterpret_cast<u32x4_any*>(out + g.c_up) = pack_eight<T>(up);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < valid) {
        out[i] = T::from_float(gate[i]);
        out[g.c_up + i] = T::from_float(up[i]);
      }
    fill_gradient(g, m);
  }
}
// A wave's 64 x 64 tile of dh staged in LDS with a pitch of 68 floats.  In two turns: all eight passes side by side are 96 KB of instructions in the
// 256 x 256 kernel, more than a CU's instruction cache holds.
template <typename T>
__device__ inline void store_staged_gate_gradient(const GemmArgs& g, const float* stg, int lane, int64_t m0, int64_t c0) {
  constexpr int PITCH = 68, AHEAD = 4;
#pragma unroll 1
  for (int first = 0; first < 8; first += AHEAD) {
    const int row0 = first * 8 + lane / 8, ch = lane % 8;
    GateAt pre[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) pre[i].load(g, m0 + row0 + 8 * i, c0 + ch * 8);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const float* at = stg + (row0 + 8 * i) * PITCH + ch * 8;
      const f32x4 lo = *reinterpret_cast<const f32x4*>(at), hi = *reinterpret_cast<const f32x4*>(at + 4);
      float dh[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      store_gate_gradient<T>(g, m0 + row0 + 8 * i, c0 + ch * 8, dh, pre[i]);
    }
  }
}

}  // namespace sd
