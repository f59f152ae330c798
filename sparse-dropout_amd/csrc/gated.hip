// The gate between the two products of a feed-forward block, as passes of its own:
//
//   forward   [G | U] -> H = act(G) U            backward   dH, [G | U] -> [dH U act'(G) | dH act(G)]
//
// Bound by bytes: 6 an element of H forward, 10 backward (8192 x 8192: 74 us and 120, 5.5 TB/s).  For products that no kernel takes with the gate in
// its store.  A thread takes eight columns of a row, one 16-byte load or store of each operand, wherever rows begin.
#include "gated.h"

namespace sd {
namespace {

constexpr int kThreads = 256;

struct Gate {
  const uint16_t *dh, *a;
  uint16_t* out;
  int64_t ldd, lda, up, ldo, M, F, cols;  // cols: of out, zeros behind the last
  int64_t eights;                         // of a row
};

struct Eight {
  float v[8];
  template <typename T>
  __device__ inline void load(const uint16_t* at, int left) {
    if (left >= 8) {
      const u32x4 w = *reinterpret_cast<const u32x4_any*>(at);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = T::to_float((uint16_t)(i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i < left ? T::to_float(at[i]) : 0.f;
    }
  }
  template <typename T>
  __device__ inline void store(uint16_t* at, int left) const {
    if (left >= 8) {
      *reinterpret_cast<u32x4_any*>(at) = u32x4{T::pack2(v[0], v[1]), T::pack2(v[2], v[3]), T::pack2(v[4], v[5]), T::pack2(v[6], v[7])};
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < left) at[i] = T::from_float(v[i]);
    }
  }
};
// zeros from column `from` of a row up to the last that is to be filled
__device__ inline void fill_row(uint16_t* row, int64_t from, int64_t cols) {
  for (int64_t i = from; i < cols; ++i) row[i] = 0;
}

template <typename T, int ACT, bool BACKWARD>
__global__ __launch_bounds__(kThreads) void gate_kernel(Gate g) {
  const int64_t total = g.M * g.eights, step = (int64_t)gridDim.x * kThreads;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += step) {
    const int64_t m = i / g.eights, c = (i - m * g.eights) * 8;
    const int left = g.F - c < 8 ? (int)(g.F - c) : 8;
    Eight gate, up;
    gate.load<T>(g.a + m * g.lda + c, left);
    up.load<T>(g.a + m * g.lda + g.up + c, left);
    if constexpr (!BACKWARD) {
#pragma unroll
      for (int e = 0; e < 8; ++e) gate.v[e] = gate_value(ACT, gate.v[e]) * up.v[e];
      gate.store<T>(g.out + m * g.ldo + c, left);
      if (c + 8 >= g.F) fill_row(g.out + m * g.ldo, g.F, g.cols);
    } else {
      Eight d;
      d.load<T>(g.dh + m * g.ldd + c, left);
#pragma unroll
      for (int e = 0; e < 8; ++e) gate_gradient(ACT, d.v[e], gate.v[e], up.v[e]);
      gate.store<T>(g.out + m * g.ldo + c, left);
      up.store<T>(g.out + m * g.ldo + g.F + c, left);
      if (c + 8 >= g.F) fill_row(g.out + m * g.ldo, 2 * g.F, g.cols);
    }
  }
}

template <typename T, bool BACKWARD>
int launch_gate(const Gate& g, int act, hipStream_t stream) {
  const int64_t wgs = ceil_div(g.M * g.eights, kThreads);
  const dim3 grid((unsigned)(wgs < 4096 ? wgs : 4096));
  auto* kernel = act == SD_ACT_SILU ? &gate_kernel<T, SD_ACT_SILU, BACKWARD> : act == SD_ACT_GELU ? &gate_kernel<T, SD_ACT_GELU, BACKWARD> : &gate_kernel<T, SD_ACT_RELU, BACKWARD>;
  hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, stream, g);
  return check_launch("gate_kernel");
}

int check_gate(const char* name, const void* a, int64_t lda, int64_t up, const void* out, int64_t ldo, int64_t wide, int64_t cols, int64_t M, int64_t F, int act,
               int dtype) {
  SD_REQUIRE(M >= 0 && F >= 0 && M < (1LL << 31) && F < (1LL << 30), "%s: bad extents %lld x %lld", name, (long long)M, (long long)F);
  SD_REQUIRE(dtype == SD_F16 || dtype == SD_BF16, "%s: dtype must be SD_F16 or SD_BF16 (got %d)", name, dtype);
  SD_REQUIRE(act == SD_ACT_RELU || act == SD_ACT_GELU || act == SD_ACT_SILU, "%s: act must be SD_ACT_RELU, SD_ACT_GELU or SD_ACT_SILU (got %d)", name, act);
  SD_REQUIRE(M == 0 || F == 0 || (a && out), "%s: null pointer", name);
  SD_REQUIRE(up >= F && (M <= 1 || lda >= up + F), "%s: U begins %lld columns behind G's %lld, at a pitch of %lld", name, (long long)up, (long long)F, (long long)lda);
  SD_REQUIRE(cols >= wide && cols <= (wide + 7) / 8 * 8 && (M <= 1 || ldo >= cols), "%s: a result of %lld columns, zeros up to %lld, at a pitch of %lld", name, (long long)wide,
             (long long)cols, (long long)ldo);
  return SD_OK;
}

}  // namespace
}  // namespace sd

using namespace sd;

extern "C" {

int sd_gated_forward(const void* A, int64_t lda, int64_t up, void* H, int64_t ldh, int64_t h_cols, int64_t M, int64_t F, int act, int dtype, void* stream) {
  if (int rc = check_gate("gated_forward", A, lda, up, H, ldh, F, h_cols, M, F, act, dtype)) return rc;
  if (M == 0 || F == 0) return SD_OK;
  Gate g = {nullptr, static_cast<const uint16_t*>(A), static_cast<uint16_t*>(H), 0, lda, up, ldh, M, F, h_cols, ceil_div(F, 8)};
  return dtype == SD_BF16 ? launch_gate<BF16, false>(g, act, (hipStream_t)stream) : launch_gate<F16, false>(g, act, (hipStream_t)stream);
}

int sd_gated_backward(const void* dH, int64_t ldd, const void* A, int64_t lda, int64_t up, void* dA, int64_t ldda, int64_t da_cols, int64_t M, int64_t F,
                      int act, int dtype, void* stream) {
  if (int rc = check_gate("gated_backward", A, lda, up, dA, ldda, 2 * F, da_cols, M, F, act, dtype)) return rc;
  if (M == 0 || F == 0) return SD_OK;
  SD_REQUIRE(dH && (M == 1 || ldd >= F), "gated_backward: null gradient, or its pitch %lld of %lld columns", (long long)ldd, (long long)F);
  Gate g = {static_cast<const uint16_t*>(dH), static_cast<const uint16_t*>(A), static_cast<uint16_t*>(dA), ldd, lda, up, ldda, M, F, da_cols, ceil_div(F, 8)};
  return dtype == SD_BF16 ? launch_gate<BF16, true>(g, act, (hipStream_t)stream) : launch_gate<F16, true>(g, act, (hipStream_t)stream);
}

}  // extern "C"
