// A gated feed-forward block for few rows, the tokens of a serving step: launches that read each weight once.
//
//   h = act(x W_g^T) (x W_u^T)        y = h W_out^T
//
// Bound by the weights' bytes, 2 (2 F K + N F), and with few of them by a memory latency and a launch each.  So weights go from memory straight
// into the matrix instruction's registers.  A workgroup owns 4 to 32 outputs, 16 to a matrix instruction (lanes of outputs that are not there load
// nothing); its waves share out the 64-deep pieces of the reduction, which are whole 128-byte lines of its weight rows, wave w every piece
// w + WAVES n, AHEAD of them on their way at a time, and meet once in LDS.  A lane takes 32 consecutive bytes of a line (two loads, four lanes to a
// line); the order of the reduction within a piece is the same for both operands and shows in nothing but the last bits.  Rows come in groups of
// 16.  What comes back to a CU is what a group of rows costs beside the weights: lanes of rows that are not there load nothing, and where a workgroup
// would read more of h than of weights, the second launch's reduction is shared out over workgroups of more outputs, whose sums a third adds up.
//
// Up to 8 rows leave room for h twice in a group: h, which nothing but the second launch reads, is then held as the sum of two 16-bit numbers, the
// low halves in rows 8 to 15, and its rounding, the largest of the path, is saved.
#include <algorithm>

#include "gated.h"

namespace sd {
namespace {

constexpr int kDeep = 64;  // elements of a piece
constexpr int kTwice = 8;  // rows up to which h is held in two halves

struct Few {
  const uint16_t *x, *w;  // x: rows of the input, or of h
  uint16_t* h;            // [rows, or high halves and from row 8 on low ones][ldh]
  uint16_t* y;
  int64_t ldx, ldw, ldh, ldy;
  int M, N, K, act;  // N: hidden columns or outputs
  int cols;          // of a workgroup
  float* parts;      // of the second launch's sums, [gridDim.y][M][N], where its reduction is shared out over more workgroups ...
  int share;         // ... of so many pieces each
};

// 16 consecutive elements of a row, 16 q .. + 15 of a piece, as whole dwords, with one more behind them where rows may begin inside a dword (ODD):
// a load that begins there takes twice as long as one that is shifted afterwards (one row of 5461 to 2048 at a pitch of 5461: 13.6 us, at 5462 8.8).  No
// dword is read of which no element is wanted.
typedef u32x4 __attribute__((aligned(4))) u32x4_dwords;
template <bool ODD>
struct Sixteen {
  u32x4 v[2];
  uint32_t behind;
  __device__ inline void none() {
    v[0] = v[1] = u32x4{0u, 0u, 0u, 0u};
    if constexpr (ODD) behind = 0u;
  }
  __device__ inline void load(const uint16_t* at) {
    if constexpr (ODD) {
      const uintptr_t a = reinterpret_cast<uintptr_t>(at);
      const char* from = reinterpret_cast<const char*>(a & ~uintptr_t(3));
      v[0] = *reinterpret_cast<const u32x4_dwords*>(from);
      v[1] = *reinterpret_cast<const u32x4_dwords*>(from + 16);
      behind = *reinterpret_cast<const uint32_t*>(from + 28 + (a & 2) * 2);
    } else {  // (the last piece of an odd reduction begins inside a dword all the same)
      v[0] = *reinterpret_cast<const u32x4_any*>(at);
      v[1] = *reinterpret_cast<const u32x4_any*>(at + 8);
    }
  }
  // those of `left` that are there, zeros behind them: the dwords in which one is wanted, the last one's upper half taken out where it is none
  __device__ inline void load_some(const uint16_t* at, int left, uint32_t shift) {
    const uint32_t* from = reinterpret_cast<const uint32_t*>(reinterpret_cast<uintptr_t>(at) & ~uintptr_t(3));
    const int halves = left <= 0 ? 0 : left + (int)(shift >> 4);  // from the first dword on
    auto dword = [&](int i) { return 2 * i >= halves ? 0u : 2 * i + 1 < halves ? from[i] : from[i] & 0xffffu; };
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i / 4][i % 4] = dword(i);
    if constexpr (ODD) behind = dword(8);
  }
  // shift: 16 where the first element is a dword's upper half
  __device__ inline void settle(uint32_t shift) {
    if constexpr (!ODD) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i / 4][i % 4] = __builtin_amdgcn_alignbit(i < 7 ? v[(i + 1) / 4][(i + 1) % 4] : behind, v[i / 4][i % 4], shift);
  }
  // zeros for the first n
  __device__ inline void drop(int n) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i / 4][i % 4] = 2 * i >= n ? v[i / 4][i % 4] : 2 * i + 1 >= n ? v[i / 4][i % 4] & 0xffff0000u : 0u;
  }
};
template <bool ODD>
__device__ inline uint32_t shift_of(const uint16_t* at) {
  return ODD ? (uint32_t)(reinterpret_cast<uintptr_t>(at) & 2u) << 3 : 0u;
}

// HIDDEN: the first launch (both projections), else the second.  ODD: rows of weights or x may begin inside a dword.  SHARED: the reduction is shared
// out (0.2 us of a row's 6 where it is not)
template <typename T, bool HIDDEN, int WAVES, int GROUPS, int COLS, int AHEAD, bool ODD, bool SHARED>
__global__ __launch_bounds__(WAVES * 64) void gated_few_kernel(Few g) {
  constexpr int WP = HIDDEN ? 2 : 1;
  constexpr bool ODD_X = ODD && HIDDEN;  // (h has rows of whole lines)
  __shared__ float sums[WAVES][WP][16][17];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), r = lane & 15, q = lane >> 4;
  const int per = g.cols, n0 = (int)blockIdx.x * per;
  const bool twice = g.M <= kTwice;
  const uint16_t* w[COLS][WP];
  uint32_t w_shift[COLS][WP], x_shift[GROUPS];
#pragma unroll
  for (int j = 0; j < COLS; ++j)
#pragma unroll
    for (int p = 0; p < WP; ++p) {
      w[j][p] = g.w + (int64_t)(min(n0 + 16 * j + r, g.N - 1) + p * g.N) * g.ldw + 16 * q;
      w_shift[j][p] = shift_of<ODD>(w[j][p]);
    }
  // (a workgroup of a COLS of two or more fills all 16-column tiles but the last)
  auto reads_w = [&](int j) { return j + 1 < COLS || 16 * j + r < per; };
  const uint16_t* x[GROUPS];
  bool reads_x[GROUPS];
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) {
    const int row = 16 * i + r;
    reads_x[i] = HIDDEN || !twice ? row < g.M : (r & (kTwice - 1)) < g.M;
    x[i] = g.x + (int64_t)(reads_x[i] ? row : 0) * g.ldx + 16 * q;
    x_shift[i] = shift_of<ODD_X>(x[i]);
  }
  f32x4 acc[GROUPS][COLS][WP] = {};
  // k: where the piece begins; over: how many of its elements pieces in front have
  auto multiply = [&](Sixteen<ODD_X> (&a)[GROUPS], Sixteen<ODD> (&b)[COLS][WP], int k, int over) {
    const uint32_t turned = (uint32_t)(k & 1) << 4;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) {
      a[i].settle(x_shift[i] ^ turned);
      if (over) a[i].drop(over - 16 * q);
    }
#pragma unroll
    for (int j = 0; j < COLS; ++j)
#pragma unroll
      for (int p = 0; p < WP; ++p) {
        b[j][p].settle(w_shift[j][p] ^ turned);
        if (over) b[j][p].drop(over - 16 * q);
      }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int p = 0; p < WP; ++p)
#pragma unroll
        for (int i = 0; i < GROUPS; ++i)
#pragma unroll
          for (int j = 0; j < COLS; ++j) acc[i][j][p] = T::mfma16(a[i].v[h], b[j][p].v[h], acc[i][j][p]);
  };
  // Workgroups begin at different pieces: rows a power of two apart lie in one channel of memory, which all of them would ask for the same pieces at a
  // time (one row, hidden of 2048 to 8192: 15.0 us, so 13.3; 64 rows 23.5 and 21.3).
  const int pieces = g.K / kDeep, from = SHARED ? (int)blockIdx.y * g.share : 0, whole = SHARED ? min(g.share, pieces - from) : pieces;
  const int first = (int)(((blockIdx.x >> 3) & 31u) * (unsigned)whole >> 5);
  auto place = [&](int c) { return (from + (c + first < whole ? c + first : c + first - whole)) * kDeep; };
  auto load = [&](Sixteen<ODD_X> (&a)[AHEAD][GROUPS], Sixteen<ODD> (&b)[AHEAD][COLS][WP], auto&& there, auto&& at) {
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
#pragma unroll
      for (int j = 0; j < COLS; ++j)
#pragma unroll
        for (int p = 0; p < WP; ++p) b[u][j][p].none();
#pragma unroll
      for (int i = 0; i < GROUPS; ++i) a[u][i].none();
    }
#pragma unroll
    for (int j = 0; j < COLS; ++j)
      if (reads_w(j)) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
          if (there(u)) {
#pragma unroll
            for (int p = 0; p < WP; ++p) b[u][j][p].load(w[j][p] + at(u));
          }
      }
#pragma unroll
    for (int i = 0; i < GROUPS; ++i)
      if (reads_x[i]) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
          if (there(u)) a[u][i].load(x[i] + at(u));
      }
  };
  Sixteen<ODD> b[AHEAD][COLS][WP];
  Sixteen<ODD_X> a[AHEAD][GROUPS];
  for (int c0 = wave; c0 < whole; c0 += WAVES * AHEAD) {
    load(a, b, [&](int u) { return c0 + u * WAVES < whole; }, [&](int u) { return place(c0 + u * WAVES); });
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (c0 + u * WAVES < whole) multiply(a[u], b[u], 0, 0);
  }
  if (g.K % kDeep && wave == whole % WAVES && from + whole == pieces) {
    if (pieces) {  // what no whole piece has, as the end of one more
      load(a, b, [](int u) { return u == 0; }, [&](int) { return g.K - kDeep; });
      multiply(a[0], b[0], g.K, kDeep - g.K % kDeep);
    } else {
#pragma unroll
      for (int j = 0; j < COLS; ++j)
#pragma unroll
        for (int p = 0; p < WP; ++p) b[0][j][p].load_some(w[j][p], reads_w(j) ? g.K - 16 * q : 0, w_shift[j][p]);
#pragma unroll
      for (int i = 0; i < GROUPS; ++i) a[0][i].load_some(x[i], reads_x[i] ? g.K - 16 * q : 0, x_shift[i]);
      multiply(a[0], b[0], 0, 0);
    }
  }
#pragma unroll
  for (int i = 0; i < GROUPS; ++i)
#pragma unroll
    for (int j = 0; j < COLS; ++j) {
      if (i || j) __syncthreads();
#pragma unroll
      for (int p = 0; p < WP; ++p)
#pragma unroll
        for (int e = 0; e < 4; ++e) sums[wave][p][4 * q + e][r] = acc[i][j][p][e];
      __syncthreads();
      if (t < 256) {
        const int at = t >> 4, col = t & 15, n = n0 + 16 * j + col, m = 16 * i + at;
        if (m < g.M && (j + 1 < COLS || 16 * j + col < per)) {
          float s[WP] = {};
#pragma unroll
          for (int o = 0; o < WAVES; ++o)
#pragma unroll
            for (int p = 0; p < WP; ++p) s[p] += sums[o][p][at][col];
          if constexpr (HIDDEN) {
            if (n < g.N) {
              const float h = gate_value(g.act, s[0]) * s[WP - 1];
              const uint16_t high = T::from_float(h);
              g.h[m * g.ldh + n] = high;
              if (twice) {
                const float rounded = T::to_float(high);
                g.h[(kTwice + m) * g.ldh + n] = __builtin_isinf(rounded) ? (uint16_t)0 : T::from_float(h - rounded);  // (what overflows stays infinite)
              }
            }
          } else {
            if (twice) {
              float low = 0.f;
#pragma unroll
              for (int o = 0; o < WAVES; ++o) low += sums[o][0][kTwice + (at & (kTwice - 1))][col];
              if (__builtin_isfinite(s[0])) s[0] += low;  // (an infinite weight is one in the high halves' sum already; times a low half of 0 it is NaN)
            }
            if (n < g.N) {
              if constexpr (SHARED) g.parts[((int64_t)blockIdx.y * g.M + m) * g.N + n] = s[0];
              else g.y[(int64_t)m * g.ldy + n] = T::from_float(s[0]);
            }
          }
        }
      }
    }
}

// the parts' sums, always in one order
template <typename T>
__global__ __launch_bounds__(256) void few_sum_kernel(Few g, int shares) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, all = (int64_t)g.M * g.N;
  if (at >= all) return;
  float sum = 0.f;
  for (int i = 0; i < shares; ++i) sum += g.parts[i * all + at];
  g.y[at / g.N * g.ldy + at % g.N] = T::from_float(sum);
}

int groups_of(int64_t M) { return M <= 16 ? 1 : M <= 32 ? 2 : 4; }

// A launch's outputs to a workgroup (4 to 16, for 17 and more rows to 32: as many as leave one to four workgroups to a CU), how many workgroups share out a
// reduction, and what it is expected to take, us: 2.5, 0.16 for each 16 x 16 sums that the waves add up, and the longer of the weights at 5.4 TB/s and, for a CU
// in as many rounds as it has workgroups, the lines that come back to it at 36 GB/s (lanes that load nothing take a quarter of it all the same); 2.8 for the
// sum of the parts, and those, written and read, at 1.7 TB/s.  Within 7 % (root mean square) of 330 launches measured, 512 to 4096 wide, hidden of 1000 to 8192;
// of their shapes it picks such as take 0.1 % longer than the best.  One row of 8192 to 2048: 16 outputs 12.3 us, 8 10.6, two shares of 16 13.0; 24 rows 8
// outputs 18.9, four shares of 32 13.4; 64 rows 36.2, 19.7.  Hidden of 24 rows of 2048: 8192 with 16 17.6, with 32 15.8.  The block of 2048 to 5464 and back, one
// and 24 rows: with powers of two 20.2 and 28.4, with 11, 22 and 8, 32 18.1 and 24.8.
struct FewPlan {
  int cols = 0, shares = 0;
  double us = 1e30;
};
FewPlan plan_few(int64_t M, int64_t N, int64_t K, int parts) {
  const int groups = groups_of(M), rows = (int)(parts == 1 && M <= kTwice ? 2 * M : M);  // (either half of h for few of them)
  const int64_t pieces = ceil_div(K, kDeep);
  const double weights = 2.0 * parts * (double)N * (double)K / 5.4e6;
  FewPlan best;
  const uint32_t n = (uint32_t)N;  // (under 2^29, as the kernels count)
  for (uint32_t shares = 1; shares <= (parts == 1 ? 8 : 1) && (shares == 1 || pieces >= 8 * shares); shares *= 2) {
    if (shares > 1 && best.us <= 5.3 + weights) break;  // (no sum of parts takes less)
    for (uint32_t round = 1, last = 0; round <= 4; ++round) {  // as many outputs as leave so many workgroups to a CU
      const uint32_t each = (n * shares - 1) / (256 * round) + 1;
      const int cols = (int)std::min(std::max(each, 4u), groups > 1 ? 32u : 16u);
      if ((uint32_t)cols == last) continue;
      last = (uint32_t)cols;
      const double rounds = (double)((((n - 1) / cols + 1) * shares + 255) / 256), none = (cols > 16 ? 32 - cols : 16 - cols) * parts + 16 * groups - rows;
      const double lines = rounds * (double)pieces / shares * 128.0 * (cols * parts + rows + 0.25 * none) / 36e3;
      const double us = 2.5 + 0.16 * groups * (cols > 16 ? 2 : 1) * parts + (lines > weights ? lines + 0.05 * weights : weights + 0.05 * lines) +
                        (shares > 1 ? 2.8 + 8.0 * shares * (double)M * (double)N / 1.7e6 : 0.0);
      if (us < best.us) best = {cols, (int)shares, us};
    }
  }
  return best;
}

template <typename T, bool HIDDEN, bool ODD, bool SHARED>
void launch_few(const Few& f, const FewPlan& plan, hipStream_t stream) {
  Few g = f;
  const int groups = groups_of(g.M);
  g.cols = plan.cols;
  g.share = (int)ceil_div(g.K / kDeep, plan.shares);
  const dim3 grid((unsigned)ceil_div(g.N, plan.cols), (unsigned)plan.shares), block(512);
  // two pieces on their way at a time for 16 rows (one row, hidden of 2048 to 8192 cold: 13.4 us, with one 14.5), one for more (24 rows 17.0, with two 18.0)
  if (groups == 1) hipLaunchKernelGGL((&gated_few_kernel<T, HIDDEN, 8, 1, 1, 2, ODD, SHARED>), grid, block, 0, stream, g);
  else if (groups == 2 && plan.cols > 16) hipLaunchKernelGGL((&gated_few_kernel<T, HIDDEN, 8, 2, 2, 1, ODD, SHARED>), grid, block, 0, stream, g);
  else if (groups == 2) hipLaunchKernelGGL((&gated_few_kernel<T, HIDDEN, 8, 2, 1, 1, ODD, SHARED>), grid, block, 0, stream, g);
  else if (plan.cols > 16) hipLaunchKernelGGL((&gated_few_kernel<T, HIDDEN, 8, 4, 2, 1, ODD, SHARED>), grid, block, 0, stream, g);
  else hipLaunchKernelGGL((&gated_few_kernel<T, HIDDEN, 8, 4, 1, 1, ODD, SHARED>), grid, block, 0, stream, g);
  if constexpr (SHARED) hipLaunchKernelGGL((&few_sum_kernel<T>), dim3((unsigned)ceil_div((int64_t)g.M * g.N, 256)), dim3(256), 0, stream, g, plan.shares);
}
template <typename T, bool HIDDEN>
void launch_few_type(const Few& g, const FewPlan& plan, bool odd, hipStream_t stream) {
  if constexpr (!HIDDEN)
    if (plan.shares > 1) return odd ? launch_few<T, HIDDEN, true, true>(g, plan, stream) : launch_few<T, HIDDEN, false, true>(g, plan, stream);
  odd ? launch_few<T, HIDDEN, true, false>(g, plan, stream) : launch_few<T, HIDDEN, false, false>(g, plan, stream);
}

template <bool HIDDEN>
void launch_few_of(const Few& g, const FewPlan& plan, int dtype, hipStream_t stream) {
  const auto inside_dwords = [](const uint16_t* at, int64_t ld) { return (reinterpret_cast<uintptr_t>(at) & 2) != 0 || ld % 2 != 0; };
  const bool odd = inside_dwords(g.w, g.ldw) || (HIDDEN && inside_dwords(g.x, g.ldx));
  if (dtype == SD_BF16) launch_few_type<BF16, HIDDEN>(g, plan, odd, stream);
  else launch_few_type<F16, HIDDEN>(g, plan, odd, stream);
}

// Pitch of h: an odd number of whole pieces (rows a power of two apart lie in one channel of the L2).
int64_t hidden_pitch(int64_t F) { return (ceil_div(F, kDeep) | 1) * kDeep; }
int64_t hidden_bytes(int64_t M, int64_t F) { return 2 * (M <= kTwice ? 2 * kTwice : M) * hidden_pitch(F); }
int64_t parts_bytes(const FewPlan& plan, int64_t M, int64_t N) { return plan.shares > 1 ? 4 * plan.shares * M * N : 0; }

}  // namespace
}  // namespace sd

using namespace sd;

extern "C" {

int64_t sd_gated_mlp_few_workspace_bytes(int64_t M, int64_t F, int64_t N) {
  if (M <= 0 || M > SD_GATED_FEW_ROWS || F <= 0 || F >= (1LL << 29) || N <= 0 || N >= (1LL << 29)) return 0;
  return hidden_bytes(M, F) + parts_bytes(plan_few(M, N, F, 1), M, N);
}

int sd_gated_mlp_few_taken(int64_t M, int64_t K, int64_t F, int64_t N) {
  if (M <= 0 || M > SD_GATED_FEW_ROWS || K <= 0 || F <= 0 || N <= 0 || K >= (1LL << 29) || F >= (1LL << 29) || N >= (1LL << 29)) return 0;
  if (M <= 16) return 1;  // (6 to 58 % less time on ten layers, 256 to 4096 wide, 1 to 16 rows)
  // Of 60 calls with 17 to 64 rows on those layers 12 are sent the slower way, one by 17 %, the others by up to 7: 2048 to 8192 and back 24 rows 29.4 us
  // against 31.0, 64 rows 41.3 and 33.5; 1024 to 4096 and back 15.2 and 17.2, 21.5 and 18.4.
  // Rows that do not begin on 16 bytes are copied first on the other way: weights and activations at 3 TB/s, a launch each.  (By widths alone: that rows of
  // whole widths lie at odd pitches, and are copied too, is not asked, and goes against this way.)
  const double copied = (K % 8 ? 4.0 + 8.0 * F * K / 3e6 : 0.0) + (F % 8 ? 4.0 + 4.0 * N * F / 3e6 : 0.0);
  return 1.05 * (plan_few(M, F, K, 2).us + plan_few(M, N, F, 1).us) <= gated_expected_us(M, F, K) + dense_expected_us(M, N, F) + copied ? 1 : 0;
}

int sd_gated_mlp_few(const void* X, int64_t ldx, const void* W_in, int64_t ldwi, const void* W_out, int64_t ldwo, void* Y, int64_t ldy, int64_t M,
                     int64_t K, int64_t F, int64_t N, int act, int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  SD_REQUIRE(M >= 0 && K > 0 && F > 0 && N > 0 && K < (1LL << 29) && F < (1LL << 29) && N < (1LL << 29), "gated_mlp_few: bad extents %lld, %lld, %lld, %lld",
             (long long)M, (long long)K, (long long)F, (long long)N);
  SD_REQUIRE(dtype == SD_F16 || dtype == SD_BF16, "gated_mlp_few: dtype must be SD_F16 or SD_BF16 (got %d)", dtype);
  SD_REQUIRE(act == SD_ACT_RELU || act == SD_ACT_GELU || act == SD_ACT_SILU, "gated_mlp_few: act must be SD_ACT_RELU, SD_ACT_GELU or SD_ACT_SILU (got %d)", act);
  if (M == 0) return SD_OK;
  if (M > SD_GATED_FEW_ROWS) return fail(SD_ERR_UNSUPPORTED, "gated_mlp_few: %lld rows, at most %d", (long long)M, SD_GATED_FEW_ROWS);
  SD_REQUIRE(X && W_in && W_out && Y, "gated_mlp_few: null pointer");
  SD_REQUIRE((M == 1 || (ldx >= K && ldy >= N)) && ldwi >= K && (N == 1 || ldwo >= F), "gated_mlp_few: a pitch is shorter than its row");
  const FewPlan hidden = plan_few(M, F, K, 2), outputs = plan_few(M, N, F, 1);
  const int64_t need = hidden_bytes(M, F) + parts_bytes(outputs, M, N);
  SD_REQUIRE(workspace && workspace_bytes >= need, "gated_mlp_few: workspace too small: need %lld bytes, got %lld", (long long)need, (long long)workspace_bytes);
  SD_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "gated_mlp_few: workspace must be 16-byte aligned");
  Few g = {};
  g.x = static_cast<const uint16_t*>(X);
  g.w = static_cast<const uint16_t*>(W_in);
  g.h = static_cast<uint16_t*>(workspace);
  g.ldx = ldx;
  g.ldw = ldwi;
  g.ldh = hidden_pitch(F);
  g.M = (int)M;
  g.N = (int)F;
  g.K = (int)K;
  g.act = act;
  launch_few_of<true>(g, hidden, dtype, (hipStream_t)stream);
  if (int rc = check_launch("gated_mlp_few")) return rc;
  g.x = g.h;
  g.w = static_cast<const uint16_t*>(W_out);
  g.y = static_cast<uint16_t*>(Y);
  if (outputs.shares > 1) g.parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + hidden_bytes(M, F));
  g.ldx = g.ldh;
  g.ldw = ldwo;
  g.ldy = ldy;
  g.N = (int)N;
  g.K = (int)F;
  launch_few_of<false>(g, outputs, dtype, (hipStream_t)stream);
  note_kernel("gated:few groups=%d cols=%d,%d shares=%d", groups_of(M), hidden.cols, outputs.cols, outputs.shares);
  return check_launch("gated_mlp_few");
}

}  // extern "C"
