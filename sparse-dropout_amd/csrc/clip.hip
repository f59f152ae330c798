// The norm of many gradients together and their clipping.
//
//   norm = sqrt(sum g^2) or max |g|        g = g min(1, max_norm / (norm + 1e-6))
//
// Bound by the gradients' bytes: read once for the norm, and once more, with a write, to be scaled.  Squares are summed in 64 bits: their sum
// neither overflows nor loses what lies under 2^-126, whatever the gradients' type, and the order of the sum, which is fixed by the sizes alone,
// shows in no bit of a 32-bit result.  Each workgroup leaves one partial sum; who needs the norm adds them up, always in the same order: the
// workgroups that scale do that by themselves, each of them, since that takes less than another launch.  Tensors of any
// number and type go by tables in the launch's arguments, a workgroup takes chunks off the whole of them.
#include <cfloat>
#include <cmath>

#include "common.h"

namespace sd {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 8192;       // elements of a workgroup at a time (the norm of 168 M bf16 elements 60 us, with 4096 71)
constexpr int kTensors = 176;
constexpr int kPartials = 1024;    // workgroups of all launches, where there are no more than kPartials / kFewest launches
constexpr int kFewest = 64;        // ... of a launch otherwise
constexpr double kSmall = 1e-6;    // beside the norm

struct GradTable {
  void* p[kTensors];
  int64_t n[kTensors];
  uint32_t first[kTensors + 1];  // chunk of the launch that a tensor begins at
  uint8_t dtype[kTensors];
  int32_t count;
};
struct NormArgs {
  GradTable t;
  double* partials;  // of this launch
};
struct ScaleArgs {
  GradTable t;
  const double* partials;  // of all launches
  int32_t n_partials, square;
  double max_norm;
  float* norm;  // null in all launches but one
};
static_assert(sizeof(NormArgs) <= 4096 && sizeof(ScaleArgs) <= 4096, "a launch's arguments");

struct F32 {
  static constexpr int id = SD_F32, per = 4;  // elements of 16 bytes
  typedef float elem;
  __device__ static inline float to_float(float v) { return v; }
  __device__ static inline float from_float(float v) { return v; }
};
template <typename T>
struct Half16 : T {
  static constexpr int per = 8;
  typedef uint16_t elem;
};

// 16 bytes of a tensor's elements, wherever it begins
template <typename T>
struct Piece {
  typedef typename T::elem elem;
  elem v[T::per];
  __device__ inline void load(const elem* at) {
    const u32x4 w = *reinterpret_cast<const u32x4_any*>(at);
    __builtin_memcpy(v, &w, 16);
  }
  __device__ inline void load_some(const elem* at, int left) {
#pragma unroll
    for (int i = 0; i < T::per; ++i) v[i] = i < left ? at[i] : elem(0);
  }
  __device__ inline void store(elem* at) const {
    u32x4 w;
    __builtin_memcpy(&w, v, 16);
    *reinterpret_cast<u32x4_any*>(at) = w;
  }
  __device__ inline void store_some(elem* at, int left) const {
#pragma unroll
    for (int i = 0; i < T::per; ++i)
      if (i < left) at[i] = v[i];
  }
};

__device__ inline double other_lane(double x, int mask) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)b, mask), hi = (uint32_t)__shfl_xor((int)(uint32_t)(b >> 32), mask);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// of numbers without a sign; NaN is the largest
__device__ inline double larger(double a, double b) {
  return __builtin_bit_cast(uint64_t, a) > __builtin_bit_cast(uint64_t, b) ? a : b;
}
template <bool SQUARE>
__device__ inline double joined(double a, double b) {
  return SQUARE ? a + b : larger(a, b);
}
// over a workgroup, in every thread
template <bool SQUARE>
__device__ inline double over_workgroup(double x, double* waves) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) x = joined<SQUARE>(x, other_lane(x, m));
  __syncthreads();
  if (threadIdx.x % 64 == 0) waves[threadIdx.x / 64] = x;
  __syncthreads();
  x = waves[0];
#pragma unroll
  for (int w = 1; w < kThreads / 64; ++w) x = joined<SQUARE>(x, waves[w]);
  return x;
}

// a chunk's elements of a thread
template <typename T>
struct Chunk {
  static constexpr int PASSES = kChunk / (kThreads * T::per);
  typedef typename T::elem elem;
  Piece<T> v[PASSES];
  __device__ static inline int place(int i) { return (i * kThreads + (int)threadIdx.x) * T::per; }
  __device__ inline void load(const void* p, int64_t at, int64_t n) {
    const elem* src = static_cast<const elem*>(p) + at;
    const int64_t left = n - at;
    if (left >= kChunk) {
#pragma unroll
      for (int i = 0; i < PASSES; ++i) v[i].load(src + place(i));
    } else {
#pragma unroll
      for (int i = 0; i < PASSES; ++i) v[i].load_some(src + place(i), (int)left - place(i));
    }
  }
  __device__ inline void scale(void* p, int64_t at, int64_t n, float by) {
    elem* dst = static_cast<elem*>(p) + at;
    const int64_t left = n - at;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
#pragma unroll
      for (int e = 0; e < T::per; ++e) v[i].v[e] = T::from_float(T::to_float(v[i].v[e]) * by);
      if (left >= kChunk) v[i].store(dst + place(i));
      else v[i].store_some(dst + place(i), (int)left - place(i));
    }
  }
};

// Where chunk number c of a table lies.  Every wave keeps the table's beginnings, a few to a lane, and finds a chunk's tensor by a comparison and a count:
// stepping through up to kTensors of them took longer than reading what they have (200 bf16 tensors of 100000 elements: 20.5 us, 15.7 so).
struct Place {
  int which;
  int64_t begin;
};
struct Finder {
  uint32_t ends[(kTensors + 63) / 64];
  __device__ inline explicit Finder(const GradTable& t) {
#pragma unroll
    for (int i = 0; i < (kTensors + 63) / 64; ++i) {
      const int k = i * 64 + (int)threadIdx.x % 64;
      ends[i] = k < t.count ? t.first[k + 1] : 0xffffffffu;
    }
  }
  __device__ inline Place operator()(const GradTable& t, uint32_t chunk) const {
    int which = 0;
#pragma unroll
    for (int i = 0; i < (kTensors + 63) / 64; ++i) which += __popcll(__ballot(ends[i] <= chunk));
    which = __builtin_amdgcn_readfirstlane(which);
    return Place{which, (int64_t)(chunk - t.first[which]) * kChunk};
  }
};

// what a thread adds of a chunk
template <bool SQUARE, typename T>
__device__ inline void add_chunk(const GradTable& t, const Place& at, double& sum) {
  Chunk<T> c;
  c.load(t.p[at.which], at.begin, t.n[at.which]);
  if constexpr (SQUARE) {
#pragma unroll
    for (int i = 0; i < Chunk<T>::PASSES; ++i)
#pragma unroll
      for (int e = 0; e < T::per; ++e) {
        const double g = (double)T::to_float(c.v[i].v[e]);
        sum = __builtin_fma(g, g, sum);
      }
  } else {
    uint32_t most = 0u;  // bits of magnitudes grow with them, NaN behind infinity
#pragma unroll
    for (int i = 0; i < Chunk<T>::PASSES; ++i)
#pragma unroll
      for (int e = 0; e < T::per; ++e) most = max(most, __builtin_bit_cast(uint32_t, T::to_float(c.v[i].v[e])) & 0x7fffffffu);
    sum = larger(sum, (double)__builtin_bit_cast(float, most));
  }
}

template <bool SQUARE>
__global__ __launch_bounds__(kThreads) void norm_partials_kernel(NormArgs a) {
  __shared__ double waves[kThreads / 64];
  const uint32_t chunks = a.t.first[a.t.count];
  const Finder find(a.t);
  double sum = 0.0;
  for (uint32_t chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    const Place at = find(a.t, chunk);
    const int dtype = a.t.dtype[at.which];
    if (dtype == SD_F32) add_chunk<SQUARE, F32>(a.t, at, sum);
    else if (dtype == SD_BF16) add_chunk<SQUARE, Half16<BF16>>(a.t, at, sum);
    else add_chunk<SQUARE, Half16<F16>>(a.t, at, sum);
  }
  sum = over_workgroup<SQUARE>(sum, waves);
  if (threadIdx.x == 0) a.partials[blockIdx.x] = sum;
}

// the norm from all partial sums, in every thread
__device__ inline double norm_of(const double* partials, int n, bool square, double* waves) {
  double x = 0.0;
  for (int i = threadIdx.x; i < n; i += kThreads) x = square ? x + partials[i] : larger(x, partials[i]);
  return square ? sqrt(over_workgroup<true>(x, waves)) : over_workgroup<false>(x, waves);
}
__device__ inline float factor_of(double norm, double max_norm) {
  const double c = max_norm / (norm + kSmall);
  return (float)(c > 1.0 ? 1.0 : c);  // (NaN stays)
}

__global__ __launch_bounds__(kThreads) void norm_finish_kernel(const double* partials, int n, int square, double max_norm, float* norm, float* scale) {
  __shared__ double waves[kThreads / 64];
  const double x = norm_of(partials, n, square != 0, waves);
  if (threadIdx.x == 0) {
    *norm = (float)x;
    if (scale) *scale = factor_of(x, max_norm);
  }
}

// A factor of one leaves every gradient as it is, so nothing more is read then; the first chunk is on its way while the partial sums are added up.
// A table's chunks are taken from the last eight on, for what the norm read last is still in the last cache (168 M bf16 elements, norm and all: 151 us,
// from the first on 165), and each on the XCD that read it for the norm, whose L2 may hold it (10 M: 12.7 us, on another XCD 19).  So it is with
// one table, up to kTensors tensors.  Several are scaled from the first on; and where the norm's workgroups of a launch (1024 shared out to the tables, 64 at
// least) are no multiple of eight, as with three tables, chunks behind a launch's first round were read on other XCDs.
template <typename T>
__device__ inline bool scale_first(const ScaleArgs& a, const Place& at, float& by, double* waves) {
  Chunk<T> c;
  c.load(a.t.p[at.which], at.begin, a.t.n[at.which]);
  const double norm = norm_of(a.partials, a.n_partials, a.square != 0, waves);
  if (a.norm && blockIdx.x == 0 && threadIdx.x == 0) *a.norm = (float)norm;
  by = factor_of(norm, a.max_norm);
  if (by == 1.f) return false;
  c.scale(a.t.p[at.which], at.begin, a.t.n[at.which], by);
  return true;
}
template <typename T>
__device__ inline void scale_chunk(const ScaleArgs& a, const Place& at, float by) {
  Chunk<T> c;
  c.load(a.t.p[at.which], at.begin, a.t.n[at.which]);
  c.scale(a.t.p[at.which], at.begin, a.t.n[at.which], by);
}
__global__ __launch_bounds__(kThreads) void scale_kernel(ScaleArgs a) {
  __shared__ double waves[kThreads / 64];
  const uint32_t chunks = a.t.first[a.t.count], eights = (chunks + 7) / 8;
  auto chunk_of = [&](uint32_t i) { return (eights - 1 - i / 8) * 8 + i % 8; };  // (of the last eight some may not be there)
  const Finder find(a.t);
  float by;
  if (blockIdx.x < 8 * eights && chunk_of(blockIdx.x) < chunks) {
    const Place at = find(a.t, chunk_of(blockIdx.x));
    const int dtype = a.t.dtype[at.which];
    if (!(dtype == SD_F32 ? scale_first<F32>(a, at, by, waves) : dtype == SD_BF16 ? scale_first<Half16<BF16>>(a, at, by, waves)
                                                                                  : scale_first<Half16<F16>>(a, at, by, waves)))
      return;
  } else {  // (nothing to scale at first, or at all)
    const double norm = norm_of(a.partials, a.n_partials, a.square != 0, waves);
    if (a.norm && blockIdx.x == 0 && threadIdx.x == 0) *a.norm = (float)norm;
    by = factor_of(norm, a.max_norm);
    if (by == 1.f) return;
  }
  for (uint32_t i = blockIdx.x + gridDim.x; i < 8 * eights; i += gridDim.x) {
    const uint32_t chunk = chunk_of(i);
    if (chunk >= chunks) continue;
    const Place at = find(a.t, chunk);
    const int dtype = a.t.dtype[at.which];
    if (dtype == SD_F32) scale_chunk<F32>(a, at, by);
    else if (dtype == SD_BF16) scale_chunk<Half16<BF16>>(a, at, by);
    else scale_chunk<Half16<F16>>(a, at, by);
  }
}

// The next launch's table from tensor i on; false: a tensor is too large.
bool fill(GradTable& t, int& i, int count, void* const* grads, const int64_t* n, const int32_t* dtypes) {
  t.count = 0;
  t.first[0] = 0;
  int64_t chunks = 0;
  for (; i < count && t.count < kTensors; ++i) {
    const int64_t more = ceil_div(n[i], kChunk);
    if (more >= (1LL << 31)) return false;
    if (chunks + more >= (1LL << 31)) break;
    if (more == 0) continue;
    t.p[t.count] = grads[i];
    t.n[t.count] = n[i];
    t.dtype[t.count] = (uint8_t)dtypes[i];
    chunks += more;
    t.first[++t.count] = (uint32_t)chunks;
  }
  return true;
}

// workgroups of a call's launches, at most
int most_workgroups(int count) {
  const int launches = (int)ceil_div(count, kTensors);
  return launches * kFewest > kPartials ? kFewest : kPartials / (launches ? launches : 1);
}
// (a launch more than the tables' number where the chunks of a table pass 2^31; sizes of 2^40 elements and more)
int64_t workspace_partials(int count, const int64_t* n) {
  int64_t chunks = 0;
  for (int i = 0; i < count; ++i) chunks += ceil_div(n[i], kChunk);
  const int64_t launches = ceil_div(count, kTensors) + chunks / (1LL << 30);
  const int64_t most = launches * most_workgroups(count);
  return chunks < most ? chunks : most;
}

int check_grads(const char* name, int count, const void* const* grads, const int64_t* n, const int32_t* dtypes, int norm_type, const float* norm,
                const void* workspace, int64_t workspace_bytes) {
  SD_REQUIRE(count >= 0, "%s: negative count", name);
  SD_REQUIRE(count == 0 || (grads && n && dtypes), "%s: null array", name);
  SD_REQUIRE(norm_type == SD_NORM_2 || norm_type == SD_NORM_MAX, "%s: norm_type must be SD_NORM_2 or SD_NORM_MAX (got %d)", name, norm_type);
  SD_REQUIRE(norm != nullptr, "%s: null norm", name);
  for (int i = 0; i < count; ++i) {
    SD_REQUIRE(n[i] >= 0, "%s: tensor %d: negative size", name, i);
    SD_REQUIRE(n[i] == 0 || grads[i], "%s: tensor %d: null pointer", name, i);
    SD_REQUIRE(dtypes[i] == SD_F16 || dtypes[i] == SD_BF16 || dtypes[i] == SD_F32, "%s: tensor %d: dtype must be SD_F16, SD_BF16 or SD_F32 (got %d)", name, i,
               dtypes[i]);
    if (n[i] >= (1LL << 42)) return fail(SD_ERR_UNSUPPORTED, "%s: a tensor of %lld elements is too large", name, (long long)n[i]);
  }
  const int64_t need = 8 * workspace_partials(count, n);
  SD_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "%s: workspace too small: need %lld bytes, got %lld", name, (long long)need,
             (long long)workspace_bytes);
  SD_REQUIRE(need == 0 || reinterpret_cast<uintptr_t>(workspace) % 8 == 0, "%s: workspace must be 8-byte aligned", name);
  return SD_OK;
}

// the partial sums of all gradients; how many there are to n_partials
int launch_partials(const char* name, int count, const void* const* grads, const int64_t* n, const int32_t* dtypes, bool square, double* partials,
                    int& n_partials, hipStream_t stream) {
  NormArgs a = {};
  const int most = most_workgroups(count);
  n_partials = 0;
  for (int i = 0; i < count;) {
    if (!fill(a.t, i, count, const_cast<void* const*>(grads), n, dtypes)) return fail(SD_ERR_UNSUPPORTED, "%s: a tensor is too large", name);
    if (a.t.count == 0) break;
    const uint32_t chunks = a.t.first[a.t.count];
    const int grid = chunks < (uint32_t)most ? (int)chunks : most;
    a.partials = partials + n_partials;
    hipLaunchKernelGGL((square ? &norm_partials_kernel<true> : &norm_partials_kernel<false>), dim3(grid), dim3(kThreads), 0, stream, a);
    if (int rc = check_launch(name)) return rc;
    n_partials += grid;
  }
  return SD_OK;
}

}  // namespace
}  // namespace sd

using namespace sd;

extern "C" {

int64_t sd_grad_norm_workspace_bytes(int count, const int64_t* numels) {
  if (count <= 0 || !numels) return 0;
  for (int i = 0; i < count; ++i)
    if (numels[i] < 0) return 0;
  return 8 * workspace_partials(count, numels);
}

int sd_grad_norm(int count, const void* const* grads, const int64_t* numels, const int32_t* dtypes, int norm_type, double max_norm, float* norm,
                 float* scale, void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check_grads("grad_norm", count, grads, numels, dtypes, norm_type, norm, workspace, workspace_bytes)) return rc;
  SD_REQUIRE(!scale || max_norm >= 0.0, "grad_norm: max_norm must not be negative (got %g)", max_norm);
  int n = 0;
  double* partials = static_cast<double*>(workspace);
  if (int rc = launch_partials("grad_norm", count, grads, numels, dtypes, norm_type == SD_NORM_2, partials, n, (hipStream_t)stream)) return rc;
  hipLaunchKernelGGL(&norm_finish_kernel, dim3(1), dim3(kThreads), 0, (hipStream_t)stream, partials, n, norm_type == SD_NORM_2 ? 1 : 0, max_norm, norm, scale);
  return check_launch("grad_norm");
}

int sd_clip_grads(int count, void* const* grads, const int64_t* numels, const int32_t* dtypes, int norm_type, double max_norm, float* norm,
                  void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check_grads("clip_grads", count, grads, numels, dtypes, norm_type, norm, workspace, workspace_bytes)) return rc;
  SD_REQUIRE(max_norm >= 0.0, "clip_grads: max_norm must not be negative (got %g)", max_norm);
  ScaleArgs a = {};
  a.partials = static_cast<const double*>(workspace);
  a.square = norm_type == SD_NORM_2 ? 1 : 0;
  a.max_norm = max_norm;
  a.norm = norm;
  if (int rc = launch_partials("clip_grads", count, grads, numels, dtypes, a.square != 0, static_cast<double*>(workspace), a.n_partials, (hipStream_t)stream))
    return rc;
  for (int i = 0; i < count || a.norm;) {
    if (!fill(a.t, i, count, grads, numels, dtypes)) return fail(SD_ERR_UNSUPPORTED, "clip_grads: a tensor is too large");
    const uint32_t chunks = a.t.first[a.t.count];
    if (chunks == 0 && !a.norm) break;
    // as many as are resident; eights of them, so that every one is on the XCD of its chunks
    const unsigned grid = chunks == 0 ? 1u : chunks < 2048u ? (chunks + 7) / 8 * 8 : 2048u;
    hipLaunchKernelGGL(&scale_kernel, dim3(grid), dim3(kThreads), 0, (hipStream_t)stream, a);
    if (int rc = check_launch("clip_grads")) return rc;
    a.norm = nullptr;
  }
  return SD_OK;
}

}  // extern "C"
