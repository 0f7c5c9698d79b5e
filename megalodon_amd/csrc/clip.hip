// The norm of many tensors together and clipping by it, for gfx950.
//   norm = sqrt(sum g^2) or max |g|; to = g min(1, max_norm / (norm + 1e-6))
// Bound by the bytes: all tensors once for the norm, once more and a write for the scaling.  The tensors' addresses and sizes
// are kernel arguments (a graph that is replayed has them with it; nothing is copied to the device), as many to a launch as
// 4 KB of arguments hold.  A launch's tensors are cut into chunks of 64 KB, walked by a grid that fills the device; every
// workgroup leaves one number, a second kernel adds them up in their order: no atomics, the same bits from call to call.
// Squares and sums are float64 (a product of two floats is exact there, and neither 1e30 nor 1e-30 is lost); the vector units have
// room for it, 4.5 elements a clock and CU at the memory's rate for 16 bits.
#include "common.hpp"

#include <algorithm>
#include <vector>

namespace mega {
namespace {

constexpr int kThreads = 256;
constexpr int kChunkBytes = 65536;
constexpr int kGroups = 2048;  // workgroups of a launch: eight of four waves for each CU
constexpr int kPerLaunch = 160;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

// The tensors of a launch.  Chunks start[i] .. start[i + 1] - 1 are those of tensor i, the last of them of `last` elements.
struct Tensors {
  const void* from[kPerLaunch];
  void* to[kPerLaunch];  // (scaling only)
  uint32_t start[kPerLaunch + 1];
  uint16_t last[kPerLaunch];  // less one
  uint8_t dtype[kPerLaunch];
  int count;
};
static_assert(sizeof(Tensors) <= 4000, "kernel arguments have 4 KB");

struct Chunk {
  const void* from;
  void* to;
  int n, dtype;
};
__device__ __forceinline__ Chunk chunk_of(const Tensors& t, uint32_t c) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (t.start[mid] <= c) lo = mid;
    else hi = mid - 1;
  }
  const int dtype = t.dtype[lo], size = dtype == MEGA_F32 ? 4 : 2;
  const int64_t at = static_cast<int64_t>(c - t.start[lo]) * kChunkBytes;
  const int n = c + 1 == t.start[lo + 1] ? t.last[lo] + 1 : kChunkBytes / size;
  return {static_cast<const char*>(t.from[lo]) + at, static_cast<char*>(t.to[lo]) + at, n, dtype};
}

template <int DT>
__device__ __forceinline__ void unpack(u32x4 q, float* v) {
  if constexpr (DT == MEGA_F32) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = __uint_as_float(q[e]);
  } else {
    unpack8<DT>(make_uint4(q[0], q[1], q[2], q[3]), v);
  }
}

// magnitudes by their bits: the order of the numbers, and NaN above all of them
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

template <int DT, bool MAX>
__device__ __forceinline__ void norm_chunk(const Chunk& c, double& sum, uint32_t& most) {
  using T = typename Elem<DT>::type;
  constexpr int kPer = DT == MEGA_F32 ? 4 : 8, kAhead = 4;
  const T* const p = static_cast<const T*>(c.from);
  const int whole = c.n / kPer;
  const auto add = [&](float v) {
    if constexpr (MAX) most = max(most, magnitude(v));
    else sum = fma(static_cast<double>(v), static_cast<double>(v), sum);
  };
  int i = threadIdx.x;
  for (; i + (kAhead - 1) * kThreads < whole; i += kAhead * kThreads) {
    u32x4 q[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) q[a] = __builtin_bit_cast(u32x4, *reinterpret_cast<const u32x4_any*>(p + static_cast<int64_t>(i + a * kThreads) * kPer));
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      float v[kPer];
      unpack<DT>(q[a], v);
#pragma unroll
      for (int e = 0; e < kPer; ++e) add(v[e]);
    }
  }
  for (; i < whole; i += kThreads) {
    float v[kPer];
    unpack<DT>(__builtin_bit_cast(u32x4, *reinterpret_cast<const u32x4_any*>(p + static_cast<int64_t>(i) * kPer)), v);
#pragma unroll
    for (int e = 0; e < kPer; ++e) add(v[e]);
  }
  if (const int rest = whole * kPer + threadIdx.x; rest < c.n) add(Elem<DT>::load(p + rest));
}

// sum over the workgroup, in an order of its own, for thread 0
template <bool MAX>
__device__ __forceinline__ double workgroup_total(double sum, uint32_t most) {
  __shared__ double sums[kThreads / kWave];
  if constexpr (MAX) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), off)));
    sum = static_cast<double>(__uint_as_float(most));
  } else {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
  }
  if (threadIdx.x % kWave == 0) sums[threadIdx.x / kWave] = sum;
  __syncthreads();
  if (threadIdx.x != 0) return 0.0;
  for (int w = 1; w < kThreads / kWave; ++w) {
    if constexpr (MAX) sum = sums[w] > sum || sums[w] != sums[w] ? sums[w] : sum;
    else sum += sums[w];
  }
  return sum;
}

template <bool MAX>
__global__ __launch_bounds__(kThreads) void norm_kernel(const Tensors t, double* totals) {
  double sum = 0;
  uint32_t most = 0;
  const uint32_t chunks = t.start[t.count];
  for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
    const Chunk k = chunk_of(t, c);
    if (k.dtype == MEGA_F32) norm_chunk<MEGA_F32, MAX>(k, sum, most);
    else if (k.dtype == MEGA_BF16) norm_chunk<MEGA_BF16, MAX>(k, sum, most);
    else norm_chunk<MEGA_F16, MAX>(k, sum, most);
  }
  sum = workgroup_total<MAX>(sum, most);
  if (threadIdx.x == 0) totals[blockIdx.x] = sum;
}

template <bool MAX>
__global__ __launch_bounds__(kThreads) void total_kernel(const double* totals, int64_t n, double* norm, float* out) {
  double sum = 0;
  uint32_t most = 0;
  for (int64_t i = threadIdx.x; i < n; i += kThreads) {
    if constexpr (MAX) most = max(most, magnitude(static_cast<float>(totals[i])));
    else sum += totals[i];
  }
  sum = workgroup_total<MAX>(sum, most);
  if (threadIdx.x != 0) return;
  if constexpr (!MAX) sum = sqrt(sum);
  *norm = sum;
  *out = static_cast<float>(sum);
}

template <int DT>
__device__ __forceinline__ void scale_chunk(const Chunk& c, float factor) {
  using T = typename Elem<DT>::type;
  constexpr int kPer = DT == MEGA_F32 ? 4 : 8, kAhead = 4;
  const T* const p = static_cast<const T*>(c.from);
  T* const to = static_cast<T*>(c.to);
  const int whole = c.n / kPer;
  const auto scaled = [&](u32x4 q, int i) {
    float v[kPer];
    unpack<DT>(q, v);
#pragma unroll
    for (int e = 0; e < kPer; ++e) v[e] *= factor;
    uint4 w;
    if constexpr (DT == MEGA_F32) w = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    else w = pack8<DT>(v);
    *reinterpret_cast<u32x4_any*>(to + static_cast<int64_t>(i) * kPer) = __builtin_bit_cast(u32x4_any, w);
  };
  int i = threadIdx.x;
  for (; i + (kAhead - 1) * kThreads < whole; i += kAhead * kThreads) {
    u32x4 q[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) q[a] = __builtin_bit_cast(u32x4, *reinterpret_cast<const u32x4_any*>(p + static_cast<int64_t>(i + a * kThreads) * kPer));
#pragma unroll
    for (int a = 0; a < kAhead; ++a) scaled(q[a], i + a * kThreads);
  }
  for (; i < whole; i += kThreads) scaled(__builtin_bit_cast(u32x4, *reinterpret_cast<const u32x4_any*>(p + static_cast<int64_t>(i) * kPer)), i);
  if (const int rest = whole * kPer + threadIdx.x; rest < c.n) Elem<DT>::store(to + rest, Elem<DT>::load(p + rest) * factor);
}

__global__ __launch_bounds__(kThreads) void scale_kernel(const Tensors t, const double* norm, double max_norm) {
  const double ratio = max_norm / (*norm + 1e-6);
  const float factor = ratio >= 1 ? 1.f : static_cast<float>(ratio);  // (NaN stays NaN)
  const uint32_t chunks = t.start[t.count];
  for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
    const Chunk k = chunk_of(t, c);
    if (factor == 1.f && k.from == k.to) continue;
    if (k.dtype == MEGA_F32) scale_chunk<MEGA_F32>(k, factor);
    else if (k.dtype == MEGA_BF16) scale_chunk<MEGA_BF16>(k, factor);
    else scale_chunk<MEGA_F16>(k, factor);
  }
}

// ---- host side ------------------------------------------------------------------------------------------
int check_tensors(const char* who, const mega_tensors* t, bool to) {
  MEGA_CHECK_ARG(t != nullptr && t->count >= 0 && (t->count == 0 || (t->from && t->size && t->dtype && (!to || t->to))), "%s: null array or bad count", who);
  for (int64_t i = 0; i < t->count; ++i) {
    MEGA_CHECK_ARG(valid_dtype(t->dtype[i]), "%s: float32, bfloat16 or float16 tensors", who);
    MEGA_CHECK_ARG(t->size[i] >= 0 && t->size[i] < (1ll << 44), "%s: bad sizes", who);
    MEGA_CHECK_ARG(t->size[i] == 0 || (t->from[i] && (!to || t->to[i])), "%s: null pointer", who);
  }
  return MEGA_OK;
}
int64_t chunks_of(const mega_tensors& t, int64_t i) { return (t.size[i] * elem_size(t.dtype[i]) + kChunkBytes - 1) / kChunkBytes; }
constexpr int64_t kMostChunks = 1ll << 31;  // of a launch

// The launches of a call, one after the other: f(tensors, workgroups).
template <typename F>
int each_launch(const mega_tensors& t, bool to, F f) {
  Tensors a{};
  const auto flush = [&]() {
    if (a.count == 0) return static_cast<int>(MEGA_OK);
    const int rc = f(a, static_cast<unsigned>(std::min<int64_t>(a.start[a.count], kGroups)));
    a.count = 0;
    return rc;
  };
  for (int64_t i = 0; i < t.count; ++i) {
    const int64_t chunks = chunks_of(t, i), size = elem_size(t.dtype[i]);
    if (chunks == 0) continue;
    if (a.count == kPerLaunch || (a.count > 0 && a.start[a.count] + chunks > kMostChunks))
      if (const int rc = flush(); rc != MEGA_OK) return rc;
    const int k = a.count++;
    a.from[k] = t.from[i];
    a.to[k] = to ? t.to[i] : nullptr;
    a.start[k + 1] = a.start[k] + static_cast<uint32_t>(chunks);
    a.last[k] = static_cast<uint16_t>(t.size[i] - (chunks - 1) * (kChunkBytes / size) - 1);
    a.dtype[k] = static_cast<uint8_t>(t.dtype[i]);
  }
  return flush();
}
int64_t totals_of(const mega_tensors& t) {
  int64_t n = 0;
  each_launch(t, false, [&](const Tensors&, unsigned groups) { return n += groups, static_cast<int>(MEGA_OK); });
  return n;
}

}  // namespace
}  // namespace mega

using namespace mega;

// workspace: the norm, then one total a workgroup
extern "C" int64_t mega_tensors_workspace_bytes(const mega_tensors* tensors) {
  if (tensors == nullptr || check_tensors("mega_tensors_workspace_bytes", tensors, false) != MEGA_OK) return 0;
  return 8 * (1 + totals_of(*tensors));
}

extern "C" int mega_tensors_norm(const mega_tensors* tensors, int kind, float* out_norm, void* workspace, void* stream) {
  if (const int rc = check_tensors("mega_tensors_norm", tensors, false); rc != MEGA_OK) return rc;
  MEGA_CHECK_ARG(kind == MEGA_NORM_2 || kind == MEGA_NORM_MAX, "mega_tensors_norm: unknown kind of norm");
  MEGA_CHECK_ARG(out_norm && workspace && reinterpret_cast<uintptr_t>(workspace) % 8 == 0, "mega_tensors_norm: null or misaligned pointer");
  hipStream_t s = static_cast<hipStream_t>(stream);
  double *const norm = static_cast<double*>(workspace), *const totals = norm + 1;
  int64_t n = 0;
  const int rc = each_launch(*tensors, false, [&](const Tensors& t, unsigned groups) {
    if (kind == MEGA_NORM_2) norm_kernel<false><<<groups, kThreads, 0, s>>>(t, totals + n);
    else norm_kernel<true><<<groups, kThreads, 0, s>>>(t, totals + n);
    MEGA_CHECK_LAUNCH();
    n += groups;
    return static_cast<int>(MEGA_OK);
  });
  if (rc != MEGA_OK) return rc;
  if (kind == MEGA_NORM_2) total_kernel<false><<<1, kThreads, 0, s>>>(totals, n, norm, out_norm);
  else total_kernel<true><<<1, kThreads, 0, s>>>(totals, n, norm, out_norm);
  MEGA_CHECK_LAUNCH();
  return MEGA_OK;
}

extern "C" int mega_tensors_clip(const mega_tensors* tensors, double max_norm, const void* workspace, void* stream) {
  if (const int rc = check_tensors("mega_tensors_clip", tensors, true); rc != MEGA_OK) return rc;
  MEGA_CHECK_ARG(max_norm >= 0, "mega_tensors_clip: max_norm must not be negative");
  MEGA_CHECK_ARG(workspace && reinterpret_cast<uintptr_t>(workspace) % 8 == 0, "mega_tensors_clip: null or misaligned pointer");
  hipStream_t s = static_cast<hipStream_t>(stream);
  return each_launch(*tensors, true, [&](const Tensors& t, unsigned groups) {
    scale_kernel<<<groups, kThreads, 0, s>>>(t, static_cast<const double*>(workspace), max_norm);
    MEGA_CHECK_LAUNCH();
    return static_cast<int>(MEGA_OK);
  });
}
