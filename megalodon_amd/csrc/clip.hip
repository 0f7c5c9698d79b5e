// The norm of many tensors together and clipping by it, for gfx950.
//   norm = sqrt(sum g^2) or max |g|; to = g min(1, max_norm / (norm + 1e-6))
// Bound by the bytes: all tensors once for the norm, once more and a write for the scaling.  The tensors' addresses and sizes
// are kernel arguments (a graph that is replayed has them with it; nothing is copied to the device), as many to a launch as
// 4 KB of arguments hold.  A launch's tensors are cut into chunks, walked by a grid that fills the device; every
// workgroup leaves one number, a second kernel adds them up in their order: no atomics, the same bits from call to call.
// Squares and sums are float64 (a product of two floats is exact there, and neither 1e30 nor 1e-30 is lost); the vector units have
// room for it, 4.5 elements a clock and CU at the memory's rate for 16 bits.
#include "common.hpp"

#include <algorithm>

namespace mega {
namespace {

constexpr int kThreads = 256;
constexpr int kGroups = 2048;  // workgroups of a launch: eight of four waves for each CU
constexpr int kPerLaunch = 160, kStarts = 16;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

// The tensors of a launch.  Chunks start[i] .. start[i + 1] - 1 are those of tensor i, the last of them of `last` elements.
struct Tensors {
  const void* from[kPerLaunch];
  void* to[kPerLaunch];  // (scaling only)
  uint32_t start[kPerLaunch + kStarts + 1];  // (behind the end: the largest number)
  uint16_t last[kPerLaunch];  // less one
  uint8_t dtype[kPerLaunch];
  int count, chunk_bytes;
};
static_assert(sizeof(Tensors) <= 4000, "kernel arguments have 4 KB");

struct Chunk {
  const void* from;
  void* to;
  int n, dtype;
};
// (Sixteen starts at a time in scalar registers: a search by halves is a chain of up to eight loads of the arguments, each waited for, and vector
// loads of them pass by the scalar cache.)
__device__ __forceinline__ Chunk chunk_of(const Tensors& t, uint32_t c) {
  int at = -1;
  for (int i = 0; i < t.count; i += kStarts) {
#pragma unroll
    for (int q = 0; q < kStarts; ++q) at += t.start[i + q] <= c;
    if (t.start[i + kStarts] > c) break;
  }
  const int dtype = t.dtype[at], size = dtype == MEGA_F32 ? 4 : 2;
  const int64_t offset = static_cast<int64_t>(c - t.start[at]) * t.chunk_bytes;
  const int n = c + 1 == t.start[at + 1] ? t.last[at] + 1 : t.chunk_bytes / size;
  return {static_cast<const char*>(t.from[at]) + offset, static_cast<char*>(t.to[at]) + offset, n, dtype};
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
template <bool MAX, int THREADS>
__device__ __forceinline__ double workgroup_total(double sum, uint32_t most) {
  __shared__ double sums[THREADS / kWave];
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
#pragma unroll
  for (int w = 1; w < THREADS / kWave; ++w) {
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
  sum = workgroup_total<MAX, kThreads>(sum, most);
  if (threadIdx.x == 0) totals[blockIdx.x] = sum;
}

// the workgroups' numbers: eight loads of a thread in flight
constexpr int kTotalThreads = 512;
template <bool MAX>
__global__ __launch_bounds__(kTotalThreads) void total_kernel(const double* totals, int64_t n, double* norm, float* out) {
  double sum = 0;
  uint32_t most = 0;
  for (int64_t i = threadIdx.x; i < n; i += 8 * kTotalThreads) {
    double v[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = totals[min(i + q * kTotalThreads, n - 1)];
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      if (i + q * kTotalThreads >= n) break;
      if constexpr (MAX) most = max(most, magnitude(static_cast<float>(v[q])));
      else sum += v[q];
    }
  }
  sum = workgroup_total<MAX, kTotalThreads>(sum, most);
  if (threadIdx.x != 0) return;
  if constexpr (!MAX) sum = sqrt(sum);
  *norm = sum;
  *out = static_cast<float>(sum);
}

// What a gradient is scaled by, in two parts: the ratio is below float32's normal numbers where gradients near the largest ones are clipped to a small norm.
// (Bit for bit the product with a float32 where that is a normal number.)
struct Factor {
  float part;
  int exponent;
  __device__ __forceinline__ float times(float v) const { return __builtin_amdgcn_ldexpf(v * part, exponent); }
};

template <int DT, bool APART>
__device__ __forceinline__ void scale_chunk(const Chunk& c, const Factor& factor) {
  using T = typename Elem<DT>::type;
  constexpr int kPer = DT == MEGA_F32 ? 4 : 8, kAhead = 4;
  const T* const p = static_cast<const T*>(c.from);
  T* const to = static_cast<T*>(c.to);
  const int whole = c.n / kPer;
  const auto scaled = [&](u32x4 q, int i) {
    float v[kPer];
    unpack<DT>(q, v);
#pragma unroll
    for (int e = 0; e < kPer; ++e) v[e] = factor.times(v[e]);
    uint4 w;
    if constexpr (DT == MEGA_F32) w = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    else w = pack8<DT>(v);
    u32x4_any* const at = reinterpret_cast<u32x4_any*>(to + static_cast<int64_t>(i) * kPer);
    if constexpr (APART) __builtin_nontemporal_store(__builtin_bit_cast(u32x4_any, w), at);
    else *at = __builtin_bit_cast(u32x4_any, w);
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
  if (const int rest = whole * kPer + threadIdx.x; rest < c.n) Elem<DT>::store(to + rest, factor.times(Elem<DT>::load(p + rest)));
}

__global__ __launch_bounds__(kThreads) void scale_kernel(const Tensors t, const double* norm, double max_norm) {
  const double ratio = max_norm / (*norm + 1e-6);
  int exponent = 0;
  const float part = ratio >= 1 ? 1.f : static_cast<float>(frexp(ratio, &exponent));  // (NaN stays NaN)
  const Factor factor{part, exponent};
  const uint32_t chunks = t.start[t.count];
  for (uint32_t i = blockIdx.x; i < chunks; i += gridDim.x) {
    // (from the end: what the norm read last is the likeliest to be in the memory-side cache)
    const Chunk k = chunk_of(t, chunks - 1 - i);
    const bool apart = k.from != k.to;
    if (part == 1.f && exponent == 0 && !apart) continue;
    const auto run = [&](auto together, auto streaming) { apart ? streaming(k, factor) : together(k, factor); };
    if (k.dtype == MEGA_F32) run(scale_chunk<MEGA_F32, false>, scale_chunk<MEGA_F32, true>);
    else if (k.dtype == MEGA_BF16) run(scale_chunk<MEGA_BF16, false>, scale_chunk<MEGA_BF16, true>);
    else run(scale_chunk<MEGA_F16, false>, scale_chunk<MEGA_F16, true>);
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
// Chunks of 64 KB, or of 16 KB (four pieces a thread, all in flight at once) where 64 KB would leave the device part empty.
int chunk_bytes_of(const mega_tensors& t) {
  int64_t bytes = 0;
  for (int64_t i = 0; i < t.count; ++i) bytes += t.size[i] * elem_size(t.dtype[i]);
  return bytes < (int64_t{kGroups} << 16) ? 1 << 14 : 1 << 16;
}
constexpr int64_t kMostChunks = 1ll << 31;  // of a launch

// The launches of a call, one after the other (`last_first`: from the end): f(tensors, workgroups).
template <typename F>
int each_launch(const mega_tensors& t, bool to, bool last_first, F f) {
  const int chunk_bytes = chunk_bytes_of(t);
  const auto chunks_of = [&](int64_t i) {
    const int64_t size = elem_size(t.dtype[i]);
    return (t.size[i] * size + chunk_bytes - 1) / chunk_bytes;
  };
  int64_t lo = 0, hi = t.count;  // the tensors that are left
  while (lo < hi) {
    // as many of them as a launch takes: [begin, end)
    int64_t count = 0, chunks = 0, n = 0;
    for (; n < hi - lo; ++n) {
      const int64_t one = chunks_of(last_first ? hi - 1 - n : lo + n);
      if (one == 0) continue;
      if (count == kPerLaunch || (count > 0 && chunks + one > kMostChunks)) break;
      ++count, chunks += one;
    }
    const int64_t begin = last_first ? hi - n : lo, end = begin + n;
    (last_first ? hi : lo) = last_first ? begin : end;
    if (count == 0) continue;
    Tensors a{};
    a.chunk_bytes = chunk_bytes;
    for (int64_t i = begin; i < end; ++i) {
      const int64_t size = elem_size(t.dtype[i]), one = chunks_of(i);
      if (one == 0) continue;
      const int k = a.count++;
      a.from[k] = t.from[i];
      a.to[k] = to ? t.to[i] : nullptr;
      a.start[k + 1] = a.start[k] + static_cast<uint32_t>(one);
      a.last[k] = static_cast<uint16_t>(t.size[i] - (one - 1) * (chunk_bytes / size) - 1);
      a.dtype[k] = static_cast<uint8_t>(t.dtype[i]);
    }
    for (int k = a.count + 1; k <= kPerLaunch + kStarts; ++k) a.start[k] = 0xffffffffu;
    if (const int rc = f(a, static_cast<unsigned>(std::min<int64_t>(a.start[a.count], kGroups))); rc != MEGA_OK) return rc;
  }
  return MEGA_OK;
}
int64_t totals_of(const mega_tensors& t) {
  int64_t n = 0;
  each_launch(t, false, false, [&](const Tensors&, unsigned groups) { return n += groups, static_cast<int>(MEGA_OK); });
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
  const int rc = each_launch(*tensors, false, false, [&](const Tensors& t, unsigned groups) {
    if (kind == MEGA_NORM_2) norm_kernel<false><<<groups, kThreads, 0, s>>>(t, totals + n);
    else norm_kernel<true><<<groups, kThreads, 0, s>>>(t, totals + n);
    MEGA_CHECK_LAUNCH();
    n += groups;
    return static_cast<int>(MEGA_OK);
  });
  if (rc != MEGA_OK) return rc;
  if (kind == MEGA_NORM_2) total_kernel<false><<<1, kTotalThreads, 0, s>>>(totals, n, norm, out_norm);
  else total_kernel<true><<<1, kTotalThreads, 0, s>>>(totals, n, norm, out_norm);
  MEGA_CHECK_LAUNCH();
  return MEGA_OK;
}

extern "C" int mega_tensors_clip(const mega_tensors* tensors, double max_norm, const void* workspace, void* stream) {
  if (const int rc = check_tensors("mega_tensors_clip", tensors, true); rc != MEGA_OK) return rc;
  MEGA_CHECK_ARG(max_norm >= 0, "mega_tensors_clip: max_norm must not be negative");
  MEGA_CHECK_ARG(workspace && reinterpret_cast<uintptr_t>(workspace) % 8 == 0, "mega_tensors_clip: null or misaligned pointer");
  hipStream_t s = static_cast<hipStream_t>(stream);
  return each_launch(*tensors, true, true, [&](const Tensors& t, unsigned groups) {
    scale_kernel<<<groups, kThreads, 0, s>>>(t, static_cast<const double*>(workspace), max_norm);
    MEGA_CHECK_LAUNCH();
    return static_cast<int>(MEGA_OK);
  });
}
