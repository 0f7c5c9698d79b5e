// The gated half of a feed-forward network for gfx950 (bfloat16 / float16 rows, float32 inside):
//   a = x w1^T, b = x w3^T, h = a sigma(a) b                       (x: tokens x n_in, w1, w3: n_out x n_in)
//   da = dh b sigma(a) (1 + a (1 - sigma(a))), db = dh a sigma(a)
//   dx = da w1 + db w3, dw1 = da^T x, dw3 = db^T x
// One kernel has both projections: a wave's accumulators hold a and b of the same elements, and the gate is taken from them
// in float32, so that neither product goes through memory.  Training keeps both for the backward, in float32 or rounded to the
// operands' type: half the memory, and a third rounding of the gradients besides those of da and db (operands of the matrix
// cores) and of the results.  (Gradients in 16 bits are off by 1.4 times what rounding them once takes where
// float32 is kept, by 1.8 where not; training on 32768 tokens, 4096 -> 11008, takes 5 % longer with it, 4084 tokens, 2048 -> 5504, 8 %.)
//
// Many tokens: tiles with the gate for an epilogue (gated_product of attention.hip, gated_tiles.hip).  Few: the weights' stream from
// memory is all the time there is, and the kernel below reads them once, straight into the operand registers of the matrix cores.
#include "common.hpp"
#include "gated.hpp"

#include <algorithm>
#include <type_traits>

namespace mega {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <int DT>
__device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (DT == MEGA_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// ---- few tokens -------------------------------------------------------------------------------------
// A workgroup has FT groups of 8 features and all of the tokens (NT blocks of 16); its waves take turns along k and meet in LDS, in
// their order.  A product of 16 rows (8 features of w1, the same 8 of w3) x 16 tokens x 32 k: lane l holds 8 k of row l % 16 and
// 8 k of token l % 16, k = 32 step + 8 (l / 16), so that both come from memory as they are, 64 bytes of a row to four lanes, and what a workgroup has
// in flight are whole pieces of rows.  It gives lane l token l % 16 of rows 4 (l / 16) .. + 3.
// Rows behind the last feature or token are the last one again, never stored.  WHOLE: rows are whole 16-byte pieces.
constexpr int kFewWaves = 8;

// Which calls go here: up to 16 tokens all; then the tokens, read again for every few features, cost more than the tiles' second launch
// the more the larger the weights are (us, here / tiles: 4096 -> 11008 16 tokens 47 / 50, 24 53 / 51, 64 80 / 54; 2048 -> 5504
// 16 15 / 19, 48 20.2 / 20.7, 64 21.9 / 20.8; 1024 -> 2752 64 8.4 / 12.7).  Rows that the small tiles do not take (n_in no multiple of 64): up to 64, since the large
// tiles' time hardly falls with the tokens (17, 32, 48, 64 tokens: 1000 -> 2736 6 / 15, 6 / 15, 8 / 16, 8 / 17; 1001 -> 2731 9 / 20, 11 / 20, 15 / 21, 16 / 21; 2056 -> 5504 17 / 27,
// 19 / 27, 23 / 28, 26 / 28; 4088 -> 11008 58 / 64, 70 / 65, 80 / 66, 90 / 67; 4085 -> 11007 89 / 115, 114 / 119, 149 / 121, 173 / 123: the largest network's 32 to 64 tokens lose by it).
bool few(int64_t tokens, int64_t n_in, int64_t n_out) {
  if (tokens <= 16 || tokens > 64) return tokens <= 16;
  return n_in % 64 != 0 || static_cast<double>(tokens - 16) * n_in * n_out <= 4e8;
}


struct FewParams {
  const uint16_t *x, *w1, *w3;
  uint16_t* h;
  void *a, *b;
  int tokens, n_in, n_out, wide, pitch;
};

template <bool WHOLE>
__device__ __forceinline__ u32x4 eight(const uint16_t* row, int k, int n) {
  if (k + 8 <= n) {
    if constexpr (WHOLE) return *reinterpret_cast<const u32x4*>(row + k);
    else return __builtin_bit_cast(u32x4, *reinterpret_cast<const u32x4_any*>(row + k));
  }
  uint32_t e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {  // (all of them asked for together)
    const uint32_t v = row[min(k + i, n - 1)];
    e[i] = k + i < n ? v : 0u;
  }
  return u32x4{e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16};
}

template <int DT, int NT, int FT, bool WHOLE>
__global__ __launch_bounds__(kFewWaves * kWave) void gated_few_kernel(const FewParams p) {
  __shared__ f32x4 sums[kFewWaves][FT * NT][kWave];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, r = lane % 16, g = lane / 16;
  const int f0 = blockIdx.x * (8 * FT);
  const uint16_t *w[FT], *x[NT];
#pragma unroll
  for (int f = 0; f < FT; ++f) w[f] = (r < 8 ? p.w1 : p.w3) + static_cast<int64_t>(min(f0 + 8 * f + r % 8, p.n_out - 1)) * p.n_in;
#pragma unroll
  for (int t = 0; t < NT; ++t) x[t] = p.x + static_cast<int64_t>(min(16 * t + r, p.tokens - 1)) * p.n_in;
  f32x4 acc[FT][NT];
#pragma unroll
  for (int f = 0; f < FT; ++f)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[f][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int steps = p.n_in / 32;  // (whole ones)
  constexpr int U = FT * NT > 1 && FT * NT <= 4 ? 4 : 1;  // steps whose operands are asked for together (measured)
  // Every workgroup begins somewhere else along k: in step with each other they would all ask the same channels of L2 and memory.
  const int rounds = steps / (U * kFewWaves);
  int at = rounds > 0 ? static_cast<int>(blockIdx.x % rounds) : 0;
  for (int i = 0; i < rounds; ++i) {
    const int s = at * (U * kFewWaves) + wave;
    if (++at == rounds) at = 0;
    u32x4 a[U][FT], v[U][NT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = 32 * (s + u * kFewWaves) + 8 * g;
#pragma unroll
      for (int f = 0; f < FT; ++f) a[u][f] = eight<WHOLE>(w[f], k, 0x7fffffff);
#pragma unroll
      for (int t = 0; t < NT; ++t) v[u][t] = eight<WHOLE>(x[t], k, 0x7fffffff);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int f = 0; f < FT; ++f)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[f][t] = mma16<DT>(a[u][f], v[u][t], acc[f][t]);
  }
  for (int s = rounds * (U * kFewWaves) + wave; 32 * s < p.n_in; s += kFewWaves) {
    const int k = 32 * s + 8 * g;
    u32x4 a[FT], v[NT];
#pragma unroll
    for (int f = 0; f < FT; ++f) a[f] = eight<WHOLE>(w[f], k, p.n_in);
#pragma unroll
    for (int t = 0; t < NT; ++t) v[t] = eight<WHOLE>(x[t], k, p.n_in);
#pragma unroll
    for (int f = 0; f < FT; ++f)
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[f][t] = mma16<DT>(a[f], v[t], acc[f][t]);
  }
#pragma unroll
  for (int f = 0; f < FT; ++f)
#pragma unroll
    for (int t = 0; t < NT; ++t) sums[wave][f * NT + t][lane] = acc[f][t];
  __syncthreads();
  // a wave adds up half a block: features 4 half .. + 3 of 16 tokens are lanes 16 half .. of a and 32 lanes on of b
  for (int i = threadIdx.x / 16; i < FT * NT * 2; i += kFewWaves * kWave / 16) {
    const int block = i / 2, half = i % 2, at = 16 * half + r;
    f32x4 a = sums[0][block][at], b = sums[0][block][at + 32];
#pragma unroll
    for (int q = 1; q < kFewWaves; ++q) a += sums[q][block][at], b += sums[q][block][at + 32];
    const int token = 16 * (block % NT) + r, f = f0 + 8 * (block / NT) + 4 * half;
    if (token >= p.tokens) continue;
    const int64_t to = static_cast<int64_t>(token) * p.n_out + f, kept = static_cast<int64_t>(token) * p.pitch + f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (f + e >= p.n_out) break;
      Elem<DT>::store(p.h + to + e, a[e] * fast_sigmoid(a[e]) * b[e]);
      if (p.a == nullptr) continue;
      if (p.wide) static_cast<float*>(p.a)[kept + e] = a[e], static_cast<float*>(p.b)[kept + e] = b[e];
      else Elem<DT>::store(static_cast<uint16_t*>(p.a) + kept + e, a[e]), Elem<DT>::store(static_cast<uint16_t*>(p.b) + kept + e, b[e]);
    }
  }
}

// 9 to 16 tokens with their rows in LDS: a workgroup for each CU walks the groups of 8 features.  The next group's weights are asked for in front of the current one's
// products, but waited for there too: the requests lie behind branches (rows' ends, the last group), and the compiler waits for all that it cannot count.  So a group's
// time is its weights' way from memory and the waves' meeting, one after the other; the variant of eight steps also keeps three addresses in
// scratch.  Read again for every group, as above, so many tokens are half as many bytes as the weights
// and more; fewer cost less than the part-filled last walk here.  (us, above / here, weights from memory, 8, 12, 16 tokens: 4096 -> 11008 47 / 47, 50 / 47.5, 52.8 / 48.6, 2048 -> 5504 12.4 / 13.5,
// 13.8 / 13.9, 15.8 / 14.3, 1536 -> 40000 63 / 60, 67 / 62, 70 / 62; 1024 -> 2752 the same.)  STEPS: of 32 k for each wave, at most.
// A row's chunk c of 16 bytes is at c ^ row: sixteen lanes on different banks.
constexpr int kRestWaves = 16;
__host__ __device__ constexpr int resident_pitch(int n_in) { return (n_in + 127) / 128 * 128; }
template <int DT, int STEPS>
__global__ __launch_bounds__(kRestWaves * kWave) void gated_resident_kernel(const FewParams p, int groups) {
  extern __shared__ __align__(16) char smem[];
  constexpr int kThreadsHere = kRestWaves * kWave;
  const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave), r = lane % 16, g = lane / 16;
  f32x4* const sums = reinterpret_cast<f32x4*>(smem);  // [2][wave][lane]
  uint16_t* const rows = reinterpret_cast<uint16_t*>(smem + 2 * kRestWaves * kWave * sizeof(f32x4));
  const int pitch = resident_pitch(p.n_in), steps = (p.n_in + 31) / 32;
  const auto weights = [&](int group, u32x4* w) {
    const uint16_t* const row = (r < 8 ? p.w1 : p.w3) + static_cast<int64_t>(min(8 * group + r % 8, p.n_out - 1)) * p.n_in;
#pragma unroll
    for (int j = 0; j < STEPS; ++j) {
      const int k = 32 * (wave + j * kRestWaves) + 8 * g;
      w[j] = k < p.n_in ? *reinterpret_cast<const u32x4*>(row + k) : u32x4{0, 0, 0, 0};
    }
  };
  u32x4 w[STEPS], next[STEPS];
  int group = blockIdx.x;
  weights(group, w);
  const int per = p.n_in / 8;
  for (int i = tid; i < p.tokens * per; i += kThreadsHere) {
    const int t = i / per, c = i - t * per;
    *reinterpret_cast<u32x4*>(rows + t * pitch + 8 * (c ^ t)) = *reinterpret_cast<const u32x4*>(p.x + static_cast<int64_t>(t) * p.n_in + 8 * c);
  }
  __syncthreads();
  const int token = min(r, p.tokens - 1);
  const uint16_t* const x = rows + token * pitch;
  for (int turn = 0; group < groups; turn ^= 1) {
    const int ahead = group + static_cast<int>(gridDim.x);
    if (ahead < groups) weights(ahead, next);
    f32x4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < STEPS; ++j) {
      const int s = wave + j * kRestWaves;
      if (s >= steps) break;
      const int k = 32 * s;
      const u32x4 v = k + 8 * g < p.n_in ? *reinterpret_cast<const u32x4*>(x + 8 * ((4 * s + g) ^ token)) : u32x4{0, 0, 0, 0};
      acc = mma16<DT>(w[j], v, acc);
    }
    f32x4* const mine = sums + turn * kRestWaves * kWave;
    mine[wave * kWave + lane] = acc;
    __syncthreads();
    // values 0 .. 3 of lanes 0 .. 31 are a, of lanes 32 on b
    if (tid < 128) {
      const float* const from = reinterpret_cast<const float*>(mine) + tid;
      float a = 0.f, b = 0.f;
#pragma unroll
      for (int q = 0; q < kRestWaves; ++q) a += from[q * 4 * kWave], b += from[q * 4 * kWave + 128];
      const int t = tid / 4 % 16, f = 8 * group + 4 * (tid / 64) + tid % 4;
      if (t < p.tokens && f < p.n_out) {
        Elem<DT>::store(p.h + static_cast<int64_t>(t) * p.n_out + f, a * fast_sigmoid(a) * b);
        if (p.a != nullptr) {
          const int64_t kept = static_cast<int64_t>(t) * p.pitch + f;
          if (p.wide) static_cast<float*>(p.a)[kept] = a, static_cast<float*>(p.b)[kept] = b;
          else Elem<DT>::store(static_cast<uint16_t*>(p.a) + kept, a), Elem<DT>::store(static_cast<uint16_t*>(p.b) + kept, b);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < STEPS; ++j) w[j] = next[j];
    group = ahead;
  }
}
constexpr size_t resident_lds(int tokens, int n_in) { return 2 * kRestWaves * kWave * sizeof(f32x4) + static_cast<size_t>(tokens) * resident_pitch(n_in) * 2; }
template <int DT, int STEPS>
int launch_resident(const FewParams& p, int cus, hipStream_t s) {
  const size_t lds = resident_lds(p.tokens, p.n_in);
  const int groups = (p.n_out + 7) / 8;
  MEGA_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&gated_resident_kernel<DT, STEPS>), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds)));
  gated_resident_kernel<DT, STEPS><<<std::min(groups, cus), kRestWaves * kWave, lds, s>>>(p, groups);
  MEGA_CHECK_LAUNCH();
  return MEGA_OK;
}

template <int DT, int NT, int FT>
int launch_few(const FewParams& p, hipStream_t s) {
  const dim3 grid((p.n_out + 8 * FT - 1) / (8 * FT)), block(kFewWaves * kWave);
  if (p.n_in % 8 == 0) gated_few_kernel<DT, NT, FT, true><<<grid, block, 0, s>>>(p);
  else gated_few_kernel<DT, NT, FT, false><<<grid, block, 0, s>>>(p);
  MEGA_CHECK_LAUNCH();
  return MEGA_OK;
}
// Groups of 8 features of a workgroup: the fewer, the more workgroups; the more, the fewer times the tokens are read.  Whatever leaves the
// CU with the most features the fewest of them, and of equals the larger: us, one / two groups, 1 and 16 tokens: 4096 -> 11008 (6 / 6
// groups a CU) 36.7 / 36.2 and 57.8 / 46.5, 2048 -> 5504 (3 / 4) 10.4 / 12.5 and 14.1 / 16.8, 1024 -> 2752 (2 / 2) 4.9 / 4.7 and 6.2 / 5.3; two / four
// groups, 32 tokens 60 / 62, 18.8 / 16.7, 6.4 / 8.3.
template <int DT, int NT, int FT>
int few_of(const FewParams& p, int cus, hipStream_t s) {
  const auto most = [&](int groups) { return ((p.n_out + 8 * groups - 1) / (8 * groups) + cus - 1) / cus * groups; };
  return most(2 * FT) <= most(FT) ? launch_few<DT, NT, 2 * FT>(p, s) : launch_few<DT, NT, FT>(p, s);
}
template <int DT>
int few_tokens(const FewParams& p, hipStream_t s) {
  int dev = 0, cus = 0;
  MEGA_CHECK_HIP(hipGetDevice(&dev));
  MEGA_CHECK_HIP(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev));
  static_assert(resident_lds(16, 4096) <= 160 * 1024, "fits the LDS");
  if (p.tokens > 8 && p.tokens <= 16 && p.n_in % 8 == 0 && p.n_in > 1024 && p.n_in <= 4096) return p.n_in <= 2048 ? launch_resident<DT, 4>(p, cus, s) : launch_resident<DT, 8>(p, cus, s);
  if (p.tokens <= 16) return few_of<DT, 1, 1>(p, cus, s);
  if (p.tokens <= 32) return few_of<DT, 2, 2>(p, cus, s);
  return few_of<DT, 4, 2>(p, cus, s);
}

// ---- rows of whole 16-byte pieces -----------------------------------------------------------------------
constexpr int kThreads = 256;

// Matrices copied in one launch, 16 bytes a thread: dst (rows, times, to) = src (rows, from), zeros behind column `from`; `to` whole
// pieces, dst on 16-byte boundaries.
struct Copies {
  struct One {
    const uint16_t* src;
    uint16_t* dst;
    uint32_t pieces, blocks;  // (operands have fewer than 2^30 elements); workgroups of this one and of those in front
    int from, to, times;
  } one[3];
  int count;
  void add(const uint16_t* src, uint16_t* dst, int64_t rows, int64_t from, int64_t to, int times = 1) {
    const uint32_t before = count > 0 ? one[count - 1].blocks : 0, pieces = static_cast<uint32_t>(rows * times * (to / 8));
    one[count++] = {src, dst, pieces, before + (pieces + kThreads - 1) / kThreads, static_cast<int>(from), static_cast<int>(to), times};
  }
};
__global__ __launch_bounds__(kThreads) void copies_kernel(const Copies c) {
  for (uint32_t block = blockIdx.x; block < c.one[c.count - 1].blocks; block += gridDim.x) {
    int m = 0;
    while (block >= c.one[m].blocks) ++m;
    const Copies::One& o = c.one[m];
    const uint32_t at = (m > 0 ? block - c.one[m - 1].blocks : block) * kThreads + threadIdx.x, per = static_cast<uint32_t>(o.to) / 8, row = at / per;
    if (at < o.pieces)
      *reinterpret_cast<u32x4*>(o.dst + 8 * static_cast<int64_t>(at)) = eight<false>(o.src + static_cast<int64_t>(row / o.times) * o.from, static_cast<int>(at - row * per) * 8, o.from);
  }
}
constexpr unsigned kMostBlocks = 16384;
int copy_all(const Copies& c, hipStream_t s) {
  if (c.count == 0) return MEGA_OK;
  copies_kernel<<<std::min(c.one[c.count - 1].blocks, kMostBlocks), kThreads, 0, s>>>(c);
  MEGA_CHECK_LAUNCH();
  return MEGA_OK;
}

// ---- the gate's backward --------------------------------------------------------------------------------
// STREAM: what is read once and written past the memory-side cache
template <bool STREAM, typename T>
__device__ __forceinline__ T read(const void* p) {
  if constexpr (STREAM) return __builtin_nontemporal_load(static_cast<const T*>(p));
  else return *static_cast<const T*>(p);
}
template <bool STREAM>
__device__ __forceinline__ void write(uint16_t* p, uint4 v) {
  if constexpr (STREAM) __builtin_nontemporal_store(__builtin_bit_cast(u32x4, v), reinterpret_cast<u32x4*>(p));
  else *reinterpret_cast<uint4*>(p) = v;
}
template <int DT, bool WIDE, bool STREAM>
__device__ __forceinline__ void kept_eight(const void* p, int64_t at, float* v) {
  if constexpr (!WIDE) {
    unpack8<DT>(__builtin_bit_cast(uint4, read<STREAM, u32x4>(static_cast<const uint16_t*>(p) + at)), v);
  } else {
    const f32x4 lo = read<STREAM, f32x4>(static_cast<const float*>(p) + at), hi = read<STREAM, f32x4>(static_cast<const float*>(p) + at + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = lo[e], v[4 + e] = hi[e];
  }
}
// What rounding v to the type has left of it (none where that is no number)
template <int DT>
__device__ __forceinline__ void remainders(const float* v, uint4 rounded, float* r) {
  unpack8<DT>(rounded, r);
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = fabsf(r[e]) < __builtin_inff() ? v[e] - r[e] : 0.f;
}
// da | db (tokens, TERMS, 2 h) from dh (tokens, n) and a, b (tokens, pitch): 8 elements a thread, zeros from column n on
template <int DT, bool WIDE, int TERMS, bool STREAM>
__global__ __launch_bounds__(kThreads) void gate_grad_kernel(const uint16_t* dh, const void* a, const void* b, uint16_t* g2,
                                                            int64_t tokens, int n, int pitch, int h) {
  const uint32_t per = static_cast<uint32_t>(h) / 8, pieces = static_cast<uint32_t>(tokens) * per;  // (fewer than 2^30 elements of da | db)
  for (uint32_t i = blockIdx.x * kThreads + threadIdx.x; i < pieces; i += gridDim.x * kThreads) {
    const int64_t row = i / per;
    const int k = static_cast<int>(i % per) * 8;
    float g[8], u[8], v[8], du[8], dv[8];
    if (k < pitch) {
      unpack8<DT>(__builtin_bit_cast(uint4, eight<false>(dh + row * n, k, n)), g);
      kept_eight<DT, WIDE, STREAM>(a, row * pitch + k, u);
      kept_eight<DT, WIDE, STREAM>(b, row * pitch + k, v);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float s = fast_sigmoid(u[e]);
      dv[e] = k + e < n ? g[e] * u[e] * s : 0.f;
      du[e] = k + e < n ? g[e] * v[e] * s * (1.f + u[e] * (1.f - s)) : 0.f;
    }
    uint16_t* const to = g2 + row * (TERMS * 2) * h + k;
    const uint4 a16 = pack8<DT>(du), b16 = pack8<DT>(dv);
    write<STREAM>(to, a16);
    write<STREAM>(to + h, b16);
    if constexpr (TERMS == 2) {
      remainders<DT>(du, a16, g);
      remainders<DT>(dv, b16, u);
      write<STREAM>(to + 2 * h, pack8<DT>(g));
      write<STREAM>(to + 3 * h, pack8<DT>(u));
    }
  }
}

// ---- sizes ----------------------------------------------------------------------------------------------
int64_t up(int64_t n, int64_t step) { return (n + step - 1) / step * step; }
constexpr int64_t kMost = 1ll << 30;  // elements of an operand: the product kernels' byte offsets have 32 bits

// What a call lays out in its workspace, in bytes from its start (0 bytes where a piece is not needed).
struct Room {
  int64_t bytes = 0;
  int64_t take(int64_t n) {
    const int64_t at = bytes;
    bytes += up(n, 256);
    return at;
  }
};
struct Forward {
  int64_t k, rows;  // n_in with its padding, tokens of a launch
  int64_t x, w1, w3, parts, bytes;
  Forward(int64_t tokens, int64_t n_in, int64_t n_out) {
    Room room;
    k = n_in, rows = tokens, x = w1 = w3 = parts = 0;
    if (!few(tokens, n_in, n_out)) {
      k = n_in % 8 == 0 ? n_in : up(n_in, 64);
      rows = std::min(tokens, std::max<int64_t>((kMost - 1) / k / 256 * 256, 256));
      if (k != n_in) {
        x = room.take(2 * rows * k);
        w1 = room.take(2 * n_out * k);
        w3 = room.take(2 * n_out * k);
      }
      parts = room.take(std::max(gated_parts_bytes(rows, k, n_out), gated_parts_bytes(std::max<int64_t>(tokens % rows, 1), k, n_out)));
    }
    bytes = room.bytes;
  }
};
// Backward: the gradients of a and b beside each other, (tokens, 2 h), for gated_tiles.hip.  (Small sizes too: networks of 1024 -> 2752
// and up are faster so than by the products of attention.hip, whose tiles are small, by 10 to 50 % up to 1024 tokens; 512 -> 1408 up to 20 % slower from
// 512 tokens on.)
// Few tokens: two terms each, what rounding left beside the rounded, so that the results are as good as rounded once; the roundings of few values
// average out less.  The second term's rows are beside the first's in dx's tile, which is not full anyway.  (us, one / two terms, dx and dw of 16 tokens:
// 1024 -> 2752 27 / 29, 2048 -> 5504 41 / 43, 4096 -> 11008 99 / 101.)
constexpr int64_t kTwoTerms = 64;
// Beyond the memory-side cache nothing of the gate's pass is worth keeping (us with the gradient of narrow rows, kept / past it: 32768 x 11008 1355 / 1260, 8192 x 5504
// 174 / 162, 4084 x 2752 51 / 54).
constexpr int64_t kCacheBytes = 256 << 20;
struct Backward {
  int terms;
  int64_t h, k, rows;  // n_out and n_in with their padding, tokens of a launch
  int64_t g, w1, w3, x, sums, parts, bytes;  // sums: float32, of the weights' gradients between launches
  Backward(int64_t tokens, int64_t n_in, int64_t n_out, int what) {  // (what: 1 dx, 2 dw1, 4 dw3)
    Room room;
    terms = tokens <= kTwoTerms ? 2 : 1;
    h = up(n_out, 64), k = up(n_in, 8);
    rows = std::min(tokens, std::max<int64_t>((kMost - 1) / std::max(2 * h, k) / 256 * 256, 256));
    g = room.take(2 * rows * terms * 2 * h);
    w1 = (what & 1) && k != n_in ? room.take(2 * n_out * k) : 0;
    w3 = (what & 1) && k != n_in ? room.take(2 * n_out * k) : 0;
    x = what > 1 && (k != n_in || terms > 1) ? room.take(2 * terms * rows * k) : 0;
    sums = what > 1 && tokens > rows ? room.take(4 * n_out * n_in * (what >= 6 ? 2 : 1)) : 0;
    // (the products run one after the other)
    int64_t most = 0;
    for (const int64_t n : {rows, std::max<int64_t>(tokens % rows, 1)}) {
      if (what & 1) most = std::max(most, gated_tiles_bytes(1, n, n_in, n_out, 2, terms));
      if (what > 1) most = std::max(most, gated_tiles_bytes(2, n, n_in, n_out, what >= 6 ? 2 : 1, terms));
    }
    parts = room.take(most);
    bytes = room.bytes;
  }
};

int check(const char* who, int dtype, int64_t tokens, int64_t n_in, int64_t n_out) {
  MEGA_CHECK_ARG(dtype == MEGA_BF16 || dtype == MEGA_F16, "%s: bfloat16 or float16 tensors", who);
  MEGA_CHECK_ARG(tokens >= 1 && n_in >= 1 && n_out >= 1 && tokens < (1ll << 31) && n_in <= (1 << 20) && n_out <= (1 << 20) &&
                     up(n_in, 64) * 2 * up(n_out, 64) < kMost,
                 "%s: bad sizes", who);
  return MEGA_OK;
}
bool aligned16(const void* q) { return reinterpret_cast<uintptr_t>(q) % 16 == 0; }

}  // namespace
}  // namespace mega

using namespace mega;

extern "C" int64_t mega_gated_linear_workspace_bytes(int64_t tokens, int64_t n_in, int64_t n_out, int backward) {
  if (tokens < 1 || n_in < 1 || n_out < 1 || n_in > (1 << 20) || n_out > (1 << 20) || tokens >= (1ll << 31) || up(n_in, 64) * 2 * up(n_out, 64) >= kMost) return 0;
  return backward == 0 ? Forward(tokens, n_in, n_out).bytes : Backward(tokens, n_in, n_out, backward).bytes;
}

extern "C" int mega_gated_linear_fwd(const void* x_, const void* w1_, const void* w3_, int dtype, int64_t tokens, int64_t n_in, int64_t n_out,
                                     void* h_, void* a, void* b, int kept, void* workspace, void* stream) {
  if (const int rc = check("mega_gated_linear_fwd", dtype, tokens, n_in, n_out); rc != MEGA_OK) return rc;
  MEGA_CHECK_ARG(x_ && w1_ && w3_ && h_ && (a == nullptr) == (b == nullptr), "mega_gated_linear_fwd: null pointer");
  MEGA_CHECK_ARG(kept == dtype || kept == MEGA_F32, "mega_gated_linear_fwd: the products are kept in the operands' type or in float32");
  for (const void* q : {x_, w1_, w3_, static_cast<const void*>(a), static_cast<const void*>(b), static_cast<const void*>(workspace)}) MEGA_CHECK_ARG(aligned16(q), "mega_gated_linear_fwd: misaligned pointer");
  const uint16_t *x = static_cast<const uint16_t*>(x_), *w1 = static_cast<const uint16_t*>(w1_), *w3 = static_cast<const uint16_t*>(w3_);
  uint16_t* h = static_cast<uint16_t*>(h_);
  const bool wide = kept == MEGA_F32;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (few(tokens, n_in, n_out)) {
    const FewParams p{x, w1, w3, h, a, b, static_cast<int>(tokens), static_cast<int>(n_in), static_cast<int>(n_out), wide, static_cast<int>(gated_pitch(n_out))};
    return dtype == MEGA_BF16 ? few_tokens<MEGA_BF16>(p, s) : few_tokens<MEGA_F16>(p, s);
  }
  const Forward f(tokens, n_in, n_out);
  MEGA_CHECK_ARG(workspace != nullptr || f.bytes == 0, "mega_gated_linear_fwd: null workspace");
  char* const ws = static_cast<char*>(workspace);
  const auto at = [&](int64_t offset) { return reinterpret_cast<uint16_t*>(ws + offset); };
  const bool padded = f.k != n_in;
  for (int64_t t = 0; t < tokens; t += f.rows) {
    const int64_t n = std::min(f.rows, tokens - t);
    const uint16_t* rows = x + t * n_in;
    if (padded) {
      Copies c{};
      c.add(rows, at(f.x), n, n_in, f.k);
      if (t == 0) {
        c.add(w1, at(f.w1), n_out, n_in, f.k);
        c.add(w3, at(f.w3), n_out, n_in, f.k);
        w1 = at(f.w1), w3 = at(f.w3);
      }
      if (const int rc = copy_all(c, s); rc != MEGA_OK) return rc;
      rows = at(f.x);
    }
    const auto rows_of = [&](void* q) { return q == nullptr ? nullptr : static_cast<char*>(q) + t * gated_pitch(n_out) * (wide ? 4 : 2); };
    if (const int rc = gated_product(dtype, rows, w1, w3, n, f.k, n_out, h + t * n_out, rows_of(a), rows_of(b), wide, reinterpret_cast<float*>(ws + f.parts), s);
        rc != MEGA_OK)
      return rc;
  }
  return MEGA_OK;
}

extern "C" int mega_gated_linear_bwd(const void* dh_, const void* x_, const void* w1_, const void* w3_, const void* a, const void* b, int kept, int dtype,
                                     int64_t tokens, int64_t n_in, int64_t n_out, void* dx_, void* dw1_, void* dw3_, void* workspace, void* stream) {
  if (const int rc = check("mega_gated_linear_bwd", dtype, tokens, n_in, n_out); rc != MEGA_OK) return rc;
  MEGA_CHECK_ARG(dh_ && x_ && w1_ && w3_ && a && b && workspace, "mega_gated_linear_bwd: null pointer");
  MEGA_CHECK_ARG(kept == dtype || kept == MEGA_F32, "mega_gated_linear_bwd: the products are kept in the operands' type or in float32");
  for (const void* q : {x_, w1_, w3_, a, b, static_cast<const void*>(workspace)})
    MEGA_CHECK_ARG(aligned16(q), "mega_gated_linear_bwd: misaligned pointer");
  const auto u = [](const void* q) { return static_cast<const uint16_t*>(q); };
  const uint16_t *dh = u(dh_), *x = u(x_), *w1 = u(w1_), *w3 = u(w3_);
  uint16_t *dx = static_cast<uint16_t*>(dx_), *dw1 = static_cast<uint16_t*>(dw1_), *dw3 = static_cast<uint16_t*>(dw3_);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int what = (dx != nullptr) + 2 * (dw1 != nullptr) + 4 * (dw3 != nullptr);
  if (what == 0) return MEGA_OK;
  const Backward f(tokens, n_in, n_out, what);
  char* const ws = static_cast<char*>(workspace);
  const auto at = [&](int64_t offset) { return reinterpret_cast<uint16_t*>(ws + offset); };
  const int64_t h = f.h, k = f.k;
  for (int64_t t = 0; t < tokens; t += f.rows) {
    const int64_t n = std::min(f.rows, tokens - t);
    uint16_t* const g = at(f.g);
    const int64_t pitch = gated_pitch(n_out), at0 = t * n_out;
    const uint16_t* rows = x + t * n_in;
    if (k != n_in || f.terms > 1) {
      Copies c{};
      if (dx != nullptr && t == 0 && k != n_in) {
        c.add(w1, at(f.w1), n_out, n_in, k);
        c.add(w3, at(f.w3), n_out, n_in, k);
        w1 = at(f.w1), w3 = at(f.w3);
      }
      if (what > 1) c.add(rows, at(f.x), n, n_in, k, f.terms), rows = at(f.x);
      if (const int rc = copy_all(c, s); rc != MEGA_OK) return rc;
    }
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>((n * (h / 8) + kThreads - 1) / kThreads, kMostBlocks));
    const bool wide = kept == MEGA_F32;
    const auto rows_of = [&](const void* q) { return static_cast<const char*>(q) + t * pitch * (wide ? 4 : 2); };
    const auto launch = [&](auto kernel) { kernel<<<grid, kThreads, 0, s>>>(dh + at0, rows_of(a), rows_of(b), g, n, (int)n_out, (int)pitch, (int)h); };
    const auto of_type = [&](auto dt, auto is_wide) {
      constexpr int DT = decltype(dt)::value;
      constexpr bool WIDE = decltype(is_wide)::value;
      if (f.terms == 2) launch(gate_grad_kernel<DT, WIDE, 2, false>);
      else if (n * h * (WIDE ? 14 : 10) > kCacheBytes) launch(gate_grad_kernel<DT, WIDE, 1, true>);
      else launch(gate_grad_kernel<DT, WIDE, 1, false>);
    };
    const auto of_width = [&](auto dt) { wide ? of_type(dt, std::true_type()) : of_type(dt, std::false_type()); };
    if (dtype == MEGA_BF16) of_width(std::integral_constant<int, MEGA_BF16>());
    else of_width(std::integral_constant<int, MEGA_F16>());
    MEGA_CHECK_LAUNCH();
    float* const parts = reinterpret_cast<float*>(ws + f.parts);
    if (dx != nullptr)
      if (const int rc = gated_tiles_input(dtype, g, w1, w3, n, n_in, n_out, k, f.terms, dx + t * n_in, parts, s); rc != MEGA_OK) return rc;
    if (what > 1)
      if (const int rc = gated_tiles_weight(dtype, g, rows, n, n_in, n_out, k, f.terms, dw1, dw3, tokens > f.rows ? reinterpret_cast<float*>(ws + f.sums) : nullptr, t == 0,
                                            t + n == tokens, parts, s);
          rc != MEGA_OK)
        return rc;
  }
  return MEGA_OK;
}
