// The gated product of many tokens in tiles of 256 tokens x 128 features of both matrices (gated_linear.hip has the formulas).
//
// Eight waves of 128 x 64 accumulators: 32 features of w1 and the same 32 of w3 beside each other, so that a lane has a and b
// of its elements.  Slabs of 64 k go from memory straight into LDS, a wave's products are 32 x 32 x 16; the layouts in LDS are those of
// the product kernels with two k-contiguous operands (attention.hip): rows of 128 bytes, whose 16-byte chunk c lies at position
// c ^ ((row >> 1) & 7); the rows of the two matrices lie 32 by 32 in turn.
//
// A workgroup's tiles are one line of slabs: the first slabs of a tile are on their way while the last ones of the tile before are
// worked on, and the gate and the stores, taken straight from the accumulators, run meanwhile.  The slabs of x and of the matrices go
// round in five buffers of 32 KB, all of the LDS, so that the requests of a slab can be spread over three of its four steps: a request
// of 1 KB takes the CU's memory path 16 cycles, the 64 of a slab half of its time, and sent under one step, as two buffers for whole slabs
// want it, they hold up the waves.  32768 tokens, 4096 -> 11008, nothing kept: 4.23 ms, 1.40 PFLOP/s, the matrix pipe 86 % busy at the
// 1.53 GHz that the power limit leaves (two buffers 4.43 ms, 75 % at 1.66; the library's product alone, without gate and at
// the same time, 3.86 ms, 86 % at 1.65).  Four waves of 128 x 128, with a third fewer reads of LDS, take the same time.
// What remains exposed are the stores: a and b in float32 0.75 ms.
#include "common.hpp"
#include "gated.hpp"
#include "gemm_params.hpp"

namespace mega {
namespace {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <int DT>
__device__ __forceinline__ floatx16 mma32(u32x4 a, u32x4 b, floatx16 c) {
  if constexpr (DT == MEGA_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

constexpr int kThreads = 512, kRows = 256, kCols = 128, kK = 64;
constexpr uint32_t kOperandBytes = 256 * kK * 2, kRing = 5 * kOperandBytes;
constexpr size_t kLds = kRing;
static_assert(kLds <= 160 * 1024, "fits the LDS");

// 64 lanes' 16 bytes from base + offset to 1 KB of LDS (its address in M0).  Assembly, since the compiler would wait for all of
// them in front of every read of LDS; the waits are the explicit ones below.
__device__ __forceinline__ void load_to_lds16(const char* base, uint32_t offset, uint32_t lds_dst) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(offset), "s"(base), "s"(lds_dst));
}

__device__ __forceinline__ float gated(float a, float b) { return a * fast_sigmoid(a) * b; }
template <int DT>
__device__ __forceinline__ uint2 pack4(float a, float b, float c, float d) {
  if constexpr (DT == MEGA_BF16) return uint2{pack_bf16x2(a, b), pack_bf16x2(c, d)};
  return uint2{static_cast<uint32_t>(float_to_f16_bits(a)) | static_cast<uint32_t>(float_to_f16_bits(b)) << 16,
               static_cast<uint32_t>(float_to_f16_bits(c)) | static_cast<uint32_t>(float_to_f16_bits(d)) << 16};
}

// Four 16-bit values of columns 8 q + 4 (lane / 32) of a row, for two q: lanes of the lower half get columns 8 q .. + 7 of the
// first, those of the upper half of the second.
__device__ __forceinline__ u32x4 rows_of_eight(uint2 first, uint2 second) {
  const auto x = __builtin_amdgcn_permlane32_swap(first.x, second.x, false, false);
  const auto y = __builtin_amdgcn_permlane32_swap(first.y, second.y, false, false);
  return u32x4{x[0], y[0], x[1], y[1]};
}

// KEEP: 0 h alone, 1 a and b in the operands' type as well, 2 in float32
template <int DT, int KEEP>
__global__ __launch_bounds__(kThreads) void gated_tiles_kernel(const GatedTiles p) {
  extern __shared__ __align__(16) char smem[];
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wm = wave / 4, wn = wave % 4, g = lane / 32, r = lane % 32;
  // a contiguous eighth of the tiles to each XCD, walked by its workgroups in turn; bands of eight column tiles
  const int G = static_cast<int>(gridDim.x), lin = static_cast<int>(blockIdx.x);
  int item, it_hi, it_step;
  if (G % kXcds == 0) {
    const int xcd = lin % kXcds;
    item = static_cast<int>(static_cast<int64_t>(p.tiles) * xcd / kXcds) + lin / kXcds;
    it_hi = static_cast<int>(static_cast<int64_t>(p.tiles) * (xcd + 1) / kXcds);
    it_step = G / kXcds;
  } else {
    item = lin, it_hi = p.tiles, it_step = G;
  }
  if (item >= it_hi) return;
  const auto place = [&](int it, int* m0, int* h0) {
    constexpr int kBand = 8;
    const int band = kBand * p.row_tiles, b0 = it / band, rest = it % band, width = min(kBand, p.col_tiles - b0 * kBand);
    *m0 = rest / width * kRows;
    *h0 = (b0 * kBand + rest % width) * kCols;
  };

  // memory side: a wave sends 1 KB pieces (8 rows) wave, wave + 8, .. of either operand; those of the matrices are all of one of them
  const char* const xb = reinterpret_cast<const char*>(p.x);
  const char* const wb = reinterpret_cast<const char*>(wave & 4 ? p.w3 : p.w1);
  const uint32_t pitch = static_cast<uint32_t>(p.n_in) * 2;
  uint32_t offx[4], offw[4];
  const auto offsets = [&](int m0, int h0) {
    const int row = 8 * wave + lane / 8;
    const uint32_t chunk = ((lane & 7) ^ (row >> 1 & 7)) * 16;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      offx[i] = static_cast<uint32_t>(min(m0 + row + 64 * i, p.tokens - 1)) * pitch + chunk;
      offw[i] = static_cast<uint32_t>(min(h0 + (row & 31) + 32 * i, p.n_out - 1)) * pitch + chunk;
    }
  };
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)(smem))));
  const uint32_t lds_wave = lds0 + wave * 1024;
  // the ring: operand slabs x 0, matrices 0, x 1, matrices 1, .. in buffers 0 .. 4 in turn
  const auto behind = [&](uint32_t at, uint32_t buffers) { return at + buffers * kOperandBytes >= kRing ? at + buffers * kOperandBytes - kRing : at + buffers * kOperandBytes; };
  const auto request_x = [&](uint32_t slab, uint32_t to, int i) { load_to_lds16(xb + slab * 128, offx[i], lds_wave + to + i * 8192); };
  const auto request_w = [&](uint32_t slab, uint32_t to, int i) { load_to_lds16(wb + slab * 128, offw[i], lds_wave + to + i * 8192); };

  // fragment side: k-step `set` of a slab takes k = 16 set + 8 g + e; its chunk 2 set + g lies at (g ^ swizzle) ^ 2 set
  const uint32_t fra = (wm * 128 + r) * 128 + (g ^ (r >> 1 & 7)) * 16, frb = (wn * 64 + r) * 128 + (g ^ (r >> 1 & 7)) * 16;
  const auto read = [&](uint32_t at) {
    return *reinterpret_cast<const __attribute__((address_space(3))) u32x4*>(static_cast<uintptr_t>(at));
  };
  u32x4 fa0[4], fb0[2], fa1[4], fb1[2];
  const auto fread = [&](u32x4* fa, u32x4* fb, uint32_t in_x, uint32_t in_w, int set, int i) {
    fa[i] = read((fra ^ (set * 32)) + lds0 + in_x + i * 32 * 128);
    if (i < 2) fb[i] = read((frb ^ (set * 32)) + lds0 + in_w + i * 32 * 128);
  };
  floatx16 acc[4][2];
  const auto mma = [&](const u32x4* fa, const u32x4* fb, int n) { acc[n / 2][n % 2] = mma32<DT>(fb[n % 2], fa[n / 2], acc[n / 2][n % 2]); };

  const int slabs = p.n_in / kK;
  int m0, h0;
  place(item, &m0, &h0);
  offsets(m0, h0);
  // `ahead`: the slab that is asked for next, of a tile `next` further on once it has reached `slabs` (behind the last tile the
  // same one again, which nobody reads)
  int ahead = 0, next = item + it_step;
  const auto turn = [&]() {
    if (ahead < slabs) return;
    ahead = 0;
    if (next < it_hi) {
      int m, h;
      place(next, &m, &h);
      offsets(m, h);
    }
    next += it_step;
  };
  uint32_t in_x = 0;  // the buffer of x's slab that is worked on; its matrices' is the next, then come the next slab's
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    turn();
#pragma unroll
    for (int i = 0; i < 4; ++i) request_x(ahead, 2 * q * kOperandBytes, i);
#pragma unroll
    for (int i = 0; i < 4; ++i) request_w(ahead, (2 * q + 1) * kOperandBytes, i);
    ++ahead;
  }
  asm volatile("s_waitcnt vmcnt(8)\n\ts_barrier" ::: "memory");
#pragma unroll
  for (int i = 0; i < 4; ++i) fread(fa0, fb0, 0, kOperandBytes, 0, i);

  // A slab's four k-steps.  The fragments of the next step are read under the products of the current one.  The slab behind the
  // next: x's under the first two steps, into the buffer that the last slab's matrices have left; the matrices' under the last one,
  // into the buffer of this slab's x, which all waves have read by then.  (Requests for 1 KB keep the memory path 16 cycles each, all 64 of a slab half the
  // slab's time: sent under one step, as with two buffers for whole slabs, they hold up the waves.)
#define MEGA_SGB(mask, n) __builtin_amdgcn_sched_group_barrier(mask, n, 0)
#define MEGA_READ_AND_MULTIPLY(FA, FB, NFA, NFB, SET)                      \
    _Pragma("unroll") for (int i = 0; i < 4; ++i) fread(NFA, NFB, in_x, in_w, (SET) + 1, i); \
    _Pragma("unroll") for (int n = 0; n < 4; ++n) mma(FA, FB, n);          \
    _Pragma("unroll") for (int sg = 0; sg < 3; ++sg) {                     \
      MEGA_SGB(0x008, 1);                                                  \
      MEGA_SGB(0x100, 2);                                                  \
    }                                                                      \
    MEGA_SGB(0x008, 1);                                                    \
    __builtin_amdgcn_sched_barrier(0);
  while (true) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    for (int s = 0; s < slabs; ++s) {
      const uint32_t in_w = behind(in_x, 1), next_x = behind(in_x, 2), next_w = behind(in_x, 3), last_w = behind(in_x, 4);
      turn();
      MEGA_READ_AND_MULTIPLY(fa0, fb0, fa1, fb1, 0)
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        if (n < 2) request_x(ahead, last_w, n);
        mma(fa0, fb0, 4 + n);
        __builtin_amdgcn_sched_barrier(0);
      }
      MEGA_READ_AND_MULTIPLY(fa1, fb1, fa0, fb0, 1)
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        if (n < 2) request_x(ahead, last_w, 2 + n);
        mma(fa1, fb1, 4 + n);
        __builtin_amdgcn_sched_barrier(0);
      }
      MEGA_READ_AND_MULTIPLY(fa0, fb0, fa1, fb1, 2)
#pragma unroll
      for (int n = 4; n < 8; ++n) mma(fa0, fb0, n);
      __builtin_amdgcn_sched_barrier(0);
      // the wave's pieces of the next slab have landed (x's of the one behind it may be on their way), its reads of this one have returned
      asm volatile("s_waitcnt vmcnt(4) lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        if (n < 4) fread(fa0, fb0, next_x, next_w, 0, n);
        if (n % 2 == 1) request_w(ahead, in_x, n / 2);
        mma(fa1, fb1, n);
        __builtin_amdgcn_sched_barrier(0);
      }
      ++ahead;
      in_x = next_x;
    }
    // the tile's elements: lane l has row l % 32 of a block of 32, register e the column 8 (e / 4) + 4 (l / 32) + e % 4
    const int col0 = h0 + wn * 32;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = m0 + wm * 128 + i * 32 + r;
      if (row >= p.tokens) continue;
      uint16_t* const h = p.h + static_cast<int64_t>(row) * p.n_out;
      const int64_t at = static_cast<int64_t>(row) * p.pitch;
#pragma unroll
      for (int q = 0; q < 4; q += 2) {
        uint2 v[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int e = 4 * (q + t);
          v[t] = pack4<DT>(gated(acc[i][0][e], acc[i][1][e]), gated(acc[i][0][e + 1], acc[i][1][e + 1]),
                           gated(acc[i][0][e + 2], acc[i][1][e + 2]), gated(acc[i][0][e + 3], acc[i][1][e + 3]));
        }
        const u32x4 eight = rows_of_eight(v[0], v[1]);
        const int col = col0 + 8 * (q + g);
        if (col + 8 <= p.n_out) {
          *reinterpret_cast<u32x4_any*>(h + col) = eight;
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (col + e < p.n_out) h[col + e] = static_cast<uint16_t>(eight[e / 2] >> (16 * (e % 2)));
        }
      }
#pragma unroll
      for (int j = 0; j < 2 && KEEP == 1; ++j)
#pragma unroll
        for (int q = 0; q < 4; q += 2) {
          const auto four = [&](int e) { return pack4<DT>(acc[i][j][e], acc[i][j][e + 1], acc[i][j][e + 2], acc[i][j][e + 3]); };
          const u32x4 eight = rows_of_eight(four(4 * q), four(4 * q + 4));
          const int col = col0 + 8 * (q + g);
          if (col < p.pitch) *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(j ? p.b : p.a) + at + col) = eight;
        }
#pragma unroll
      for (int j = 0; j < 2 && KEEP == 2; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int col = col0 + 8 * q + 4 * g;
          if (col < p.pitch)
            *reinterpret_cast<float4*>(static_cast<float*>(j ? p.b : p.a) + at + col) =
                make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
        }
    }
    item += it_step;
    if (item >= it_hi) break;
    place(item, &m0, &h0);
  }
#undef MEGA_READ_AND_MULTIPLY
#undef MEGA_SGB
  // (nothing may land in LDS that is another workgroup's by then)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

template <int DT, int KEEP>
int launch(const GatedTiles& p, int grid, hipStream_t s) {
  MEGA_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&gated_tiles_kernel<DT, KEEP>), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kLds)));
  gated_tiles_kernel<DT, KEEP><<<dim3(static_cast<unsigned>(grid)), kThreads, kLds, s>>>(p);
  MEGA_CHECK_LAUNCH();
  return MEGA_OK;
}

}  // namespace

int gated_tiles(int dtype, int keep, const GatedTiles& p, int grid, hipStream_t s) {
  if (dtype == MEGA_BF16) return keep == 0 ? launch<MEGA_BF16, 0>(p, grid, s) : keep == 1 ? launch<MEGA_BF16, 1>(p, grid, s) : launch<MEGA_BF16, 2>(p, grid, s);
  return keep == 0 ? launch<MEGA_F16, 0>(p, grid, s) : keep == 1 ? launch<MEGA_F16, 1>(p, grid, s) : launch<MEGA_F16, 2>(p, grid, s);
}

}  // namespace mega
