// The products of the gated half of a feed-forward network in tiles of 256 x 256, for many tokens (gated_linear.hip has the formulas):
//   kGate: h = silu(x w1^T) o (x w3^T): a tile is 256 tokens x 128 features of both matrices, whose rows lie 32 by 32 in turn, so that a lane has
//          a and b of its elements; the gate is taken from the accumulators
//   kInput: dx = da w1 + db w3, one sum along the features of both: da | db by rows, the matrices as they are (rows of k)
//   kWeight: dw1 = da^T x, dw3 = db^T x, one product of da | db and x, both as they are
//
// Eight waves of 128 x 64 accumulators.  Slabs of 64 k go from memory straight into LDS, through buffer descriptors: what lies
// behind a matrix arrives as zeros.  An operand with k along its rows lies in LDS in rows of 128 bytes, whose 16-byte chunk c is at
// position c ^ ((row >> 1) & 7); one whose rows are k in 64 rows of 512 bytes, chunk c at c ^ ((k & 3) << 2) ^ ((k >> 3 & 1) << 1), read
// back through the transposing read (sixteen lanes or rows at a time on different banks in both).
//
// A workgroup's tiles are one line of slabs: the first slabs of a tile are on their way while the last ones of the tile before are
// worked on, and the stores run meanwhile.  The operands' slabs go round in five buffers of 32 KB, all of the LDS, so that the requests of a slab can be
// spread over three quarters of its time: a request of 1 KB takes the CU's memory path 16 cycles, the 64 of a slab half of its time, and sent together,
// as two buffers for whole slabs want it, they hold up the waves (the matrix pipe 75 % busy, 86 % so).
// The products are 16 x 16 x 32: the power limit sets the clock, and 32 x 32 x 16 move twice the accumulators for the same operations
// (1.43 against 1.54 PFLOP/s).  32768 tokens, 4096 -> 11008, 5.9 TFLOP each: kGate 3.85 ms, as long as a general library takes for the two products
// without the gate (4.57 with a and b kept in float32: the stores of all units' tiles come together, 12 us of 100), kInput 3.8, kWeight 4.2 (twice
// the reads of LDS, 8 bytes each, for an operand whose rows are k).
#include "common.hpp"
#include "gated.hpp"
#include "gemm_params.hpp"

#include <algorithm>
#include <type_traits>

namespace mega {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short short4v __attribute__((ext_vector_type(4)));

template <int DT>
__device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (DT == MEGA_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

enum { kGate, kInput, kWeight, kInputTwo };  // (kInputTwo: kInput of two terms)
constexpr int kThreads = 512, kTileRows = 256, kK = 64, kBand = 8;
constexpr uint32_t kOperandBytes = 256 * kK * 2, kRing = 5 * kOperandBytes;
constexpr size_t kLds = kRing;
constexpr int64_t kPieceBytes = 256 * 256 * 4;
static_assert(kLds <= 160 * 1024, "fits the LDS");

// 64 lanes' 16 bytes from a buffer's offsets to 1 KB of LDS (its address in M0); zeros for offsets at and behind its end.  Assembly, since the
// compiler would wait for all of them in front of every read of LDS; the waits are the explicit ones below.
__device__ __forceinline__ u32x4 buffer_of(const void* base, uint32_t bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(base);
  return u32x4{static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(a))), static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(a >> 32) & 0xffff)),
               static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(bytes))), 0x00020000u};
}
__device__ __forceinline__ void load_to_lds16(u32x4 buffer, uint32_t offset, uint32_t lds_dst) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" : : "v"(offset), "s"(buffer), "s"(lds_dst));
}

__device__ __forceinline__ float gated(float a, float b) { return a * fast_sigmoid(a) * b; }
template <int DT>
__device__ __forceinline__ uint2 pack4(f32x4 v) {
  if constexpr (DT == MEGA_BF16) return uint2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
  return uint2{static_cast<uint32_t>(float_to_f16_bits(v[0])) | static_cast<uint32_t>(float_to_f16_bits(v[1])) << 16,
               static_cast<uint32_t>(float_to_f16_bits(v[2])) | static_cast<uint32_t>(float_to_f16_bits(v[3])) << 16};
}
// Four 16-bit values of columns 4 g .. + 3 of a row (g = lane / 16) for two blocks of 16 columns: 16 bytes at columns
// 16 (g & 1) + 8 (g >> 1) of the 32.
__device__ __forceinline__ u32x4 rows_of_eight(uint2 first, uint2 second) {
  const auto x = __builtin_amdgcn_permlane16_swap(first.x, second.x, false, false);
  const auto y = __builtin_amdgcn_permlane16_swap(first.y, second.y, false, false);
  return u32x4{x[0], y[0], x[1], y[1]};
}
// Eight elements of a row of any pitch, those in front of its end
__device__ __forceinline__ void store_eight(uint16_t* to, int left, u32x4 v) {
  if (left >= 8) {
    *reinterpret_cast<u32x4_any*>(to) = __builtin_bit_cast(u32x4_any, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < left) to[e] = static_cast<uint16_t>(v[e / 2] >> (16 * (e % 2)));
  }
}

// 16 rows x 64 accumulators of a wave in their places: lane l has row l % 16, columns 4 (l / 16) .. + 3 of each block of 16 (kGate: of a, a, b, b).
// KEEP (kGate): 0 h alone, 1 a and b in the operands' type as well, 2 in float32
template <int DT, int MODE, int KEEP>
__device__ __forceinline__ void finish(const GatedTiles& p, const f32x4* acc, int row0, int n0, int wn, int lane) {
  const int g = lane / 16, in32 = 16 * (g & 1) + 8 * (g >> 1), row = row0 + lane % 16;
  if (row >= p.m) return;
  if constexpr (MODE == kGate) {
    const int col0 = n0 + wn * 32, col = col0 + in32;
    const int64_t at = static_cast<int64_t>(row) * p.pitch;
    uint2 v[2];
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      const f32x4 a = acc[f], b = acc[2 + f];
      v[f] = pack4<DT>(f32x4{gated(a[0], b[0]), gated(a[1], b[1]), gated(a[2], b[2]), gated(a[3], b[3])});
    }
    store_eight(p.c + static_cast<int64_t>(row) * p.n + col, p.n - col, rows_of_eight(v[0], v[1]));
#pragma unroll
    for (int j = 0; j < 2 && KEEP == 1; ++j) {
      const u32x4 kept = rows_of_eight(pack4<DT>(acc[2 * j]), pack4<DT>(acc[2 * j + 1]));
      if (col < p.pitch) *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(j ? p.kept_b : p.kept_a) + at + col) = kept;
    }
#pragma unroll
    for (int j = 0; j < 2 && KEEP == 2; ++j)
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const int to = col0 + 16 * f + 4 * g;
        if (to < p.pitch) *reinterpret_cast<f32x4*>(static_cast<float*>(j ? p.kept_b : p.kept_a) + at + to) = acc[2 * j + f];
      }
  } else {
    // kWeight: rows behind n_out of either half are padding
    const bool second = MODE == kWeight && row >= p.half;
    const int in_half = second ? row - p.half : row;
    if (MODE == kWeight && in_half >= p.n_out) return;
    const int64_t at = static_cast<int64_t>(in_half) * p.cols;
    uint16_t* const to = (second ? p.c2 : p.c) + at;
#pragma unroll
    for (int f = 0; f < 4; f += 2) {
      uint2 v[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        f32x4 c = acc[f + t];
        if (MODE == kWeight && p.sum != nullptr) {
          float* const sum = p.sum + (second ? at + static_cast<int64_t>(p.n_out) * p.cols : at);
          const int col = n0 + wn * 64 + 16 * (f + t) + 4 * g;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (col + e >= p.cols) break;
            if (!p.first) c[e] += sum[col + e];
            if (!p.last) sum[col + e] = c[e];
          }
        }
        v[t] = pack4<DT>(c);
      }
      const int col = n0 + wn * 64 + 16 * f + in32;
      if (MODE == kWeight && !p.last) continue;
      store_eight(to + col, p.cols - col, rows_of_eight(v[0], v[1]));
    }
  }
}

template <int DT, int MODE, int KEEP>
__global__ __launch_bounds__(kThreads) void gated_tiles_kernel(const GatedTiles p) {
  constexpr bool kRowsA = MODE == kWeight, kRowsB = MODE != kGate;  // the operand's rows are k
  constexpr int kTileCols = MODE == kGate ? 128 : 256;
  extern __shared__ __align__(16) char smem[];
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wm = wave / 4, wn = wave % 4, g = lane / 16, r = lane % 16;
  // To each XCD a contiguous eighth of the whole tiles, then of the pieces, walked by its workgroups in turn; bands of eight column tiles.
  // The pieces of the same slabs lie beside each other.
  const int step = static_cast<int>(gridDim.x) / kXcds, xcd = static_cast<int>(blockIdx.x) % kXcds, pieces = p.left * p.cut;
  const auto eighth = [](int n, int i) { return static_cast<int>(static_cast<int64_t>(n) * i / kXcds); };
  const int whole0 = eighth(p.full, xcd), whole = eighth(p.full, xcd + 1) - whole0, piece0 = eighth(pieces, xcd);
  const int items = whole + eighth(pieces, xcd + 1) - piece0;
  int item = static_cast<int>(blockIdx.x) / kXcds;
  if (item >= items) return;
  const int slabs = (p.k + kK - 1) / kK;
  struct Item {
    int m0, n0, lo, hi, piece;  // the slabs lo .. hi - 1 of a tile (piece: -1, or all of them)
  };
  const auto place = [&](int it) {
    Item o{0, 0, 0, slabs, -1};
    int tile = whole0 + it;
    if (it >= whole) {
      o.piece = piece0 + it - whole;
      const int c = o.piece / p.left;
      tile = p.full + o.piece - c * p.left;
      o.lo = slabs * c / p.cut, o.hi = slabs * (c + 1) / p.cut;
    }
    const int band = kBand * p.row_tiles, b0 = tile / band, rest = tile % band, width = min(kBand, p.col_tiles - b0 * kBand);
    o.m0 = rest / width * kTileRows, o.n0 = (b0 * kBand + rest % width) * kTileCols;
    return o;
  };

  // Memory side: a wave sends the 1 KB pieces wave, wave + 8, .. of either operand.  k along the rows: 8 rows, lanes l a chunk of row l / 8;
  // rows of k: two of them, lanes l a chunk of row l / 32 (columns behind the last: the last ones again).
  const u32x4 buf_a = buffer_of(p.a, p.a_bytes);
  const u32x4 buf_b = buffer_of(MODE == kGate && wave & 4 ? p.b2 : p.b, p.b_bytes), buf_b2 = buffer_of(p.b2, p.b_bytes);  // (kGate: a wave's pieces are of one matrix)
  const uint32_t pitch_a = static_cast<uint32_t>(p.lda) * 2, pitch_b = static_cast<uint32_t>(p.ldb) * 2;
  const int krow = 2 * wave + lane / 32, kswizzle = (krow & 3) << 2 ^ (krow >> 3 & 1) << 1;
  const int row8 = 8 * wave + lane / 8, chunk8 = (lane & 7) ^ (row8 >> 1 & 7);
  uint32_t off_a[4], off_b[4];
  const auto offsets = [&](int m0, int n0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (kRowsA) off_a[i] = (krow + 16 * i) * pitch_a + min(m0 + ((lane & 31) ^ kswizzle) * 8, p.m - 8) * 2;
      else off_a[i] = static_cast<uint32_t>(m0 + row8 + 64 * i) * pitch_a + chunk8 * 16;
      // (two terms of up to 64 tokens: 64 rows of the first, 64 of the second, which lies behind it in their row of memory, and none)
      if constexpr (MODE == kInputTwo) off_a[i] = i < 2 ? row8 * pitch_a + i * (pitch_a / 2) + chunk8 * 16 : p.a_bytes;
      if constexpr (kRowsB) off_b[i] = (krow + 16 * i) * pitch_b + min(n0 + ((lane & 31) ^ kswizzle) * 8, p.n - 8) * 2;
      else off_b[i] = static_cast<uint32_t>(n0 + (row8 & 31) + 32 * i) * pitch_b + chunk8 * 16;
    }
  };
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)(smem))));
  const uint32_t lds_wave = lds0 + wave * 1024;
  // the ring: operand slabs A 0, B 0, A 1, B 1, .. in buffers 0 .. 4 in turn
  const auto behind = [&](uint32_t at, uint32_t buffers) { return at + buffers * kOperandBytes >= kRing ? at + buffers * kOperandBytes - kRing : at + buffers * kOperandBytes; };
  // (kGate: chunks behind the last k, where a row goes on with the next one or ends, are asked for behind the operands' ends)
  const int k_last = p.k - (slabs - 1) * kK;
  const auto along = [&](uint32_t offset, int slab, uint32_t end) { return MODE == kGate && slab == slabs - 1 && 8 * chunk8 >= k_last ? end : offset + slab * (kK * 2); };
  const auto request_a = [&](int slab, uint32_t to, int i) {
    load_to_lds16(buf_a, kRowsA ? off_a[i] + slab * kK * pitch_a : along(off_a[i], slab, p.a_bytes), lds_wave + to + i * 8192);
  };
  const auto request_b = [&](int slab, uint32_t to, int i) {
    if constexpr (MODE == kInput || MODE == kInputTwo) {
      const bool second = slab >= p.seg;
      const u32x4 buf = second ? buf_b2 : buf_b;
      load_to_lds16(buf, off_b[i] + (second ? slab - p.seg : slab) * kK * pitch_b, lds_wave + to + i * 8192);
    } else {
      load_to_lds16(buf_b, kRowsB ? off_b[i] + slab * kK * pitch_b : along(off_b[i], slab, p.b_bytes), lds_wave + to + i * 8192);
    }
  };

  // Fragment side: k-step `set` (0, 1) of a slab takes k = 32 set + 8 g + e.  k along the rows: row 16 i + r's chunk 4 set + g lies at
  // (g ^ swizzle) ^ 4 set.  Rows of k: source lane 4 a + b of sixteen points at row 32 set + 8 g + 4 half + a, columns 16 i + 4 b of the tile, and
  // lane t receives column t; the swizzle's and the block's bits (32 bytes and up) meet no others, so that block i is an exclusive or away.
  const int ta = r >> 2, tb = r & 3, tswizzle = ta << 2 ^ (g & 1) << 1;
  const uint32_t frag_a = kRowsA ? (8 * g + ta) * 512 + wm * 256 + tswizzle * 16 + (tb >> 1) * 16 + (tb & 1) * 8 : (wm * 128 + r) * 128 + (g ^ (r >> 1 & 7)) * 16;
  const uint32_t frag_b = kRowsB ? (8 * g + ta) * 512 + (wn >> 1) * 256 + ((wn & 1) * 128 ^ tswizzle * 16) + (tb >> 1) * 16 + (tb & 1) * 8
                                 : (wn * 64 + r) * 128 + (g ^ (r >> 1 & 7)) * 16;
  const auto read = [&](auto rows, uint32_t frag, uint32_t in, int set, int i) {
    if constexpr (decltype(rows)::value) {
      const uint32_t at = ((frag + lds0 + in) ^ (i * 32)) + set * 32 * 512;
      typedef __attribute__((address_space(3))) short4v* Ptr;
      const uint2 lo = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)(static_cast<uintptr_t>(at))));
      const uint2 hi = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)(static_cast<uintptr_t>(at + 4 * 512))));
      return u32x4{lo.x, lo.y, hi.x, hi.y};
    } else {
      return *reinterpret_cast<const __attribute__((address_space(3))) u32x4*>(static_cast<uintptr_t>((frag ^ (set * 64)) + lds0 + in + i * 16 * 128));
    }
  };
  // rows 16 i .. of A (i = 0 .. 7, four at a time), the four blocks of 16 columns of B (kGate: w1, w1, w3, w3)
  u32x4 fa0[4], fa1[4], fb0[4], fb1[4];
  const auto read_a = [&](u32x4* fa, uint32_t in, int set, int i) { fa[i % 4] = read(std::integral_constant<bool, kRowsA>(), frag_a, in, set, i); };
  const auto read_b = [&](u32x4* fb, uint32_t in, int set, int i) { fb[i] = read(std::integral_constant<bool, kRowsB>(), frag_b, in, set, i); };
  f32x4 acc[8][4];
  // product n (0 .. 15) of a half
  const auto mma = [&](const u32x4* fa, const u32x4* fb, int half, int n) { acc[4 * half + n / 4][n % 4] = mma16<DT>(fb[n % 4], fa[n / 4], acc[4 * half + n / 4][n % 4]); };

  Item at = place(item);
  offsets(at.m0, at.n0);
  // `ahead`: the slab that is asked for next, of an item `next` further on once it has reached `ahead_hi` (behind the last item the
  // same one again, which nobody reads)
  int ahead = at.lo, ahead_lo = at.lo, ahead_hi = at.hi, next = item + step;
  const auto turn = [&]() {
    if (ahead < ahead_hi) return;
    if (next < items) {
      const Item o = place(next);
      offsets(o.m0, o.n0);
      ahead_lo = o.lo, ahead_hi = o.hi;
    }
    ahead = ahead_lo;
    next += step;
  };
  uint32_t in_a = 0;  // the buffer of A's slab that is worked on; B's is the next, then come the next slab's
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    turn();
#pragma unroll
    for (int i = 0; i < 4; ++i) request_a(ahead, 2 * q * kOperandBytes, i);
#pragma unroll
    for (int i = 0; i < 4; ++i) request_b(ahead, (2 * q + 1) * kOperandBytes, i);
    ++ahead;
  }
  asm volatile("s_waitcnt vmcnt(8)\n\ts_barrier" ::: "memory");
#pragma unroll
  for (int i = 0; i < 4; ++i) read_a(fa0, 0, 0, i), read_b(fb0, kOperandBytes, 0, i);

  // A slab's two steps in two halves of 16 products; the fragments of the next half are read under the products of the current one.  The slab
  // behind the next: A's under the first two halves, into the buffer that the last slab's B has left; B's under the last one, into the
  // buffer of this slab's A, which all waves have read by then.
  constexpr int kReadsA = kRowsA ? 2 : 1, kReadsB = kRowsB ? 2 : 1;  // instructions
#define MEGA_SGB(mask, n) __builtin_amdgcn_sched_group_barrier(mask, n, 0)
  while (true) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int s = at.lo; s < at.hi; ++s) {
      const uint32_t in_b = behind(in_a, 1), next_a = behind(in_a, 2), next_b = behind(in_a, 3), last_b = behind(in_a, 4);
      turn();
      // first step, first half
#pragma unroll
      for (int i = 4; i < 8; ++i) read_a(fa1, in_a, 0, i);
#pragma unroll
      for (int n = 0; n < 8; ++n) mma(fa0, fb0, 0, n);
#pragma unroll
      for (int sg = 0; sg < 4; ++sg) {
        MEGA_SGB(0x008, 1);
        MEGA_SGB(0x100, kReadsA);
      }
      MEGA_SGB(0x008, 4);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 8; n < 16; ++n) {
        if (n % 4 == 0) request_a(ahead, last_b, n / 4 - 2);
        mma(fa0, fb0, 0, n);
        __builtin_amdgcn_sched_barrier(0);
      }
      // second half
#pragma unroll
      for (int i = 0; i < 4; ++i) read_a(fa0, in_a, 1, i), read_b(fb1, in_b, 1, i);
#pragma unroll
      for (int n = 0; n < 8; ++n) mma(fa1, fb0, 1, n);
#pragma unroll
      for (int sg = 0; sg < 4; ++sg) {
        MEGA_SGB(0x008, 1);
        MEGA_SGB(0x100, kReadsA);
        MEGA_SGB(0x008, 1);
        MEGA_SGB(0x100, kReadsB);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 8; n < 16; ++n) {
        if (n % 4 == 0) request_a(ahead, last_b, n / 4);
        mma(fa1, fb0, 1, n);
        __builtin_amdgcn_sched_barrier(0);
      }
      // second step, first half
#pragma unroll
      for (int i = 4; i < 8; ++i) read_a(fa1, in_a, 1, i);
#pragma unroll
      for (int n = 0; n < 16; ++n) mma(fa0, fb1, 0, n);
#pragma unroll
      for (int sg = 0; sg < 4; ++sg) {
        MEGA_SGB(0x008, 1);
        MEGA_SGB(0x100, kReadsA);
      }
      MEGA_SGB(0x008, 12);
      __builtin_amdgcn_sched_barrier(0);
      // the wave's pieces of the next slab have landed (A's of the one behind it may be on their way), its reads of this one have returned
      asm volatile("s_waitcnt vmcnt(4) lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
      for (int n = 0; n < 16; ++n) {
        if (n < 8) {
          if (n % 2 == 0) read_a(fa0, next_a, 0, n / 2);
          else read_b(fb0, next_b, 0, n / 2);
        }
        if (n % 4 == 3) request_b(ahead, in_a, n / 4);
        mma(fa1, fb1, 1, n);
        __builtin_amdgcn_sched_barrier(0);
      }
      ++ahead;
      in_a = next_a;
    }
    if constexpr (MODE == kInputTwo) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += acc[i + 4][j];
    }
    if (at.piece >= 0) {
      f32x4* const to = reinterpret_cast<f32x4*>(p.parts) + (static_cast<int64_t>(at.piece) * 8 + wave) * (8 * 4 * kWave) + lane;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (at.m0 + wm * 128 + i * 16 >= p.m) break;  // (never read)
#pragma unroll
        for (int j = 0; j < 4; ++j) to[(i * 4 + j) * kWave] = acc[i][j];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) finish<DT, MODE, KEEP>(p, acc[i], at.m0 + wm * 128 + i * 16, at.n0, wn, lane);
    }
    item += step;
    if (item >= items) break;
    at = place(item);
  }
#undef MEGA_SGB
  // (nothing may land in LDS that is another workgroup's by then)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// The pieces of a tile added up in their order: a wave has 16 rows x 64 accumulators of one of its waves.
template <int DT, int MODE, int KEEP>
__global__ __launch_bounds__(kWave) void gated_join_kernel(const GatedTiles p) {
  const int lane = threadIdx.x, j = static_cast<int>(blockIdx.x) / 64, wave = static_cast<int>(blockIdx.x) / 8 % 8, i = static_cast<int>(blockIdx.x) % 8;
  const int band = kBand * p.row_tiles, tile = p.full + j, b0 = tile / band, rest = tile % band, width = min(kBand, p.col_tiles - b0 * kBand);
  const int row0 = rest / width * kTileRows + wave / 4 * 128 + i * 16, n0 = (b0 * kBand + rest % width) * (MODE == kGate ? 128 : 256);
  if (row0 >= p.m) return;
  const f32x4* from = reinterpret_cast<const f32x4*>(p.parts) + ((static_cast<int64_t>(j) * 8 + wave) * 8 + i) * (4 * kWave) + lane;
  f32x4 acc[4];
#pragma unroll
  for (int f = 0; f < 4; ++f) acc[f] = from[f * kWave];
#pragma unroll 4
  for (int c = 1; c < p.cut; ++c) {
    from += static_cast<int64_t>(p.left) * (8 * 8 * 4 * kWave);
#pragma unroll
    for (int f = 0; f < 4; ++f) acc[f] += from[f * kWave];
  }
  finish<DT, MODE, KEEP>(p, acc, row0, n0, wave % 4, lane);
}

int workgroups(int* most) {
  int dev = 0, cus = 0;
  MEGA_CHECK_HIP(hipGetDevice(&dev));
  MEGA_CHECK_HIP(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev));
  *most = std::max(cus / kXcds, 1) * kXcds;  // one a CU, in whole rounds of the XCDs
  return MEGA_OK;
}
// Tiles in rounds of `most`; those of a last round that is not full are cut along k into pieces, one for each workgroup at most, their sums joined by a
// second launch, where that is shorter: a slab takes 1.45 us, a piece is written and read at 2.5 TB/s, the launch takes 8 us.  (Over 60 calls, 64 to 8192
// tokens of networks from 512 -> 1408 to 4096 -> 11008, these cuts are 1 % off the best of 24 ways to choose them in the mean, 4 % at most; dw of 32768 tokens,
// 4096 -> 11008, 1376 tiles: 4.2 ms, 4.6 uncut.)
void cut_last(GatedTiles& p, int most) {
  const int tiles = p.row_tiles * p.col_tiles, slabs = (p.k + kK - 1) / kK, left = tiles % most;
  p.full = tiles, p.left = 0, p.cut = 1;
  double best = slabs * 1.45;
  for (int cut = 2; cut <= slabs / 4 && left * cut <= most && left > 0; ++cut) {
    const double t = (slabs + cut - 1) / cut * 1.45 + left * cut * (kPieceBytes / 2.5e6) + 8;
    if (t < best) best = t, p.full = tiles - left, p.left = left, p.cut = cut;
  }
}

template <int DT, int MODE, int KEEP>
int launch(GatedTiles p, int most, hipStream_t s) {
  const int grid = std::min((p.full + p.left * p.cut + kXcds - 1) / kXcds * kXcds, most);
  MEGA_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&gated_tiles_kernel<DT, MODE, KEEP>), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kLds)));
  gated_tiles_kernel<DT, MODE, KEEP><<<dim3(static_cast<unsigned>(grid)), kThreads, kLds, s>>>(p);
  MEGA_CHECK_LAUNCH();
  if (p.left == 0) return MEGA_OK;
  gated_join_kernel<DT, MODE, KEEP><<<dim3(static_cast<unsigned>(p.left * 64)), kWave, 0, s>>>(p);
  MEGA_CHECK_LAUNCH();
  return MEGA_OK;
}
int64_t half_of(int64_t n_out) { return (n_out + kK - 1) / kK * kK; }
// the last byte of `rows` rows of `n` elements
uint32_t bytes_of(int64_t rows, int64_t pitch, int64_t n) { return static_cast<uint32_t>(2 * ((rows - 1) * pitch + n)); }
GatedTiles sizes_of(int mode, int64_t tokens, int64_t n_in, int64_t n_out, int matrices, int terms) {
  GatedTiles p{};
  const int64_t half = half_of(n_out);
  p.m = static_cast<int>(mode == kWeight ? matrices * half : tokens), p.k = static_cast<int>(mode == kGate ? n_in : mode == kInput ? 2 * half : terms * tokens);
  p.row_tiles = (p.m + kTileRows - 1) / kTileRows, p.col_tiles = static_cast<int>(mode == kGate ? (n_out + 127) / 128 : (n_in + 255) / 256);
  p.n_out = static_cast<int>(n_out), p.half = static_cast<int>(half), p.cols = static_cast<int>(n_in), p.seg = static_cast<int>(half / kK);
  return p;
}
template <int MODE, int KEEP>
int launch_of(int dtype, GatedTiles p, float* parts, hipStream_t s) {
  int most = 0;
  if (const int rc = workgroups(&most); rc != MEGA_OK) return rc;
  cut_last(p, most);
  p.parts = parts;
  if (p.left > 0 && parts == nullptr) return set_error(MEGA_ERR_INVALID_ARG, "gated_linear: null workspace");
  return dtype == MEGA_BF16 ? launch<MEGA_BF16, MODE, KEEP>(p, most, s) : launch<MEGA_F16, MODE, KEEP>(p, most, s);
}

}  // namespace

int64_t gated_tiles_bytes(int kind, int64_t tokens, int64_t n_in, int64_t n_out, int matrices, int terms) {
  int most = 0;
  if (workgroups(&most) != MEGA_OK) return 0;
  GatedTiles p = sizes_of(kind, tokens, n_in, n_out, matrices, terms);
  cut_last(p, most);
  return static_cast<int64_t>(p.left) * p.cut * kPieceBytes;
}

int gated_tiles(int dtype, const uint16_t* x, const uint16_t* w1, const uint16_t* w3, int64_t tokens, int64_t n_in, int64_t n_out,
                uint16_t* h, void* a, void* b, bool wide, float* parts, hipStream_t s) {
  GatedTiles p = sizes_of(kGate, tokens, n_in, n_out, 2, 1);
  p.a = x, p.b = w1, p.b2 = w3, p.a_bytes = bytes_of(tokens, n_in, n_in), p.b_bytes = bytes_of(n_out, n_in, n_in);
  p.n = static_cast<int>(n_out), p.lda = p.ldb = static_cast<int>(n_in);
  p.c = h, p.kept_a = a, p.kept_b = b, p.pitch = static_cast<int>(gated_pitch(n_out));
  if (a == nullptr) return launch_of<kGate, 0>(dtype, p, parts, s);
  return wide ? launch_of<kGate, 2>(dtype, p, parts, s) : launch_of<kGate, 1>(dtype, p, parts, s);
}

int gated_tiles_input(int dtype, const uint16_t* g, const uint16_t* w1, const uint16_t* w3, int64_t tokens, int64_t n_in, int64_t n_out, int64_t ld,
                      int terms, uint16_t* dx, float* parts, hipStream_t s) {
  const int64_t all = terms * 2 * half_of(n_out);
  GatedTiles p = sizes_of(kInput, tokens, n_in, n_out, 2, terms);
  p.a = g, p.b = w1, p.b2 = w3, p.a_bytes = bytes_of(tokens, all, all), p.b_bytes = bytes_of(n_out, ld, ld);
  p.n = static_cast<int>(ld), p.lda = static_cast<int>(all), p.ldb = static_cast<int>(ld), p.c = dx;
  return terms == 2 ? launch_of<kInputTwo, 0>(dtype, p, parts, s) : launch_of<kInput, 0>(dtype, p, parts, s);
}

int gated_tiles_weight(int dtype, const uint16_t* g, const uint16_t* x, int64_t tokens, int64_t n_in, int64_t n_out, int64_t ld,
                       int terms, uint16_t* dw1, uint16_t* dw3, float* sums, bool first, bool last, float* parts, hipStream_t s) {
  const int64_t both = 2 * half_of(n_out);
  GatedTiles p = sizes_of(kWeight, tokens, n_in, n_out, dw1 != nullptr && dw3 != nullptr ? 2 : 1, terms);
  const int64_t from = dw1 != nullptr ? 0 : both / 2;
  p.a = g + from, p.b = p.b2 = x, p.a_bytes = bytes_of(terms * tokens, both, both - from), p.b_bytes = bytes_of(terms * tokens, ld, ld);
  p.n = static_cast<int>(ld), p.lda = static_cast<int>(both), p.ldb = static_cast<int>(ld), p.c = dw1 != nullptr ? dw1 : dw3, p.c2 = dw3;
  p.sum = sums, p.first = first, p.last = last;
  return launch_of<kWeight, 0>(dtype, p, parts, s);
}

}  // namespace mega
