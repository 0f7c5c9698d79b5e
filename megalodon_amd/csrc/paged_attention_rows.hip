// Paged attention for many rows of a sequence at a time (more than 32 on average): prompts and their pieces.
//
// The mathematics and the lane layout are those of paged_attention.hip; what differs is what bounds it.  A value that has been read serves 64
// rows; a wave has 64 rows x 128 columns of accumulators, half of its registers, and two waves share a SIMD: one's products beside the
// other's scores and exponentials.
//   - More than 128 value columns: up to eight waves with their columns and 32 keys of a tile each, as there.  A tile's keys are asked for a
//     tile ahead, into LDS and in operand order, the next step's values while the last two columns of this one's are multiplied.
//     Bound by what a CU is given of L2, 41 bytes a cycle while values are read: those of 256 keys take 17000 cycles, their products 8200,
//     the tile's scores and softmax 4000 more.  The waves meet once a tile (twice, at the maxima and at the probabilities: 489 us).  A prompt
//     of 8192 tokens in chunks of 4096, four heads of 256 / 2048: 463 us, 668 TFLOP/s.  One wave to a SIMD with 64 x 256 spilled 1.5 KB a lane;
//     four-wave workgroups of 64 x 512, whose scores are made twice, took a fifth longer, two-wave ones twice as long; blocks in other orders over
//     the XCDs 5 and 40 % longer; the first values of a tile on their way during its scores do not fit the registers.
//   - Up to 128: a workgroup is one wave, eight to a CU, and probabilities never leave the registers.  Bound by the issue of vector
//     instructions (conversions, exponentials, maxima: 1750 cycles for 32 keys) beside 1000 of products: 255 to 1023 tokens behind up to
//     7001 in 8 bits, 260 us, 663 TFLOP/s.  32 rows a wave: 589 us; its keys ahead in registers: 469 us (spills).
// A piece leaves 64 rows in float32: 512 tokens behind 1531 write and read 67 MB beside a cache of 38, 57 us.
#include "paged_attention.hpp"

namespace mega {
namespace {

constexpr int RT = 4, CT = 8;                        // row and column tiles of a wave
constexpr int kRows = 16 * RT;
// of a key's 16-byte parts to a lane, those that come through LDS: all, or as many as it has room for beside the rows and the probabilities
constexpr int in_lds(bool solo, int parts) { return solo ? 0 : parts < 3 ? parts : 3; }

// A wave's accumulators to out, or to the workspace: there sixteen rows at a time through the wave's own LDS (free behind the last keys), as an
// instruction would write 16 bytes of 64 lines from the registers -- 512 tokens behind 1531: 25 us more.  Out has half the bytes,
// and one write of them for many keys: a prompt takes the same time either way.
constexpr int kTurned = 16 * CT + 4;  // floats of a row there: sixteen rows' equal columns are in different banks
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
template <int DT>
__device__ __forceinline__ void store_piece(const AttnArgs& a, const Block& k, const Destination& to, int head, bool notes, int first_column, float* turned,
                                            const f32x4 (&acc)[RT][CT], const float (&m)[RT], const float (&l)[RT]) {
  const int lane = opaque(static_cast<int>(threadIdx.x) & 63), n = lane & 15, h = lane >> 4;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int64_t at = place_of_row(a, k, to, head, rt * 16 + n, notes && h == 0, m[rt], l[rt]);
    if (to.alone) {
      if (rt * 16 + n >= k.count) continue;
      const float inverse = l[rt] == 0.f ? 0.f : 1.f / l[rt];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = first_column + CT * (4 * h + i);
        if (c >= a.v.width) continue;
        float o[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = l[rt] == 0.f ? 0.f : acc[rt][j][i] * inverse;
        *reinterpret_cast<uint4*>(a.out + at * a.v.width + c) =
            make_uint4(pack2<DT>(o[0], o[1]), pack2<DT>(o[2], o[3]), pack2<DT>(o[4], o[5]), pack2<DT>(o[6], o[7]));
      }
    } else {
      wave_lds_fence();
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < CT; j += 4)
          *reinterpret_cast<float4*>(turned + n * kTurned + CT * (4 * h + i) + j) = make_float4(acc[rt][j][i], acc[rt][j + 1][i], acc[rt][j + 2][i], acc[rt][j + 3][i]);
      wave_lds_fence();
      const int c = (lane & 31) * 4, row = rt * 16 + (lane >> 5);
      float* const part = a.part + (to.slot + row) * a.v.width + first_column + c;
      if (first_column + c < a.v.width)
#pragma unroll
        for (int pair = 0; pair < 16; pair += 2)
          if (row + pair < k.count)
            *reinterpret_cast<float4*>(part + static_cast<int64_t>(pair) * a.v.width) = *reinterpret_cast<const float4*>(turned + (pair + (lane >> 5)) * kTurned + c);
    }
  }
}

// KS: 32-wide steps of a key row; kFull: it has 32 KS elements; kSolo: a workgroup is one wave
template <int DT, bool kEight, int KS, bool kFull, bool kSolo>
__global__ __launch_bounds__(kSolo ? kWave : kMaxWaves * kWave, 2) void paged_rows_kernel(AttnArgs a) {
  constexpr int kBytes = kEight ? 1 : 2, kParts = kEight ? KS / 2 : KS, kInLds = in_lds(kSolo, kParts);
  // parts that come through registers, and how many of them are there at a time
  constexpr int kRest = kParts - kInLds, kMost = kSolo && !kEight ? 4 : 2, kHeld = kRest < kMost ? kRest : kMost;
  extern __shared__ __align__(16) uint4 lds[];
  __shared__ Progress progress;
  const int wave = kSolo ? 0 : __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6), waves = kSolo ? 1 : static_cast<int>(blockDim.x) >> 6;
  uint4* const lds_q = lds;                  // [RT][KS][64]
  uint4* const lds_k = lds + RT * KS * 64;                             // [waves][2][kInLds][64]
  uint4* const lds_p = lds_k + waves * 2 * kInLds * 64;                // [2][waves][RT][64]: a tile's and the next one's
  float* const lds_m = reinterpret_cast<float*>(lds_p + (kSolo ? 0 : 2 * waves * RT * 64));  // [kRows][kMaxWaves]
  int* const lds_says = reinterpret_cast<int*>(lds_m + kRows * kMaxWaves);              // [2][kMaxWaves]: the waves' keys have pages (1), and no score above the slack (2)
  int2* const lds_sees = reinterpret_cast<int2*>(lds_says + 2 * kMaxWaves);                // [kRows]

  // (as in paged_attention.hip)
  uint32_t id = group_number();
  const int slab = id % a.slabs;
  id /= a.slabs;
  const int head = id % a.heads;
  id /= a.heads;
  const int page_mask = (1 << a.view.page_shift) - 1;
  const int first_column = (slab * waves + wave) * CT * 16;
  Block k;
  Progress at;
  if (!first_piece<kRows>(a, static_cast<int>(id), at, k)) return;

  for (;;) {
    const int lane = opaque(static_cast<int>(threadIdx.x) & 63);
    int begin, end;
    take_piece<kRows>(a, at, progress, k, begin, end);
    for (int c = threadIdx.x; c < kRows * KS * 4; c += blockDim.x) row_piece_to_lds<kEight, KS>(row_piece<KS>(a, k, head, c), c, lds_q);
    ranges_to_lds<kRows>(a, k, end, lds_sees);
    if constexpr (!kSolo) {
      for (int c = threadIdx.x; c < kRows * kMaxWaves; c += blockDim.x) lds_m[c] = -__builtin_inff();  // (of waves that there are not, too)
      if (threadIdx.x < 2 * kMaxWaves) lds_says[threadIdx.x] = 3;
    }
    // keys all_low .. all_high are seen by every row of the block
    const int all_low = chunk_start(a, k.position0 + token_of(a, k.row0 + k.count - 1)), all_high = min(k.position0 + token_of(a, k.row0), end - 1);

    // ---- keys: part `part` of a lane is 16 bytes of key 16 half + (lane & 15).  Those that come through LDS are asked for a tile ahead, into the
    // wave's own place and in operand order
    u32x4 kx[2][kHeld > 0 ? kHeld : 1];
    float unit[2];  // of the lane's keys (8 bits)
    struct Keys {
      const uint8_t* from[2];
      const uint8_t* exponents[2];
      bool there[2];
    };
    const auto keys_at = [&](int first) {
      Keys t;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int held = min(first + 16 * half, (end - 1) & ~15), place = held & page_mask;
        const Page page = page_of(a, k.sequence, held);
        t.there[half] = page.there;
        t.from[half] = static_cast<const uint8_t*>(a.k.rows) + (page.number * a.k.page + static_cast<int64_t>(head) * a.k.head + static_cast<int64_t>(place) * a.k.slot) * kBytes;
        if constexpr (kEight) t.exponents[half] = a.k.exponents + (page.number * a.k.ePage + static_cast<int64_t>(head) * a.k.eHead + static_cast<int64_t>(place) * a.k.eSlot);
      }
      return t;
    };
    const auto key_offset = [&](int part) {
      const int l = opaque(lane), d = kFull ? (kEight ? 64 : 32) * part + (kEight ? 16 : 8) * (l >> 4)
                                           : min((kEight ? 64 : 32) * part + (kEight ? 16 : 8) * (l >> 4), a.k.width - (kEight ? 16 : 8));
      return (static_cast<uint32_t>(l & 15) * a.k.slot + d) * kBytes;
    };
    const auto load_key = [&](const Keys& t, int half, int part) {
      kx[half][(part - kInLds) % (kHeld > 0 ? kHeld : 1)] = *reinterpret_cast<const u32x4*>(t.from[half] + key_offset(part));
    };
    const auto load_key_exponents = [&](const Keys& t) {
      if constexpr (kEight) {
#pragma unroll
        for (int half = 0; half < 2; ++half) unit[half] = exponent_value(t.exponents[half][static_cast<uint32_t>(opaque(lane) & 15) * a.k.eSlot]);
      }
    };
    const auto ask_for_keys = [&](int tile) {
      if constexpr (kInLds > 0) {
        const Keys t = keys_at(min(tile + 32 * wave, (end - 1) & ~31));
        const uint32_t to = lds_address(lds_k + wave * 2 * kInLds * 64);
#pragma unroll
        for (int part = 0; part < kInLds; ++part) {
          const uint32_t offset = key_offset(part);
#pragma unroll
          for (int half = 0; half < 2; ++half) load_to_lds16(t.from[half], offset, to + (half * kInLds + part) * 1024);
        }
      }
    };

    // ---- values: eight columns of eight of a step's 32 keys to a lane and column group
    typedef uint32_t Piece __attribute__((ext_vector_type(kEight ? 2 : 4)));
    Piece x[8];
    uint32_t e[8];
    bool there[2] = {false, false};
    struct Step {
      const uint8_t* from[2];
      const uint8_t* exponents[2];
      bool there[2];
    };
    const auto step_at = [&](int first) {
      Step t;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int held = min(first + 16 * half, (end - 1) & ~15), place = held & page_mask;
        const Page page = page_of(a, k.sequence, held);
        t.there[half] = page.there;
        t.from[half] = static_cast<const uint8_t*>(a.v.rows) + (page.number * a.v.page + static_cast<int64_t>(head) * a.v.head + static_cast<int64_t>(place) * a.v.slot) * kBytes;
        if constexpr (kEight) t.exponents[half] = a.v.exponents + (page.number * a.v.ePage + static_cast<int64_t>(head) * a.v.eHead + static_cast<int64_t>(place) * a.v.eSlot);
      }
      return t;
    };
    const auto load_values = [&](const Step& t) {
      // (columns behind the last are computed from others and not written)
      const int l = opaque(lane);
      const uint32_t offset = (static_cast<uint32_t>(4 * (l >> 4)) * a.v.slot + min(first_column + (l & 15) * 8, a.v.width - 8)) * kBytes;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = *reinterpret_cast<const Piece*>(t.from[i >> 2] + (offset + static_cast<uint32_t>((i & 3) * a.v.slot * kBytes)));
    };
    const auto load_exponents = [&](const Step& t) {
      if constexpr (kEight) {
        const uint32_t offset = static_cast<uint32_t>(4 * (opaque(lane) >> 4)) * a.v.eSlot;
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = t.exponents[i >> 2][offset + static_cast<uint32_t>((i & 3) * a.v.eSlot)];
      }
    };
    const auto load_step = [&](int first) {
      const Step t = step_at(first);
      load_exponents(t);
      load_values(t);
      there[0] = t.there[0], there[1] = t.there[1];
    };

    f32x4 acc[RT][CT];
    float m[RT], l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      m[rt] = -__builtin_inff(), l[rt] = 0.f;
#pragma unroll
      for (int c = 0; c < CT; ++c) acc[rt][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (begin < end) ask_for_keys(begin);
    __syncthreads();

    int side = 0;  // of the probabilities: a wave that is done with its values goes on while others read theirs, so that the waves meet once a tile
    for (int tile = begin; tile < end; tile += 32 * waves, side ^= 1) {
      // ---- scores of the wave's keys (a wave behind the end computes others' again: nothing is seen of them)
      const int mine = tile + 32 * wave;
      f32x4 s[2][RT];
      const Keys keys = keys_at(min(mine, (end - 1) & ~31));
      bool pages_there = keys.there[0] && keys.there[1];
      const bool whole = pages_there && mine >= all_low && mine + 31 <= all_high;
      if constexpr (kInLds > 0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the keys are in LDS)
#pragma unroll
      for (int part = kInLds; part < kInLds + kHeld; ++part)
#pragma unroll
        for (int half = 0; half < 2; ++half) load_key(keys, half, part);
      load_key_exponents(keys);
      {
        const auto fetch = [&](int c, u32x4 (&q)[RT]) {
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) q[rt] = __builtin_bit_cast(u32x4, lds_q[(rt * KS + c) * 64 + lane]);
        };
        u32x4 q[2][RT];
        fetch(0, q[0]);
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) s[half][rt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < KS; ++c) {  // (the rows' operands one step ahead; the fence keeps it at that)
          const int part = kEight ? c >> 1 : c;
          if (c + 1 < KS) fetch(c + 1, q[(c + 1) & 1]);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            u32x4 x = part < kInLds ? __builtin_bit_cast(u32x4, lds_k[((wave * 2 + half) * kInLds + part) * 64 + lane]) : kx[half][(part - kInLds) % (kHeld > 0 ? kHeld : 1)];
            if constexpr (kEight) {
              const uint32_t lo = (c & 1) ? x[2] : x[0], hi = (c & 1) ? x[3] : x[1];
              x = u32x4{widen<DT, false>(lo, unit[half]), widen<DT, true>(lo, unit[half]), widen<DT, false>(hi, unit[half]), widen<DT, true>(hi, unit[half])};
            }
            if constexpr (!kFull) {  // (behind the row's end the rows' operands are zero, and infinity times zero is not)
              const int d = kEight ? (c >> 1) * 64 + (opaque(lane) >> 4) * 16 : c * 32 + (opaque(lane) >> 4) * 8;
              if (d >= a.k.width) x = u32x4{0, 0, 0, 0};
            }
            if (part >= kInLds && part + kHeld < kParts && (!kEight || (c & 1))) load_key(keys, half, part + kHeld);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) s[half][rt] = mma<DT>(x, q[c & 1][rt], s[half][rt]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      load_step(tile);
      if (!whole) {
        const int l = opaque(lane), n = l & 15, first = mine + 4 * (l >> 4);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const int2 range = lds_sees[rt * 16 + n];
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (!keys.there[half] || !in_range(range, first + 16 * half + i)) s[half][rt][i] = -__builtin_inff();
        }
      }

      // ---- probabilities and sums.  A tile whose scores are all within the rows' slack above m, as nearly all are behind the first, needs no maxima
      float top[RT];  // of the lane's scores
      bool over = false;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        float t = s[0][rt][0];
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int i = 0; i < 4; ++i) t = fmaxf(t, s[half][rt][i]);
        top[rt] = t * a.scale;
        over = over || top[rt] > m[rt] + kSlack;
      }
      u32x4 own[RT];  // (kSolo: the operands themselves)
      float sum[RT];
      const auto weigh = [&] {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const float base = (m[rt] == -__builtin_inff() ? 0.f : m[rt]) - kLift<DT>;
          float p[8];
          sum[rt] = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            p[i] = __builtin_amdgcn_exp2f(fmaf(s[i >> 2][rt][i & 3], a.scale, -base));
            sum[rt] += p[i];
          }
          own[rt] = u32x4{pack2<DT>(p[0], p[1]), pack2<DT>(p[2], p[3]), pack2<DT>(p[4], p[5]), pack2<DT>(p[6], p[7])};
          if constexpr (!kSolo) lds_p[((side * waves + wave) * RT + rt) * 64 + lane] = __builtin_bit_cast(uint4, own[rt]);
        }
      };
      // (top: of the whole rows)
      const auto follow = [&] {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const float now = top[rt] > m[rt] + kSlack ? top[rt] : m[rt], alpha = __builtin_amdgcn_exp2f(m[rt] - (now == -__builtin_inff() ? 0.f : now));
          m[rt] = now;
          // (a score that only the scale makes infinite is finite in the fused product below, which would give it no weight instead of NaN)
          l[rt] = now == __builtin_inff() ? __builtin_nanf("") : l[rt] * alpha;
#pragma unroll
          for (int c = 0; c < CT; ++c) acc[rt][c] *= alpha;
        }
      };
      if constexpr (kSolo) {
        if (__any(over)) {
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) top[rt] = four_max(top[rt]);
          follow();
        }
        weigh();
      } else {
        over = __any(over);
        if (!over) weigh();
        if (opaque(lane) == 0) lds_says[side * kMaxWaves + wave] = (pages_there ? 1 : 0) | (over ? 0 : 2);
        __syncthreads();
        int says = 3;
#pragma unroll
        for (int w = 0; w < kMaxWaves; w += 4) {
          const int4 u = *reinterpret_cast<const int4*>(lds_says + side * kMaxWaves + w);
          says &= u.x & u.y & u.z & u.w;
        }
        says = __builtin_amdgcn_readfirstlane(says);
        pages_there = (says & 1) != 0;
        if ((says & 2) == 0) {
          const int l = opaque(lane), n = l & 15;
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            top[rt] = four_max(top[rt]);
            if (l < 16) lds_m[(rt * 16 + n) * kMaxWaves + wave] = top[rt];
          }
          __syncthreads();
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int w = 0; w < kMaxWaves; w += 4) {
              const float4 v = *reinterpret_cast<const float4*>(lds_m + (rt * 16 + n) * kMaxWaves + w);
              top[rt] = fmaxf(top[rt], fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)));
            }
          follow();
          weigh();
          __syncthreads();
        }
      }
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) l[rt] += sum[rt];

      // ---- values: 32 keys a step
      // (kSolo: in front of the other wave, whose scores and exponentials fill the gaps; the older of two equals has them all, and the younger ends
      // alone -- four pieces of prompts on shared heads: 289 us without, 272 with)
      if constexpr (kSolo) __builtin_amdgcn_s_setprio(1);
      const int steps = kSolo ? 1 : min(waves, (end - tile + 31) >> 5);
#pragma unroll 1
      for (int step = 0; step < steps; ++step) {
        u32x4 p[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) p[rt] = kSolo ? own[rt] : __builtin_bit_cast(u32x4, lds_p[((side * waves + step) * RT + rt) * 64 + lane]);
        const int first = tile + 32 * step;
        const Step next = step_at(min(first + 32, (end - 1) & ~31));
        float unit[8];
        if constexpr (kEight)
#pragma unroll
          for (int i = 0; i < 8; ++i) unit[i] = exponent_value(e[i]);
        bool odd = false;
        if (first < all_low || first + 31 > all_high || !pages_there) {
          // what is not there, or not this workgroup's, must not meet a probability of zero as an infinity or NaN; nor must such a
          // value of a key that only some rows see, which goes to those alone below
          const int h = opaque(lane) >> 4;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int key = first + 16 * (i >> 2) + 4 * h + (i & 3);
            const uint32_t keep = key >= k.begin && key < end && there[i >> 2] ? ~0u : 0u;
#pragma unroll
            for (int j = 0; j < (kEight ? 2 : 4); ++j) {
              uint32_t finite;
              if constexpr (kEight)
                finite = finite_codes<DT>(x[i][j], unit[i]);
              else
                finite = finite_halves<DT>(x[i][j]);
              odd = odd || (~finite & keep) != 0;
              x[i][j] &= keep & finite;
            }
            // (nor their exponents, which nobody need have written: a byte of 255 makes NaN of a zero)
            if constexpr (kEight) unit[i] = keep != 0 && unit[i] < __builtin_inff() ? unit[i] : 1.f;
          }
        }
        if constexpr (kEight && !kSolo) load_exponents(next);
        // columns 2 j, 2 j + 1 of a lane's eight as operands
        const auto convert = [&](int j, u32x4 (&vt)[2]) {
          uint32_t w[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if constexpr (kEight)
              w[i] = (j & 1) ? widen<DT, true>(x[i][j >> 1], unit[i]) : widen<DT, false>(x[i][j >> 1], unit[i]);
            else
              w[i] = x[i][j];
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            vt[0][i] = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], 0x05040100);
            vt[1][i] = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], 0x07060302);
          }
        };
        u32x4 vt[2][2];
        convert(0, vt[0]);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (u + 1 < 4) convert(u + 1, vt[(u + 1) & 1]);
          // (the last columns have just been converted; the next 32 keys' values, of these once more behind the last)
          if constexpr (!kSolo)
            if (u == 2) {
              // (the next tile's keys in front of them: requests come back in their order, and nobody waits for these alone)
              if (step == 0 && tile + 32 * waves < end) ask_for_keys(tile + 32 * waves);
              load_values(next);
            }
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) acc[rt][2 * u + j] = mma<DT>(vt[u & 1][j], p[rt], acc[rt][2 * u + j]);
        }
        if (__builtin_expect(__any(odd), 0))  // (out of the loop's way: 256 us for four pieces of prompts on shared heads, 257.5 in it)
          add_odd_values<DT, kEight, 8>(a, k, end, first, first_column, step_at(first), lds_sees, [&](int rt, int slot) -> uint32_t {
            // (the lane of this row and slot has the probability, in its place of eight)
            const int place = slot & 7;
            uint32_t word = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) word = (place >> 1) == i ? p[rt][i] : word;
            word = static_cast<uint32_t>(__shfl(static_cast<int>(word), (slot & ~7) * 2 + (opaque(lane) & 15), 64));
            return (place & 1) ? word >> 16 : word;
          }, acc);
        there[0] = next.there[0], there[1] = next.there[1];
      }
      if constexpr (kSolo) __builtin_amdgcn_s_setprio(0);
    }

    // ---- the rows' sums over the lanes and waves that had their keys
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) l[rt] = four_sum(l[rt]);
    if constexpr (!kSolo) {
      const int at = opaque(lane), n = at & 15;
      __syncthreads();  // (the maxima of the last tile have been read)
      if (at < 16)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) lds_m[(rt * 16 + n) * kMaxWaves + wave] = l[rt];
      __syncthreads();
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) l[rt] = sum_of_waves(lds_m + (rt * 16 + n) * kMaxWaves, waves);
    }
    const Destination to = destination_of(a, progress, static_cast<int>(id), head);
    if (to.fits) store_piece<DT>(a, k, to, head, slab == 0 && wave == 0, first_column, reinterpret_cast<float*>(lds) + wave * 16 * kTurned, acc, m, l);
    if (to.last) break;
    at = next_piece<kRows>(a, progress, k);
    __syncthreads();  // (the rows, maxima, probabilities and progress of this piece have been read)
  }
}

template <int DT, bool kEight, int KS, bool kFull, bool kSolo>
int launch(const AttnArgs& a, const RowsPlan& p, void* stream) {
  const auto kernel = paged_rows_kernel<DT, kEight, KS, kFull, kSolo>;
  const int parts = kEight ? KS / 2 : KS, kept = p.waves * 2 * in_lds(kSolo, parts) * 64;
  const size_t bytes = (RT * KS * 64 + kept + (kSolo ? 0 : 2 * p.waves * RT * 64)) * sizeof(uint4) + (kRows * sizeof(float) + 2 * sizeof(int)) * kMaxWaves + kRows * sizeof(int2);
  if (bytes > 65536)
    MEGA_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)));
  kernel<<<grid_of(p.workgroups), dim3(p.waves * kWave), bytes, static_cast<hipStream_t>(stream)>>>(a);
  MEGA_CHECK_LAUNCH();
  return MEGA_OK;
}

template <int DT, bool kEight, int KS, bool kFull>
int launch_columns(const AttnArgs& a, const RowsPlan& p, void* stream) {
  return p.waves == 1 ? launch<DT, kEight, KS, kFull, true>(a, p, stream) : launch<DT, kEight, KS, kFull, false>(a, p, stream);
}

template <int DT, bool kEight>
int launch_width(const AttnArgs& a, const RowsPlan& p, void* stream) {
  if (a.k.width == 128) return launch_columns<DT, kEight, 4, true>(a, p, stream);
  if (a.k.width == 256) return launch_columns<DT, kEight, 8, true>(a, p, stream);
  return p.ks == 4 ? launch_columns<DT, kEight, 4, false>(a, p, stream) : launch_columns<DT, kEight, 8, false>(a, p, stream);
}

}  // namespace

int launch_paged_rows(const AttnArgs& a, const RowsPlan& p, int dtype, bool eight, void* stream) {
  if (dtype == MEGA_BF16) return eight ? launch_width<MEGA_BF16, true>(a, p, stream) : launch_width<MEGA_BF16, false>(a, p, stream);
  return eight ? launch_width<MEGA_F16, true>(a, p, stream) : launch_width<MEGA_F16, false>(a, p, stream);
}

}  // namespace mega
