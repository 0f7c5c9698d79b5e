// Attention of new tokens over the paged key / value cache.
//
// For row r (a new token's query of one head) with visible keys lo .. hi
//   s_j = scale q . k_j,  m = max_j s_j,  l = sum_j e^(s_j - m),  o = sum_j e^(s_j - m) v_j / l,
// in one pass over the keys with the running m and l; accumulators follow a rising m by the factor
// e^(m_old - m_new).  Scores, m, l and o are float32; the probabilities that go into the second product are
// rounded to the operands' type, which is what the matrix cores take (each is off by 2^-8 or 2^-11 of itself at most,
// as the result is by its own rounding); l sums them unrounded.
//
// Layout.  A workgroup has kRows = 16 RT rows (new tokens of one sequence, and the query heads that share a key /
// value head, side by side) of one cache head, and W waves; wave w has 16 CT of its value columns.  A tile is
// 32 W keys:
//   scores   wave w takes 32 of them, all rows: S^T = K Q^T with K by whole rows through the wave's own LDS (rows too wide for that: in
//            operand order into registers, as keys are the instruction's k-contiguous operand) and Q from LDS in operand order;
//   softmax  a row's keys lie in four lanes of a wave and in W waves: maxima meet in LDS, P^T goes there;
//   values   every wave takes all 32 W keys for its own columns: O^T = V^T P^T.  No value is read twice in a
//            workgroup, so values pass through registers only: a lane reads eight columns of eight keys, and a byte
//            permutation pairs neighbouring keys -- column 8 n + j of lane n's eight becomes row n of operand j.
// Both products have the rows along the lanes, so a row's m, l and rescaling factor live in its lanes, and P^T
// leaves the first product in the very registers that the second one takes: which of the 32 keys sits in which k slot is
// free as long as V agrees, and slot (8 h + i) is key 4 h + i of the first 16 for i < 4, of the second 16 above.
//
// A page holds 16 keys at least, and key groups are aligned, so a lane group's keys share a page: its base is a scalar, its number a
// load of the scalar unit (a vector load would be waited for in turn with the keys and values in flight).
//
// Few row blocks (single tokens, drafts, a prompt's piece).  The blocks' keys, in units of 32, form one line, block after block, which is
// cut into as many equal parts as workgroups fill the chip, whatever the sequences' lengths: a workgroup goes through the
// pieces of blocks that its part holds, leaves each one's (o, m, l) in a workspace in float32, and a second kernel joins them.
// Many row blocks: a workgroup each.
//
// This file: up to 32 rows of a sequence on average.  Bound by the cache's bytes: 32 tokens on shared heads over 16-bit caches of up to 16000
// positions, 205 us, 5.3 TB/s (a large read reaches 6.0); sixteen tokens over 8-bit ones of up to 4000, 79 us, 4.7 TB/s; drafts of eight
// sequences, 76 us, 4.2 TB/s.  Short of that by what comes before the first and behind the last key of a workgroup, some 8 us: chains of
// dependent loads (bounds, lengths, page numbers, keys; 4 us), the results' way out, the join (4 us); one token over 1531 positions
// takes 21 us, of them 5 on the cache.  A third wave on a SIMD for narrow heads: 229 us against 205, the registers of the values in flight.
#include "paged_attention.hpp"

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>

namespace mega {
namespace {

// A lane's values of 32 keys in one group of 16 kCols columns, as they lie in the pool: kCols columns of eight keys.
template <bool kEight, int kCols>
struct Values {
  static constexpr int kWords = kCols * (kEight ? 1 : 2) / 4;
  typedef uint32_t Piece __attribute__((ext_vector_type(kWords)));
  Piece x[8];
};

// Whether a tile's keys go through LDS (eight waves' 32 rows each, beside the rows and the probabilities): requests then cover whole rows.  Otherwise
// they go to registers in operand order, where a request touches 64 bytes of sixteen rows -- one token over 1531 positions: the keys
// of a run are there 2 us later.
constexpr bool staged(bool eight, int rt, int ks) { return 8 * 32 * ks * (eight ? 32 : 64) + rt * (ks + 8) * 1024 <= 156 * 1024; }

// A wave's accumulators to out or to the workspace.  Accumulator element i of column operand j is column kCols (4 h + i) + j of its group of
// 16 kCols; eight columns are stored at a time.
template <int DT, int RT, int CT, int kCols>
__device__ __forceinline__ void store_piece(const AttnArgs& a, const Block& k, const Destination& to, int head, bool notes, int first_column,
                                            const f32x4 (&acc)[RT][CT], const float (&m)[RT], const float (&l)[RT]) {
  const int lane = opaque(static_cast<int>(threadIdx.x) & 63), n = lane & 15, h = lane >> 4;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int row = rt * 16 + n;
    if (row >= k.count) continue;
    const int64_t at = place_of_row(a, k, to, head, row, notes && h == 0, m[rt], l[rt]);
    const float inverse = l[rt] == 0.f ? 0.f : 1.f / l[rt];
#pragma unroll
    for (int cg = 0; cg < CT / kCols; ++cg)
#pragma unroll
      for (int i = 0; i < 4; i += 8 / kCols) {
        const int c = first_column + 16 * kCols * cg + kCols * (4 * h + i);
        if (c >= a.v.width) continue;
        float o[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = acc[rt][kCols * cg + j % kCols][i + j / kCols];
        if (!to.alone) {
          float4* part = reinterpret_cast<float4*>(a.part + (to.slot + row) * a.v.width + c);
          part[0] = make_float4(o[0], o[1], o[2], o[3]);
          part[1] = make_float4(o[4], o[5], o[6], o[7]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) o[j] = l[rt] == 0.f ? 0.f : o[j] * inverse;
          *reinterpret_cast<uint4*>(a.out + at * a.v.width + c) =
              make_uint4(pack2<DT>(o[0], o[1]), pack2<DT>(o[2], o[3]), pack2<DT>(o[4], o[5]), pack2<DT>(o[6], o[7]));
        }
      }
  }
}

template <int DT, bool kEight, int RT, int CT, int KS>  // KS: 32-wide steps of a key row
__global__ __launch_bounds__(kMaxWaves * kWave, 2) void paged_attn_kernel(AttnArgs a) {
  // 16-byte loads of values where the registers allow it: eight of a lane's columns at a time, else four
  constexpr int kRows = 16 * RT, kCols = RT > 1 && !kEight ? 4 : 8, kGroups = CT / kCols;
  extern __shared__ __align__(16) uint4 lds[];
  __shared__ Progress progress;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6), waves = static_cast<int>(blockDim.x) >> 6;
  uint4* const lds_q = lds;                       // [RT][KS][64]
  constexpr bool kStaged = staged(kEight, RT, KS);
  constexpr int kPieces = KS * (kEight ? 2 : 4);  // 16-byte pieces of a key row
  uint4* const lds_k = lds + RT * KS * 64;        // kStaged: [waves][32][kPieces]
  uint4* const lds_p = lds_k + (kStaged ? waves * 32 * kPieces : 0);  // [waves][RT][64]
  float* const lds_m = reinterpret_cast<float*>(lds_p + waves * RT * 64);  // [kRows][8]
  int* const lds_pages = reinterpret_cast<int*>(lds_m + kRows * 8);        // [8]: the waves' keys have pages
  int2* const lds_sees = reinterpret_cast<int2*>(lds_pages + kMaxWaves);   // [kRows]: first key and number of further ones that a row sees

  // column slab and head fastest: workgroups that read the same keys and values share an XCD's L2 (the hardware deals
  // workgroups to the eight XCDs in turn); late row blocks, which see the most keys, first
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
    // (anew for each piece and each use: kept out of the registers in between)
    const int lane = opaque(static_cast<int>(threadIdx.x) & 63), n = lane & 15, h = lane >> 4;
    int begin, end;
    take_piece<kRows>(a, at, progress, k, begin, end);
    // keys all_low .. all_high are seen by every row of the block
    const int all_low = chunk_start(a, k.position0 + token_of(a, k.row0 + k.count - 1)), all_high = min(k.position0 + token_of(a, k.row0), end - 1);

    // the two 16-key groups of a step: where this head's first value lies, and whether the group has a page
    constexpr int kBytes = kEight ? 1 : 2;
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
    const auto load_values = [&](const Step& t, int g, Values<kEight, kCols>& x) {
      // (columns behind the last are computed from others and not written)
      const int l = opaque(lane);
      const uint32_t offset = (static_cast<uint32_t>(4 * (l >> 4)) * a.v.slot + min(first_column + g * 16 * kCols + (l & 15) * kCols, a.v.width - kCols)) * kBytes;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        x.x[i] = *reinterpret_cast<const typename Values<kEight, kCols>::Piece*>(t.from[i >> 2] + (offset + static_cast<uint32_t>((i & 3) * a.v.slot * kBytes)));
    };
    const auto load_exponents = [&](const Step& t, uint32_t* e) {
      if constexpr (kEight) {
        const uint32_t offset = static_cast<uint32_t>(4 * (opaque(lane) >> 4)) * a.v.eSlot;
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = t.exponents[i >> 2][offset + static_cast<uint32_t>((i & 3) * a.v.eSlot)];
      }
    };

    f32x4 acc[RT][CT];
    float m[RT], l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      m[rt] = -__builtin_inff(), l[rt] = 0.f;
#pragma unroll
      for (int c = 0; c < CT; ++c) acc[rt][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    // the next 32 keys' values are on their way while these are worked on
    Values<kEight, kCols> x[kGroups];
    uint32_t e[8];
    bool there[2] = {false, false};
    // keys: the first 128 elements of the wave's 32 are on their way before the tile is reached, the others follow into their registers
    constexpr int kChunk = KS < 4 ? KS : 4, kLoads = kEight ? kChunk / 2 : kChunk;  // steps; a lane's 16-byte parts: 8 elements of 32, or 16 of 64
    struct Keys {
      const uint8_t* from[2];
      const uint8_t* exponents[2];
      int place[2];
      bool there[2];
    };
    u32x4 kx[2][kStaged ? 1 : kLoads];
    uint32_t ke[2];
    const auto keys_at = [&](int group) {
      Keys t;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int held = min(group + 16 * half, (end - 1) & ~15);
        const Page page = page_of(a, k.sequence, held);
        t.there[half] = page.there, t.place[half] = held & page_mask;
        t.from[half] = static_cast<const uint8_t*>(a.k.rows) + (page.number * a.k.page + static_cast<int64_t>(head) * a.k.head) * kBytes;
        if constexpr (kEight) t.exponents[half] = a.k.exponents + (page.number * a.k.ePage + static_cast<int64_t>(head) * a.k.eHead + static_cast<int64_t>(t.place[half]) * a.k.eSlot);
      }
      return t;
    };
    const auto load_key = [&](const Keys& t, int half, int part) {
      const int l = opaque(lane), d = min((kEight ? 64 : 32) * part + (kEight ? 16 : 8) * (l >> 4), a.k.width - (kEight ? 16 : 8));
      kx[half][part % kLoads] = *reinterpret_cast<const u32x4*>(t.from[half] + (static_cast<uint32_t>(t.place[half] + (l & 15)) * a.k.slot + d) * kBytes);
    };
    const auto load_first_keys_at = [&](const Keys& t) {
      if constexpr (kEight) {
        const uint32_t offset = static_cast<uint32_t>(opaque(lane) & 15) * a.k.eSlot;
#pragma unroll
        for (int half = 0; half < 2; ++half) ke[half] = t.exponents[half][offset];
      }
      if constexpr (kStaged) {
        // piece p of row r lies at p ^ (r & 15) (& 7 where there are eight): sixteen rows' equal pieces are in different banks
        constexpr int kRowsAtOnce = 64 / kPieces, kMix = kPieces < 16 ? kPieces - 1 : 15;
        const int l = opaque(lane), row = l / kPieces, last = a.k.width * kBytes / 16 - 1;
        const uint32_t to = lds_address(lds_k + wave * 32 * kPieces);
#pragma unroll
        for (int i = 0; i < 32 / kRowsAtOnce; ++i) {
          const int in_half = (i * kRowsAtOnce & 15) + row, half = i * kRowsAtOnce >> 4;
          const uint32_t offset = static_cast<uint32_t>(t.place[half] + in_half) * a.k.slot * kBytes + min((l % kPieces) ^ (in_half & kMix), last) * 16;
          load_to_lds16(t.from[half], offset, to + i * 1024);
        }
      } else {
#pragma unroll
        for (int part = 0; part < kLoads; ++part)
#pragma unroll
          for (int half = 0; half < 2; ++half) load_key(t, half, part);
      }
    };
    const auto load_first_keys = [&](int tile) {
      if (tile + 32 * wave < end) load_first_keys_at(keys_at(tile + 32 * wave));
    };
    const uint4 first_rows = static_cast<int>(threadIdx.x) < kRows * KS * 4 ? row_piece<KS>(a, k, head, threadIdx.x) : make_uint4(0, 0, 0, 0);
    if (begin < end) {  // (all of the pages first: one wait for their numbers)
      const Keys keys = keys_at(min(begin + 32 * wave, (end - 1) & ~31));
      const Step t = step_at(begin);
      if (begin + 32 * wave < end) load_first_keys_at(keys);
      load_exponents(t, e);
#pragma unroll
      for (int g = 0; g < kGroups; ++g) load_values(t, g, x[g]);
      there[0] = t.there[0], there[1] = t.there[1];
    }
    if (static_cast<int>(threadIdx.x) < kRows * KS * 4) row_piece_to_lds<kEight, KS>(first_rows, threadIdx.x, lds_q);
    for (int c = threadIdx.x + blockDim.x; c < kRows * KS * 4; c += blockDim.x) row_piece_to_lds<kEight, KS>(row_piece<KS>(a, k, head, c), c, lds_q);
    ranges_to_lds<kRows>(a, k, end, lds_sees);
    for (int c = threadIdx.x; c < kRows * 8; c += blockDim.x) lds_m[c] = -__builtin_inff();  // (of waves that there are not, too)
    if (threadIdx.x < kMaxWaves) lds_pages[threadIdx.x] = 1;
    __syncthreads();

    // 32 keys' values into the accumulators, those of the 32 after them called for (of these once more at the end: a load that is
    // always made needs no wait where it might not have been).  kAll: every row sees every one of the keys
    const auto values_of = [&](int tile, int step, auto all) {
      constexpr bool kAll = decltype(all)::value;
      const int first = tile + 32 * step;
      const Step next = step_at(min(first + 32, (end - 1) & ~31));
      u32x4 p[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) p[rt] = __builtin_bit_cast(u32x4, lds_p[(step * RT + rt) * 64 + lane]);
      bool odd = false;
      float unit[8];
      if constexpr (kEight) {
#pragma unroll
        for (int i = 0; i < 8; ++i) unit[i] = exponent_value(e[i]);
        load_exponents(next, e);
      }
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        uint32_t w[8][kCols / 2];
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int j = 0; j < kCols / 2; ++j) {
            if constexpr (kEight)
              w[i][j] = (j & 1) ? widen<DT, true>(x[g].x[i][j >> 1], unit[i]) : widen<DT, false>(x[g].x[i][j >> 1], unit[i]);
            else
              w[i][j] = x[g].x[i][j];
          }
        // what is not there, or not this workgroup's, must not meet a probability of zero as an infinity or NaN; nor must such a
        // value of a key that only some rows see, which goes to those alone below
        if constexpr (!kAll)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int key = first + 16 * (i >> 2) + 4 * h + (i & 3);
            const uint32_t keep = key >= k.begin && key < end && there[i >> 2] ? ~0u : 0u;
#pragma unroll
            for (int j = 0; j < kCols / 2; ++j) {
              const uint32_t finite = finite_halves<DT>(w[i][j]);
              odd = odd || (~finite & keep) != 0;
              w[i][j] &= keep & finite;
            }
          }
        u32x4 vt[kCols];
#pragma unroll
        for (int j = 0; j < kCols / 2; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            vt[2 * j][i] = __builtin_amdgcn_perm(w[2 * i + 1][j], w[2 * i][j], 0x05040100);
            vt[2 * j + 1][i] = __builtin_amdgcn_perm(w[2 * i + 1][j], w[2 * i][j], 0x07060302);
          }
        load_values(next, g, x[g]);
        __builtin_amdgcn_sched_barrier(0);  // (in front of the products, not behind them)
#pragma unroll
        for (int c = 0; c < kCols; ++c)
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) acc[rt][g * kCols + c] = mma<DT>(vt[c], p[rt], acc[rt][g * kCols + c]);
      }
      if constexpr (!kAll)
        if (__any(odd))
          add_odd_values<DT, kEight, kCols>(a, k, end, first, first_column, step_at(first), lds_sees, [&](int rt, int slot) -> uint32_t {
            return reinterpret_cast<const uint16_t*>(lds_p + (step * RT + rt) * 64 + (slot & ~7) * 2 + (opaque(lane) & 15))[slot & 7];
          }, acc);
      there[0] = next.there[0], there[1] = next.there[1];
    };

    for (int tile = begin; tile < end; tile += 32 * waves) {
      // ---- scores of the wave's 32 keys
      const int mine = tile + 32 * wave;
      f32x4 s[2][RT];
      bool pages_there = true;
      if (mine < end) {
        const bool whole = mine >= all_low && mine + 31 <= all_high;
        const Keys keys = keys_at(mine);
        pages_there = keys.there[0] && keys.there[1];
        // (younger than the keys: the values of the next step, and their exponents)
        if constexpr (kStaged) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kGroups * 8 + (kEight ? 8 : 0)) : "memory");
        u32x4 q[RT], q_next[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          q_next[rt] = __builtin_bit_cast(u32x4, lds_q[rt * KS * 64 + lane]);
          s[0][rt] = s[1][rt] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int c = 0; c < KS; ++c) {
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {  // (the rows' operands one step ahead; the fence keeps it at that)
            q[rt] = q_next[rt];
            if (c + 1 < KS) q_next[rt] = __builtin_bit_cast(u32x4, lds_q[(rt * KS + c + 1) * 64 + lane]);
          }
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int part = kEight ? c >> 1 : c;
            u32x4 key;
            if constexpr (kStaged) {
              const int l = opaque(lane), n = l & 15;
              key = __builtin_bit_cast(u32x4, lds_k[(wave * 32 + 16 * half + n) * kPieces + ((4 * part + (l >> 4)) ^ (n & (kPieces < 16 ? kPieces - 1 : 15)))]);
            } else {
              key = kx[half][part % kLoads];
            }
            if constexpr (kEight) {
              const uint32_t lo = (c & 1) ? key[2] : key[0], hi = (c & 1) ? key[3] : key[1];
              const float unit = exponent_value(ke[half]);
              key = u32x4{widen<DT, false>(lo, unit), widen<DT, true>(lo, unit), widen<DT, false>(hi, unit), widen<DT, true>(hi, unit)};
            }
            if (a.k.width != 32 * KS) {  // (behind the row's end the rows' operands are zero, and infinity times zero is not)
              const int d = kEight ? (c >> 1) * 64 + (opaque(lane) >> 4) * 16 : c * 32 + (opaque(lane) >> 4) * 8;
              if (d >= a.k.width) key = u32x4{0, 0, 0, 0};
            }
            if (!kStaged && c + kChunk < KS && (!kEight || (c & 1))) load_key(keys, half, part + kLoads);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) s[half][rt] = mma<DT>(key, q[rt], s[half][rt]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) s[half][rt] *= a.scale;
          if (!whole || !keys.there[half]) {
            const int l = opaque(lane), first = mine + 16 * half + 4 * (l >> 4);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
              const int2 range = lds_sees[rt * 16 + (l & 15)];
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (!keys.there[half] || !in_range(range, first + i)) s[half][rt][i] = -__builtin_inff();
            }
          }
        }
      } else {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s[0][rt] = s[1][rt] = f32x4{-__builtin_inff(), -__builtin_inff(), -__builtin_inff(), -__builtin_inff()};
      }
      load_first_keys(tile + 32 * waves);

      // ---- the rows' new maxima
      float top[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        float t = fmaxf(fmaxf(s[0][rt][0], s[0][rt][1]), fmaxf(s[0][rt][2], s[0][rt][3]));
        t = fmaxf(t, fmaxf(fmaxf(s[1][rt][0], s[1][rt][1]), fmaxf(s[1][rt][2], s[1][rt][3])));
        top[rt] = four_max(t);
      }
      if (waves > 1) {
        if (h == 0)
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) lds_m[(rt * 16 + n) * 8 + wave] = top[rt];
        if (lane == 0) lds_pages[wave] = pages_there;
        __syncthreads();
        const int4 u = *reinterpret_cast<const int4*>(lds_pages), v = *reinterpret_cast<const int4*>(lds_pages + 4);
        pages_there = __builtin_amdgcn_readfirstlane(u.x & u.y & u.z & u.w & v.x & v.y & v.z & v.w) != 0;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const float4 u = *reinterpret_cast<const float4*>(lds_m + (rt * 16 + n) * 8), v = *reinterpret_cast<const float4*>(lds_m + (rt * 16 + n) * 8 + 4);
          top[rt] = fmaxf(fmaxf(fmaxf(u.x, u.y), fmaxf(u.z, u.w)), fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)));
        }
      }

      // ---- probabilities, in the operand order of the second product
      bool moved = false;
      float alpha[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const float now = top[rt] > m[rt] + kSlack ? top[rt] : m[rt], held = now == -__builtin_inff() ? 0.f : now, base = held - kLift<DT>;
        alpha[rt] = __builtin_amdgcn_exp2f(m[rt] - held);
        moved = moved || now != m[rt];
        m[rt] = now;
        float p[8], sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          p[i] = __builtin_amdgcn_exp2f(s[i >> 2][rt][i & 3] - base);
          sum += p[i];
        }
        l[rt] = l[rt] * alpha[rt] + sum;
        lds_p[(wave * RT + rt) * 64 + lane] = make_uint4(pack2<DT>(p[0], p[1]), pack2<DT>(p[2], p[3]), pack2<DT>(p[4], p[5]), pack2<DT>(p[6], p[7]));
        __builtin_amdgcn_sched_barrier(0);
      }
      if (__any(moved))
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int c = 0; c < CT; ++c) acc[rt][c] *= alpha[rt];
      __syncthreads();

      // ---- values: 32 keys a step
      const int steps = min(waves, (end - tile + 31) >> 5);
      int step = 0;
      const int all = pages_there && tile >= all_low ? min(steps, (all_high + 1 - tile) >> 5) : 0;
      for (; step < all; ++step) values_of(tile, step, std::true_type());
      for (; step < steps; ++step) values_of(tile, step, std::false_type());
    }

    // ---- the rows' sums over the lanes and waves that had their keys
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) l[rt] = four_sum(l[rt]);
    if (waves > 1) {
      __syncthreads();  // (the maxima of the last tile have been read)
      if (h == 0)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) lds_m[(rt * 16 + n) * 8 + wave] = l[rt];
      __syncthreads();
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) l[rt] = sum_of_waves(lds_m + (rt * 16 + n) * 8, waves);
    }
    const Destination to = destination_of(a, progress, static_cast<int>(id), head);
    if (to.fits) store_piece<DT, RT, CT, kCols>(a, k, to, head, slab == 0 && wave == 0, first_column, acc, m, l);
    if (to.last) break;
    at = next_piece<kRows>(a, progress, k);
    __syncthreads();  // (the rows, maxima, probabilities and progress of this piece have been read)
  }
}

// Joins the pieces of the blocks that several workgroups had: o = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i with
// m = max_i m_i.  2^span_log2 lanes have a row: a group of 2^lanes_log2 of them, eight columns each, takes every n-th piece, n groups, in the
// pieces' order; the groups meet through the lanes.  Bound by the latency of three dependent loads where there are few rows (4 us), by the pieces' bytes
// else (100 MB read, 18 written: 21 us, 5.6 TB/s).
constexpr int kJoinThreads = 256;
template <int DT>
__global__ __launch_bounds__(kJoinThreads) void paged_join_kernel(AttnArgs a, int lanes_log2, int span_log2, uint32_t strips) {
  const int span = 1 << span_log2, lane = static_cast<int>(threadIdx.x) & (span - 1), lanes = 1 << lanes_log2, groups = span >> lanes_log2;
  const uint32_t item = blockIdx.x * (kJoinThreads >> span_log2) + (threadIdx.x >> span_log2), row = item / strips;
  const int64_t q_heads = a.heads * a.shared, all = a.clear_rest ? a.rows : row_bound(a.cu, a.view.batch, a.rows);
  if (row >= all * q_heads || row < row_bound(a.cu, 0, a.rows) * q_heads) return;
  const int2 join = a.joins[row];
  // (nor has every row one where cu decreases)
  if (join.x < 0 || join.y <= 0 || join.x + (join.y - 1) * static_cast<int64_t>(a.part_rows) >= static_cast<int64_t>(a.heads) * a.slots * a.part_rows) return;
  const int c = static_cast<int>(item - row * strips) * lanes * 8 + (lane & (lanes - 1)) * 8;
  const bool column = c < a.v.width;
  float m = -__builtin_inff(), l = 0.f, o[8] = {};
#pragma unroll 4
  for (int i = lane >> lanes_log2; i < join.y; i += groups) {
    const int64_t at = join.x + static_cast<int64_t>(i) * a.part_rows;
    const float2 stat = *reinterpret_cast<const float2*>(a.stats + at * 2);
    const float4* from = reinterpret_cast<const float4*>(a.part + at * a.v.width + (column ? c : 0));
    const float4 x = from[0], y = from[1];
    const float now = fmaxf(m, stat.x), base = now == -__builtin_inff() ? 0.f : now;
    const float before = __builtin_amdgcn_exp2f(m - base), with = __builtin_amdgcn_exp2f(stat.x - base);
    const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    m = now;
    l = l * before + stat.y * with;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = o[j] * before + v[j] * with;
  }
  float now = m;
  for (int off = lanes; off < span; off <<= 1) now = fmaxf(now, across(now, off));
  const float with = __builtin_amdgcn_exp2f(m - (now == -__builtin_inff() ? 0.f : now));
  l *= with;
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j] *= with;
  for (int off = lanes; off < span; off <<= 1) {
    l += across(l, off);
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] += across(o[j], off);
  }
  if (lane >= lanes || !column) return;
  const float inverse = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j] = l == 0.f ? 0.f : o[j] * inverse;
  *reinterpret_cast<uint4*>(a.out + static_cast<int64_t>(row) * a.v.width + c) = pack8<DT>(o);
}

// How a call is cut.
struct Plan {
  int rt, ct, ks, waves, slabs;
  int64_t blocks, parts;  // row blocks at most; parts of the line of units for each head and slab (0: a workgroup a block)
  int64_t slots, part_rows;
  int join_lanes_log2, join_span_log2;  // of the join: lanes to a row's strip in a piece, in all pieces
  int64_t workgroups(int64_t heads) const { return (parts > 0 ? parts : blocks) * heads * slabs; }
};

Plan plan_of(const mega_paged_cache* c, int64_t rows, int64_t q_heads) {
  Plan p{};
  const int64_t shared = q_heads / c->heads, sequences = std::max<int64_t>(c->batch, 1);
  // rows of a sequence, on average: a block's rows pad to the next size
  const int64_t mean = (rows * shared + sequences - 1) / sequences;
  p.ks = c->k_width <= 128 ? 4 : c->k_width <= 256 ? 8 : 16;
  p.rt = mean <= 16 ? 1 : mean <= 32 || p.ks == 16 ? 2 : 4;  // (keys of 512 and four row tiles do not fit the registers)
  p.ct = p.rt == 1 && c->v_width > 1024 ? 16 : 8;
  const int64_t per_wave = 16 * p.ct, kRows = 16 * p.rt;
  p.slabs = static_cast<int>((c->v_width + kMaxWaves * per_wave - 1) / (kMaxWaves * per_wave));
  const int64_t slab = (c->v_width + p.slabs - 1) / p.slabs;
  p.waves = static_cast<int>((slab + per_wave - 1) / per_wave);
  p.blocks = rows * shared / kRows + c->batch + 1;
  // workgroups that the chip holds at a time: eight waves to a CU
  const int64_t resident = kCus * kMaxWaves / p.waves, pairs = c->heads * p.slabs;
  const int64_t full = std::max(rows * shared / kRows, std::min(c->batch, rows)) * pairs;
  // A line of units up to four times that many blocks, a workgroup a block above.  Two to four times: 128 single tokens behind 100 - 4000, wide heads,
  // 854 us on the line against 988, 256 on shared heads 414 against 484; prompts the other way, 4096 tokens 265 against 210, as their pieces' rows are more
  // bytes than their keys.  Behind four times: 8192 tokens 614 against 431, 512 single tokens on shared heads the same.
  if (c->batch > 0 && full < 4 * resident && p.blocks * (c->table_width * c->page_size / 32 + 9) < 0x40000000 &&
      (resident + p.blocks) * c->heads * kRows < 0x40000000 && rows * q_heads < 0x1000000) {
    p.parts = std::max<int64_t>(1, resident / pairs);
    p.part_rows = std::min(kRows, rows * shared);
    p.slots = p.parts + p.blocks;
    // the join: as many pieces of a row at a time as it has on average
    const int64_t pieces = p.parts * pairs / std::max<int64_t>(full, 1);
    p.join_lanes_log2 = pieces > 8 ? 2 : pieces > 4 ? 3 : pieces > 2 ? 4 : 5;
    while (p.join_lanes_log2 > 1 && (8 << (p.join_lanes_log2 - 1)) >= c->v_width) --p.join_lanes_log2;
    // (lanes for no more pieces than twice that, the rest have other rows: 1.6 pieces of 128 columns, 28 us with a wave a row)
    p.join_span_log2 = p.join_lanes_log2;
    while (p.join_span_log2 < 6 && (int64_t{1} << (p.join_span_log2 - p.join_lanes_log2)) < 2 * pieces) ++p.join_span_log2;
  }
  return p;
}

template <int DT, bool kEight, int RT, int CT, int KS>
int launch_few(const AttnArgs& a, const Plan& p, void* stream) {
  const auto kernel = paged_attn_kernel<DT, kEight, RT, CT, KS>;
  const size_t bytes = (RT * KS * 64 + p.waves * (RT * 64 + (staged(kEight, RT, KS) ? 32 * KS * (kEight ? 2 : 4) : 0))) * sizeof(uint4) + RT * 16 * 8 * sizeof(float) + kMaxWaves * sizeof(int) + RT * 16 * sizeof(int2);
  if (bytes > 65536)
    MEGA_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)));
  hipStream_t s = static_cast<hipStream_t>(stream);
  kernel<<<grid_of(p.workgroups(a.heads)), dim3(p.waves * kWave), bytes, s>>>(a);
  MEGA_CHECK_LAUNCH();
  return MEGA_OK;
}

template <int DT, bool kEight, int KS>
int launch_rows(const AttnArgs& a, const Plan& p, void* stream) {
  if (p.rt == 2) return launch_few<DT, kEight, 2, 8, KS>(a, p, stream);
  return p.ct == 16 ? launch_few<DT, kEight, 1, 16, KS>(a, p, stream) : launch_few<DT, kEight, 1, 8, KS>(a, p, stream);
}

template <int DT, bool kEight>
int launch_width(const AttnArgs& a, const Plan& p, void* stream) {
  if (p.ks == 4) return launch_rows<DT, kEight, 4>(a, p, stream);
  if (p.ks == 8) return launch_rows<DT, kEight, 8>(a, p, stream);
  return launch_rows<DT, kEight, 16>(a, p, stream);
}

template <int DT>
int launch_attn(const AttnArgs& a, const Plan& p, bool eight, void* stream) {
  int rc;
  if (p.rt == 4)
    rc = launch_paged_rows(a, RowsPlan{p.ks, p.waves, p.workgroups(a.heads)}, DT, eight, stream);
  else
    rc = eight ? launch_width<DT, true>(a, p, stream) : launch_width<DT, false>(a, p, stream);
  if (rc != MEGA_OK || p.parts == 0) return rc;
  const int64_t strip = 8 << p.join_lanes_log2, strips = (a.v.width + strip - 1) / strip, items = static_cast<int64_t>(a.rows) * a.heads * a.shared * strips;
  const int64_t at_once = kJoinThreads >> p.join_span_log2;
  paged_join_kernel<DT><<<dim3(static_cast<uint32_t>((items + at_once - 1) / at_once)), dim3(kJoinThreads), 0, static_cast<hipStream_t>(stream)>>>(
      a, p.join_lanes_log2, p.join_span_log2, static_cast<uint32_t>(strips));
  MEGA_CHECK_LAUNCH();
  return MEGA_OK;
}

// the logarithm of a power of two, else -1
int log2_of(int64_t n) {
  int l = 0;
  while ((int64_t{1} << l) < n) ++l;
  return (int64_t{1} << l) == n ? l : -1;
}

bool sizes_fit(const mega_paged_cache* c, int64_t rows, int64_t q_heads, int64_t chunk) {
  return c != nullptr && c->heads >= 1 && c->v_width >= 16 && rows >= 0 && rows <= 0x7fffffff && q_heads >= 1 && q_heads <= 65536 &&
         q_heads % c->heads == 0 && chunk >= 0 && chunk <= 0x7fffffff && rows * q_heads <= (int64_t{1} << 40) / c->v_width;
}

}  // namespace
}  // namespace mega

using namespace mega;

extern "C" int64_t mega_paged_attention_workspace_bytes(const mega_paged_cache* cache, int64_t rows, int64_t q_heads, int64_t chunk) {
  if (!sizes_fit(cache, rows, q_heads, chunk) || rows == 0) return 0;
  const Plan p = plan_of(cache, rows, q_heads);
  return p.parts > 0 ? cache->heads * p.slots * p.part_rows * (cache->v_width + 2) * static_cast<int64_t>(sizeof(float)) + rows * q_heads * static_cast<int64_t>(sizeof(int2)) : 0;
}

extern "C" int mega_paged_attention_fwd(const mega_paged_cache* cache, int dtype, const void* q, int64_t q_row, int64_t q_head,
                                        const int32_t* lengths, const int32_t* cu, int64_t rows, int64_t q_heads, double scale,
                                        int64_t chunk, void* out, int clear_rest, void* workspace, void* stream) {
  if (const int rc = check_paged_cache(cache, dtype, "mega_paged_attention_fwd"); rc != MEGA_OK) return rc;
  MEGA_CHECK_ARG(sizes_fit(cache, rows, q_heads, chunk), "mega_paged_attention_fwd: bad sizes (q_heads has to be a multiple of the cache's heads)");
  MEGA_CHECK_ARG(cache->k_width <= kMaxKeyWidth, "mega_paged_attention_fwd: k_width must be at most 512");
  if (rows == 0 || (cache->batch == 0 && clear_rest == 0)) return MEGA_OK;
  MEGA_CHECK_ARG(q != nullptr && out != nullptr && (lengths != nullptr || cache->batch == 0) && cu != nullptr, "mega_paged_attention_fwd: null pointer");
  MEGA_CHECK_ARG(reinterpret_cast<uintptr_t>(q) % 16 == 0 && q_row % 8 == 0 && q_head % 8 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0,
                 "mega_paged_attention_fwd: q and out must be 16-byte aligned");
  const Plan p = plan_of(cache, rows, q_heads);
  MEGA_CHECK_ARG(p.workgroups(cache->heads) <= 0x7fffffff && rows * (q_heads / cache->heads) <= 0x7fffffff, "mega_paged_attention_fwd: too many rows for one launch");
  MEGA_CHECK_ARG(p.parts == 0 || (workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
                 "mega_paged_attention_fwd: a 16-byte aligned workspace is needed");
  AttnArgs a{};
  a.view = paged_view(cache), a.k = paged_pool(cache, false), a.v = paged_pool(cache, true);
  a.q = static_cast<const uint16_t*>(q), a.q_row = q_row, a.q_head = q_head;
  a.lengths = lengths, a.cu = cu, a.out = static_cast<uint16_t*>(out);
  a.part = static_cast<float*>(workspace);
  if (p.parts > 0) {
    a.stats = a.part + cache->heads * p.slots * p.part_rows * cache->v_width;
    a.joins = reinterpret_cast<int2*>(a.stats + cache->heads * p.slots * p.part_rows * 2);
  }
  a.rows = static_cast<int32_t>(rows), a.heads = static_cast<int32_t>(cache->heads), a.shared = static_cast<int32_t>(q_heads / cache->heads);
  a.chunk = static_cast<int32_t>(chunk), a.slabs = p.slabs, a.blocks = static_cast<int32_t>(p.blocks);
  a.parts = static_cast<int32_t>(p.parts), a.slots = static_cast<int32_t>(p.slots), a.part_rows = static_cast<int32_t>(p.part_rows);
  a.clear_rest = clear_rest != 0;
  a.chunk_shift = log2_of(a.chunk), a.shared_shift = log2_of(a.shared);
  // (0, 1, 8, 16 units: few rows, 16 tokens behind 10 - 400 29, 24, 24, 27 us, 128 on shared heads behind 500 - 16000 778, 775, 782, 792; many rows, eight pieces
  // on shared heads in 8 bits 654, 606, 506, 526, a prompt of 2048 156, 140, 99, 104)
  a.lead = p.rt == 4 ? 8 : 1;
  a.per_part = p.parts > 0 ? 1.0 / static_cast<double>(p.parts) : 0.0;
  a.scale = static_cast<float>(std::fabs(scale) * 1.4426950408889634);
  if (a.scale < FLT_MIN) a.scale = FLT_MIN;  // (a scale of zero: every score is zero, and a masked one's infinity stays one)
  a.sign = scale < 0.0 ? 0x80008000u : 0u;
  const bool eight = cache->k_exponents != nullptr;
  return dtype == MEGA_BF16 ? launch_attn<MEGA_BF16>(a, p, eight, stream) : launch_attn<MEGA_F16>(a, p, eight, stream);
}
