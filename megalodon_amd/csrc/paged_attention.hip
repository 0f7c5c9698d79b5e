// Attention of new tokens over the paged key / value cache.
//
// For row r (a new token's query of one head) with visible keys lo .. hi
//   s_j = scale q . k_j,  m = max_j s_j,  l = sum_j e^(s_j - m),  o = sum_j e^(s_j - m) v_j / l,
// in one pass over the keys with the running m and l; accumulators follow a rising m by the factor
// e^(m_old - m_new).  Scores, m, l and o are float32; the probabilities that go into the second product are
// rounded to the operands' type, which is what the matrix cores take (each is off by 2^-9 or 2^-12 of itself at most,
// below the rounding of the result); l sums them unrounded.
//
// Layout.  A workgroup has kRows = 16 RT rows (new tokens of one sequence, and the query heads that share a key /
// value head, side by side) of one cache head, and W waves; wave w has 16 CT of its value columns.  A tile is
// 32 W keys:
//   scores   wave w takes 32 of them, all rows: S^T = K Q^T with K straight from the pool into registers (its rows
//            are the instruction's k-contiguous operand) and Q from LDS in operand order;
//   softmax  a row's keys lie in four lanes of a wave and in W waves: maxima meet in LDS, P^T goes there;
//   values   every wave takes all 32 W keys for its own columns: O^T = V^T P^T.  No value is read twice in a
//            workgroup, so values pass through registers only: a lane reads eight columns of eight keys, and a byte
//            permutation pairs neighbouring keys -- column 8 n + j of lane n's eight becomes row n of operand j.
// Both products have the rows along the lanes, so a row's m, l and rescaling factor live in its lanes, and P^T
// leaves the first product in the very registers that the second one takes: which of the 32 keys sits in which k slot is
// free as long as V agrees, and slot (8 h + i) is key 4 h + i of the first 16 for i < 4, of the second 16 above.
//
// A page holds 16 keys at least, and key groups are aligned, so a lane group's keys share a page: its base is a scalar.
//
// Few row blocks (single tokens, drafts, one prompt's piece): bound by the cache's bytes.  The blocks' keys, in units of 32,
// form one line, block after block, which is cut into as many equal parts as workgroups fill the chip, whatever
// the sequences' lengths: a workgroup goes through the pieces of blocks that its part holds, leaves each one's (o, m, l)
// in a workspace in float32, and a second kernel joins them.  Many row blocks: a workgroup each, bound by the
// matrix cores and by what L2 gives for the operands.
#include "paged.hpp"

#include <algorithm>
#include <type_traits>

namespace mega {
namespace {

constexpr int kMaxWaves = 8;
constexpr int kMaxKeyWidth = 512;
constexpr int kCus = 256;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct AttnArgs {
  PagedView view;
  PagedPool k, v;
  const uint16_t* q;
  int64_t q_row, q_head;
  const int32_t *lengths, *cu;
  uint16_t* out;
  float *part, *stats;        // parts > 0: (heads, slots, part_rows, v_width), (heads, slots, part_rows, 2)
  int2* joins;                // ... (rows, q_heads): a row's first place in the former and its number of pieces (0: out has it)
  int32_t rows, heads, shared, chunk, slabs, blocks;
  int32_t parts, slots, part_rows;  // parts of the line of units for each head and slab; 0: a workgroup a block
  int32_t clear_rest;
  float scale;                // times log2(e)
};

// A row block of one sequence and the keys that any of its rows sees.
struct Block {
  int32_t sequence;
  int32_t start, row0, count;  // first packed row of the sequence; first row (token * shared + head) and their number
  int32_t position0;           // position of the sequence's first new token
  int32_t keys;                // positions that have a place
  int32_t begin, end;          // keys that the block sees, [begin, end)
};

// A load that the scalar unit may make: of what no kernel writes while this one runs, at an address that a wave has in common.
typedef const int32_t __attribute__((address_space(4))) ConstInt;
__device__ __forceinline__ int32_t constant_at(const int32_t* p, int64_t i) { return reinterpret_cast<ConstInt*>(reinterpret_cast<uint64_t>(p))[i]; }

__device__ __forceinline__ int chunk_start(int position, int chunk) { return chunk > 0 && position > 0 ? position / chunk * chunk : 0; }

// Sequences, the rows behind the last one counted as one more where they are to be cleared.
__device__ __forceinline__ int sequences_of(const AttnArgs& a) { return a.view.batch + (a.clear_rest ? 1 : 0); }

// Sequence b (the rows behind the last one are one more, without keys) and its row block `number`; false: it has no such block.
template <int kRows>
__device__ __forceinline__ bool block_of(const AttnArgs& a, int b, int64_t number, Block& k) {
  k.sequence = b;
  k.start = row_bound(a.cu, b, a.rows);
  const int n = (b < a.view.batch ? row_bound(a.cu, b + 1, a.rows) : a.rows) - k.start;
  const int64_t row0 = number * kRows;
  if (row0 < 0 || row0 >= static_cast<int64_t>(n) * a.shared) return false;
  k.row0 = static_cast<int32_t>(row0);
  k.count = static_cast<int32_t>(min(static_cast<int64_t>(kRows), static_cast<int64_t>(n) * a.shared - row0));
  const int length = b < a.view.batch ? max(a.lengths[b], 0) : 0;
  k.keys = static_cast<int32_t>(min(static_cast<int64_t>(length), static_cast<int64_t>(a.view.table_width) << a.view.page_shift));
  k.position0 = length - n;
  k.begin = chunk_start(k.position0 + k.row0 / a.shared, a.chunk);
  k.end = min(k.position0 + (k.row0 + k.count - 1) / a.shared + 1, k.keys);
  return true;
}

// A workgroup a block: blocks are numbered so that sequence b's begin at cu[b] shared / kRows + b, which leaves ceil(n shared / kRows)
// numbers before the next sequence's whatever the lengths are, and the host need not know these.
template <int kRows>
__device__ __forceinline__ bool find_block(const AttnArgs& a, int number, Block& k) {
  const int sequences = sequences_of(a);
  const auto first = [&](int b) { return static_cast<int64_t>(row_bound(a.cu, b, a.rows)) * a.shared / kRows + b; };
  const int b = last_not_above(sequences, number, first);
  return block_of<kRows>(a, b, number - first(b), k);
}

// The line of units.  Every block of a sequence has as many units as its last one sees keys from the first one's first on
// (all of them in front of a chunk's border alike; the earlier blocks' last units are empty), and one if there are none.
struct Share {
  int32_t blocks, units;  // of a sequence: row blocks, units of each
  int32_t from;           // its first unit's first key
};
template <int kRows>
__device__ __forceinline__ Share share_of(const AttnArgs& a, int b) {
  const bool rest = b >= a.view.batch;
  const int start = row_bound(a.cu, b, a.rows), n = (rest ? a.rows : row_bound(a.cu, b + 1, a.rows)) - start, length = rest ? 0 : max(a.lengths[b], 0);
  if (n <= 0) return {0, 0, 0};
  const int keys = static_cast<int>(min(static_cast<int64_t>(length), static_cast<int64_t>(a.view.table_width) << a.view.page_shift));
  const int from = chunk_start(length - n, a.chunk) & ~31;
  return {static_cast<int32_t>((static_cast<int64_t>(n) * a.shared + kRows - 1) / kRows), max(keys - from + 31, 32) >> 5, from};
}
// A place on the line: the sequence, its share, and the blocks and units in front of it.
struct Mark {
  int32_t sequence;
  Share share;
  int32_t blocks_before, units_before, total;  // total: of the whole line (the host cuts no line of 2^31 units)
};
// units of a part; the parts behind the line's end are empty
__device__ __forceinline__ int part_units(int total, int parts) { return (total + parts - 1) / parts; }
// The sequence in which part `part` begins (false: the part is empty); all lanes of a wave together, 64 sequences a round.
template <int kRows>
__device__ __forceinline__ bool find_mark(const AttnArgs& a, int part, Mark& mark) {
  const int lane = static_cast<int>(threadIdx.x) & 63, sequences = sequences_of(a);
  Share s{};
  int units = 0, blocks = 0;
  const auto round = [&](int b0) {  // inclusive sums over the lanes' sequences
    const int b = b0 + lane;
    s = b < sequences ? share_of<kRows>(a, b) : Share{0, 0, 0};
    units = s.blocks * s.units, blocks = s.blocks;
    for (int off = 1; off < min(64, sequences); off <<= 1) {
      const int u = __shfl_up(units, off, 64), c = __shfl_up(blocks, off, 64);
      if (lane >= off) units += u, blocks += c;
    }
  };
  mark.total = 0;
  for (int b0 = 0; b0 < sequences; b0 += 64) {
    round(b0);
    mark.total += __builtin_amdgcn_readlane(units, min(63, sequences - 1 - b0));
  }
  const int first = part * part_units(mark.total, a.parts);
  if (first >= mark.total) return false;
  int units_before = 0, blocks_before = 0;
  for (int b0 = 0; b0 < sequences; b0 += 64) {
    if (sequences > 64) round(b0);
    const uint64_t which = __ballot(b0 + lane < sequences && units_before + units > first);
    if (which != 0) {
      const int l = __ffsll(static_cast<unsigned long long>(which)) - 1;
      mark.sequence = b0 + l;
      mark.share = {__builtin_amdgcn_readlane(s.blocks, l), __builtin_amdgcn_readlane(s.units, l), __builtin_amdgcn_readlane(s.from, l)};
      mark.units_before = units_before + __builtin_amdgcn_readlane(units, l) - mark.share.blocks * mark.share.units;
      mark.blocks_before = blocks_before + __builtin_amdgcn_readlane(blocks, l) - mark.share.blocks;
      return true;
    }
    units_before += __builtin_amdgcn_readlane(units, 63);
    blocks_before += __builtin_amdgcn_readlane(blocks, 63);
  }
  return false;
}

template <int DT>
__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (DT == MEGA_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <int DT, bool kUpper>
__device__ __forceinline__ uint32_t widen(uint32_t codes, float scale) {
  if constexpr (DT == MEGA_BF16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, kUpper));
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, kUpper));
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (DT == MEGA_BF16) return pack_bf16x2(lo, hi);
  return static_cast<uint32_t>(float_to_f16_bits(lo)) | (static_cast<uint32_t>(float_to_f16_bits(hi)) << 16);
}

// ones over those halves of a word whose 16-bit numbers are finite
template <int DT>
__device__ __forceinline__ uint32_t finite_halves(uint32_t w) {
  constexpr uint32_t top = DT == MEGA_BF16 ? 0x7f80u : 0x7c00u;
  return ((w & top) == top ? 0u : 0xffffu) | ((w >> 16 & top) == top ? 0u : 0xffff0000u);
}

// v, of which the compiler knows nothing: what is computed from it is computed where it is used, not once ahead of a loop
// and kept in registers that the loop has no room for
__device__ __forceinline__ int opaque(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

__device__ __forceinline__ float across(float v, int mask) { return __shfl_xor(v, mask, 64); }

// The page of 16 keys: its number and whether there is one (0 otherwise, so that addresses stay in the pool).
struct Page {
  uint32_t number;
  bool there;
};
__device__ __forceinline__ Page page_of(const AttnArgs& a, int sequence, int key) {
  const uint32_t e = static_cast<uint32_t>(constant_at(a.view.table, sequence * a.view.table_stride + (key >> a.view.page_shift)));
  const bool there = e < static_cast<uint32_t>(a.view.pages);
  return {there ? e : 0, there};
}

// A lane's values of 32 keys in one group of 16 kCols columns, as they lie in the pool: kCols columns of eight keys.
template <bool kEight, int kCols>
struct Values {
  static constexpr int kWords = kCols * (kEight ? 1 : 2) / 4;
  typedef uint32_t Piece __attribute__((ext_vector_type(kWords)));
  Piece x[8];
};

// Where a workgroup is on the line of units, kept in LDS while it works on a piece.
struct Progress {
  Mark mark;
  int32_t unit, unit_end, per, number;
  int32_t pieces;  // of the block, this one included if it is the first; 0 for the others
  bool alone;      // the whole block is this workgroup's
};

template <int DT, bool kEight, int RT, int CT, int KS>  // KS: 32-wide steps of a key row
__global__ __launch_bounds__(kMaxWaves * kWave, 2) void paged_attn_kernel(AttnArgs a) {
  // 16-byte loads of values where the registers allow it: eight of a lane's columns at a time, else four
  constexpr int kRows = 16 * RT, kCols = RT > 1 && !kEight ? 4 : 8, kGroups = CT / kCols;
  extern __shared__ __align__(16) uint4 lds[];
  __shared__ Progress progress;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6), waves = static_cast<int>(blockDim.x) >> 6;
  uint4* const lds_q = lds;                       // [RT][KS][64]
  uint4* const lds_p = lds + RT * KS * 64;        // [waves][RT][64]
  float* const lds_m = reinterpret_cast<float*>(lds_p + waves * RT * 64);  // [kRows][8]
  int* const lds_pages = reinterpret_cast<int*>(lds_m + kRows * 8);        // [8]: the waves' keys have pages
  int2* const lds_sees = reinterpret_cast<int2*>(lds_pages + kMaxWaves);   // [kRows]: first key and number of further ones that a row sees

  // column slab and head fastest: workgroups that read the same keys and values share an XCD's L2 (the hardware deals
  // workgroups to the eight XCDs in turn); late row blocks, which see the most keys, first
  uint32_t id = blockIdx.x;
  const int slab = id % a.slabs;
  id /= a.slabs;
  const int head = id % a.heads;
  id /= a.heads;
  const int page_mask = (1 << a.view.page_shift) - 1;
  const int first_column = (slab * waves + wave) * CT * 16;

  Block k;
  if (a.parts == 0) {
    if (!find_block<kRows>(a, a.blocks - 1 - static_cast<int>(id), k)) return;
  } else {
    Progress at;
    if (!find_mark<kRows>(a, static_cast<int>(id), at.mark)) return;
    at.per = part_units(at.mark.total, a.parts);
    at.unit = static_cast<int>(id) * at.per, at.unit_end = min(at.unit + at.per, at.mark.total);
    if (threadIdx.x == 0) progress = at;
    __syncthreads();
  }

  for (;;) {
    // (anew for each piece and each use: kept out of the registers in between)
    const int lane = opaque(static_cast<int>(threadIdx.x) & 63), n = lane & 15, h = lane >> 4;
    int begin, end;
    if (a.parts == 0) {
      begin = k.begin & ~31, end = k.end;
    } else {
      Progress at = progress;
      __syncthreads();
      while (at.unit >= at.mark.units_before + at.mark.share.blocks * at.mark.share.units) {  // (unit < total: there is one)
        at.mark.units_before += at.mark.share.blocks * at.mark.share.units;
        at.mark.blocks_before += at.mark.share.blocks;
        at.mark.share = share_of<kRows>(a, ++at.mark.sequence);
      }
      const int units = at.mark.share.units;
      at.number = (at.unit - at.mark.units_before) / units;
      const int first = at.mark.units_before + at.number * units, last = min(first + units, at.unit_end);
      block_of<kRows>(a, __builtin_amdgcn_readfirstlane(at.mark.sequence), __builtin_amdgcn_readfirstlane(at.number), k);
      begin = __builtin_amdgcn_readfirstlane(max(at.mark.share.from + (at.unit - first) * 32, k.begin & ~31));
      end = __builtin_amdgcn_readfirstlane(min(at.mark.share.from + (last - first) * 32, k.end));
      const int begins_in = first / at.per, ends_in = (first + units - 1) / at.per;
      at.alone = begins_in == ends_in;
      at.pieces = begins_in == static_cast<int>(id) ? ends_in - begins_in + 1 : 0;
      at.unit = last;
      if (threadIdx.x == 0) progress = at;
    }

    // rows to LDS, in the order in which the matrix instructions take them
    for (int c = threadIdx.x; c < kRows * KS * 4; c += blockDim.x) {
      const int row = c / (KS * 4), d = c % (KS * 4);  // eight elements of a row
      uint4 x = make_uint4(0, 0, 0, 0);
      if (row < k.count && d * 8 < a.k.width) {
        const int r = k.row0 + row, t = r / a.shared, g = r - t * a.shared;
        x = *reinterpret_cast<const uint4*>(a.q + (static_cast<int64_t>(k.start) + t) * a.q_row + (static_cast<int64_t>(head) * a.shared + g) * a.q_head + d * 8);
      }
      // (8-bit keys: a lane reads 16 codes at a time, which serve two steps)
      const int step = kEight ? (d >> 3) * 2 + (d & 1) : d >> 2, quarter = kEight ? (d >> 1) & 3 : d & 3;
      lds_q[((row >> 4) * KS + step) * 64 + quarter * 16 + (row & 15)] = x;
    }

    // the rows' visible keys of this piece to LDS: low .. low + span (none: a low that no key reaches)
    for (int row = threadIdx.x; row < kRows; row += blockDim.x) {
      const int position = k.position0 + (k.row0 + row) / a.shared, low = chunk_start(position, a.chunk), high = min(position, end - 1);
      const bool none = row >= k.count || high < low;
      lds_sees[row] = none ? make_int2(0x7fffffff, 0) : make_int2(low, high - low);
    }
    const auto sees = [&](int2 range, int key) { return static_cast<uint32_t>(key) - static_cast<uint32_t>(range.x) <= static_cast<uint32_t>(range.y); };
    // keys all_low .. all_high are seen by every row of the block
    const int all_low = chunk_start(k.position0 + (k.row0 + k.count - 1) / a.shared, a.chunk), all_high = min(k.position0 + k.row0 / a.shared, end - 1);

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
    // the next 32 keys' values are on their way while these are worked on (four row tiles: within a tile of keys; beside the
    // scores there is no room for them)
    constexpr bool kAcross = RT < 4;
    Values<kEight, kCols> x[kGroups];
    uint32_t e[8];
    bool there[2] = {false, false};
    // keys: the wave's first 16 of a tile are on their way before the tile is reached, the second 16 take their registers
    constexpr int kLoads = kEight ? KS / 2 : KS;  // a lane's 16-byte parts of a row: 8 elements of 32, or 16 of 64
    struct Keys {
      const uint8_t* from;
      const uint8_t* exponents;
      int place;
      bool there;
    };
    u32x4 kx[kLoads];
    uint32_t ke[4];
    const auto keys_at = [&](int group) {
      Keys t;
      const int held = min(group, (end - 1) & ~15);
      const Page page = page_of(a, k.sequence, held);
      t.there = page.there, t.place = held & page_mask;
      t.from = static_cast<const uint8_t*>(a.k.rows) + (page.number * a.k.page + static_cast<int64_t>(head) * a.k.head) * kBytes;
      if constexpr (kEight) t.exponents = a.k.exponents + (page.number * a.k.ePage + static_cast<int64_t>(head) * a.k.eHead + static_cast<int64_t>(t.place) * a.k.eSlot);
      return t;
    };
    const auto load_key = [&](const Keys& t, int c) {
      const int l = opaque(lane), d = min((kEight ? 64 : 32) * c + (kEight ? 16 : 8) * (l >> 4), a.k.width - (kEight ? 16 : 8));
      kx[c] = *reinterpret_cast<const u32x4*>(t.from + (static_cast<uint32_t>(t.place + (l & 15)) * a.k.slot + d) * kBytes);
    };
    const auto load_key_exponents = [&](const Keys& t) {
      if constexpr (kEight) {
        const uint32_t offset = static_cast<uint32_t>(4 * (opaque(lane) >> 4)) * a.k.eSlot;
#pragma unroll
        for (int i = 0; i < 4; ++i) ke[i] = t.exponents[offset + static_cast<uint32_t>(i * a.k.eSlot)];
      }
    };
    const auto load_first_keys = [&](int tile) {
      if (tile + 32 * wave >= end) return;
      const Keys t = keys_at(tile + 32 * wave);
      load_key_exponents(t);
#pragma unroll
      for (int c = 0; c < kLoads; ++c) load_key(t, c);
    };
    const auto load_step = [&](int first) {
      const Step t = step_at(first);
      load_exponents(t, e);
#pragma unroll
      for (int g = 0; g < kGroups; ++g) load_values(t, g, x[g]);
      there[0] = t.there[0], there[1] = t.there[1];
    };
    if (kAcross) load_first_keys(begin);
    if (kAcross && begin < end) load_step(begin);
    for (int c = threadIdx.x; c < kRows * 8; c += blockDim.x) lds_m[c] = -__builtin_inff();  // (of waves that there are not, too)
    if (threadIdx.x < kMaxWaves) lds_pages[threadIdx.x] = 1;
    __syncthreads();

    // 32 keys' values into the accumulators, those of the 32 after them called for (kNext; of these once more at the end: a load that is
    // always made needs no wait where it might not have been).  kAll: every row sees every one of the keys
    const auto values_of = [&](int tile, int step, auto all, auto call) {
      constexpr bool kAll = decltype(all)::value, kNext = decltype(call)::value;
      const int first = tile + 32 * step;
      Step next;
      if constexpr (kNext) next = step_at(min(first + 32, (end - 1) & ~31));
      u32x4 p[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) p[rt] = __builtin_bit_cast(u32x4, lds_p[(step * RT + rt) * 64 + lane]);
      bool odd = false;
      float unit[8];
      if constexpr (kEight) {
#pragma unroll
        for (int i = 0; i < 8; ++i) unit[i] = exponent_value(e[i]);
        if constexpr (kNext) load_exponents(next, e);
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
        if constexpr (kNext) load_values(next, g, x[g]);
        __builtin_amdgcn_sched_barrier(0);  // (in front of the products, not behind them)
#pragma unroll
        for (int c = 0; c < kCols; ++c)
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) acc[rt][g * kCols + c] = mma<DT>(vt[c], p[rt], acc[rt][g * kCols + c]);
      }
      if constexpr (!kAll)
        if (__any(odd)) {  // key by key, its infinities and NaN into the rows that see it
          const Step t = step_at(first);
#pragma unroll 1
          for (int slot = 0; slot < 32; ++slot) {
            const int l = opaque(lane), n = l & 15, h = l >> 4;
            const int place = slot & 7, half = place >> 2, in_group = 4 * (slot >> 3) + (place & 3), key = first + 16 * half + in_group;
            if (key < k.begin || key >= end || !(half ? t.there[1] : t.there[0])) continue;
            const uint8_t* const row = (half ? t.from[1] : t.from[0]) + static_cast<int64_t>(in_group) * a.v.slot * kBytes;
            float weight[RT];
            bool its[RT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
              const uint16_t bits = reinterpret_cast<const uint16_t*>(lds_p + (step * RT + rt) * 64 + (slot & ~7) * 2 + n)[place];
              weight[rt] = DT == MEGA_BF16 ? bf16_bits_to_float(bits) : f16_bits_to_float(bits);
              its[rt] = sees(lds_sees[rt * 16 + n], key);
            }
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int at = min(first_column + 16 * kCols * (c / kCols) + kCols * (4 * h + i) + c % kCols, a.v.width - 1);
                float v;
                if constexpr (kEight) {
                  v = (row[at] & 0x7f) == 0x7f ? __builtin_nanf("") : 0.f;
                } else {
                  const uint16_t bits = reinterpret_cast<const uint16_t*>(row)[at];
                  v = DT == MEGA_BF16 ? bf16_bits_to_float(bits) : f16_bits_to_float(bits);
                }
                const bool finite = fabsf(v) < __builtin_inff();
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) acc[rt][c][i] = finite || !its[rt] ? acc[rt][c][i] : fmaf(weight[rt], v, acc[rt][c][i]);
                __builtin_amdgcn_sched_barrier(0);
              }
          }
        }
      if constexpr (kNext) there[0] = next.there[0], there[1] = next.there[1];
    };

    for (int tile = begin; tile < end; tile += 32 * waves) {
      // ---- scores of the wave's 32 keys
      const int mine = tile + 32 * wave;
      if (!kAcross) load_first_keys(tile);
      f32x4 s[2][RT];
      bool pages_there = true;
      if (mine < end) {
        const bool whole = mine >= all_low && mine + 31 <= all_high;
        Keys now = keys_at(mine);
        const Keys second = keys_at(mine + 16);
        pages_there = now.there && second.there;
        u32x4 q[RT], q_next[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) q_next[rt] = __builtin_bit_cast(u32x4, lds_q[rt * KS * 64 + lane]);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          f32x4 factor = {a.scale, a.scale, a.scale, a.scale};
          if constexpr (kEight) {
#pragma unroll
            for (int i = 0; i < 4; ++i) factor[i] *= exponent_value(ke[i]);
            if (half == 0) load_key_exponents(second);
          }
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) s[half][rt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < KS; ++c) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {  // (the rows' operands one step ahead; fences keep it at that)
              q[rt] = q_next[rt];
              if (half == 0 || c + 1 < KS) q_next[rt] = __builtin_bit_cast(u32x4, lds_q[(rt * KS + (c + 1) % KS) * 64 + lane]);
            }
            u32x4 key;
            if constexpr (kEight) {
              const u32x4 w = kx[c >> 1];
              const uint32_t lo = (c & 1) ? w[2] : w[0], hi = (c & 1) ? w[3] : w[1];
              key = u32x4{widen<DT, false>(lo, 1.f), widen<DT, true>(lo, 1.f), widen<DT, false>(hi, 1.f), widen<DT, true>(hi, 1.f)};
            } else {
              key = kx[c];
            }
            if (a.k.width != 32 * KS) {  // (behind the row's end the rows' operands are zero, and infinity times zero is not)
              const int d = kEight ? (c >> 1) * 64 + (opaque(lane) >> 4) * 16 : c * 32 + (opaque(lane) >> 4) * 8;
              if (d >= a.k.width) key = u32x4{0, 0, 0, 0};
            }
            if (half == 0 && (!kEight || (c & 1))) load_key(second, kEight ? c >> 1 : c);  // into the registers that have become free
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) s[half][rt] = mma<DT>(key, q[rt], s[half][rt]);
            __builtin_amdgcn_sched_barrier(0);
          }
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) s[half][rt] *= factor;
          const bool there = half ? second.there : now.there;
          if (!whole || !there) {
            const int l = opaque(lane), first = mine + 16 * half + 4 * (l >> 4);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
              const int2 range = lds_sees[rt * 16 + (l & 15)];
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (!there || !sees(range, first + i)) s[half][rt][i] = -__builtin_inff();
            }
          }
        }
      } else {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s[0][rt] = s[1][rt] = f32x4{-__builtin_inff(), -__builtin_inff(), -__builtin_inff(), -__builtin_inff()};
      }
      if (!kAcross) load_step(tile);
      if (kAcross) load_first_keys(tile + 32 * waves);

      // ---- the rows' new maxima
      float top[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        float t = fmaxf(fmaxf(s[0][rt][0], s[0][rt][1]), fmaxf(s[0][rt][2], s[0][rt][3]));
        t = fmaxf(t, fmaxf(fmaxf(s[1][rt][0], s[1][rt][1]), fmaxf(s[1][rt][2], s[1][rt][3])));
        t = fmaxf(t, across(t, 16));
        top[rt] = fmaxf(t, across(t, 32));
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
      // (m follows the maximum when that is 2^8 above it, not at each step: the factor leaves p, l and o alike, and a probability
      // of up to 2^8 is as exact as one of up to 1)
      bool moved = false;
      float alpha[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const float now = top[rt] > m[rt] + 8.f ? top[rt] : m[rt], base = now == -__builtin_inff() ? 0.f : now;
        alpha[rt] = __builtin_amdgcn_exp2f(m[rt] - base);
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
      const bool some = pages_there && tile >= all_low;
      if (some) {
        const int all = min(steps, (all_high + 1 - tile) >> 5);
        for (; step < (kAcross ? all : min(all, steps - 1)); ++step) values_of(tile, step, std::true_type(), std::true_type());
        if (!kAcross && step < all) values_of(tile, step++, std::true_type(), std::false_type());
      }
      for (; step < steps; ++step) values_of(tile, step, std::false_type(), std::true_type());
    }

    // ---- the rows' sums over the lanes and waves that had their keys
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      l[rt] += across(l[rt], 16);
      l[rt] += across(l[rt], 32);
    }
    if (waves > 1) {
      __syncthreads();  // (the maxima of the last tile have been read)
      if (h == 0)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) lds_m[(rt * 16 + n) * 8 + wave] = l[rt];
      __syncthreads();
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        l[rt] = 0.f;
        for (int w = 0; w < waves; ++w) l[rt] += lds_m[(rt * 16 + n) * 8 + w];
      }
    }
    const int l_ = opaque(lane), n_ = l_ & 15, h_ = l_ >> 4;
    bool alone = true, last = true;
    int64_t slot = 0;
    int pieces = 0;
    if (a.parts > 0) {
      slot = (static_cast<int64_t>(head) * a.slots + id + progress.mark.blocks_before + progress.number) * a.part_rows;
      alone = progress.alone, pieces = progress.pieces, last = progress.unit >= progress.unit_end;
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int row = rt * 16 + n_;
      if (row >= k.count) continue;
      const int r = k.row0 + row, t = r / a.shared, g = r - t * a.shared;
      const int64_t at = (static_cast<int64_t>(k.start) + t) * (a.heads * a.shared) + head * a.shared + g;
      const float inverse = l[rt] == 0.f ? 0.f : 1.f / l[rt];
      if (a.parts > 0 && slab == 0 && wave == 0 && h_ == 0) {
        if (!alone) *reinterpret_cast<float2*>(a.stats + (slot + row) * 2) = make_float2(m[rt], l[rt]);
        // (places are 32-bit numbers: the host sees to that)
        if (pieces > 0) a.joins[at] = make_int2(static_cast<int>(slot + row), alone ? 0 : pieces);
      }
#pragma unroll
      for (int cg = 0; cg < kGroups; ++cg)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // accumulator element i of column operand j is column kCols (4 h + i) + j of the group
          const int c = first_column + 16 * kCols * cg + kCols * (4 * h_ + i);
          if (c >= a.v.width) continue;
          float o[kCols];
#pragma unroll
          for (int j = 0; j < kCols; ++j) o[j] = acc[rt][kCols * cg + j][i];
          if (!alone) {
            float4* to = reinterpret_cast<float4*>(a.part + (slot + row) * a.v.width + c);
#pragma unroll
            for (int j = 0; j < kCols / 4; ++j) to[j] = make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
          } else {
#pragma unroll
            for (int j = 0; j < kCols; ++j) o[j] = l[rt] == 0.f ? 0.f : o[j] * inverse;
            uint32_t* to = reinterpret_cast<uint32_t*>(a.out + at * a.v.width + c);
            if constexpr (kCols == 8)
              *reinterpret_cast<uint4*>(to) = make_uint4(pack2<DT>(o[0], o[1]), pack2<DT>(o[2], o[3]), pack2<DT>(o[4], o[5]), pack2<DT>(o[6], o[7]));
            else
              *reinterpret_cast<uint2*>(to) = make_uint2(pack2<DT>(o[0], o[1]), pack2<DT>(o[2], o[3]));
          }
        }
    }
    if (last) break;
    __syncthreads();  // (the rows, maxima and probabilities of this piece have been read)
  }
}

// Joins the pieces of the blocks that several workgroups had: o = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i with
// m = max_i m_i.  A group of 2^lanes_log2 lanes, eight columns each, takes every n-th piece of a row, n groups to a wave, in the
// pieces' order; the groups meet through the lanes.  Bound by the latency of three dependent loads where there are few rows, by the pieces' bytes else.
constexpr int kJoinThreads = 256;
template <int DT>
__global__ __launch_bounds__(kJoinThreads) void paged_join_kernel(AttnArgs a, int lanes_log2, uint32_t strips) {
  const int lane = static_cast<int>(threadIdx.x) & 63, lanes = 1 << lanes_log2, groups = 64 >> lanes_log2;
  const uint32_t item = blockIdx.x * (kJoinThreads / kWave) + (threadIdx.x >> 6), row = item / strips;
  const int64_t q_heads = a.heads * a.shared, all = a.clear_rest ? a.rows : row_bound(a.cu, a.view.batch, a.rows);
  if (row >= all * q_heads) return;
  const int2 join = a.joins[row];
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
  if (join.y <= 0) return;
  float now = m;
  for (int off = lanes; off < 64; off <<= 1) now = fmaxf(now, across(now, off));
  const float with = __builtin_amdgcn_exp2f(m - (now == -__builtin_inff() ? 0.f : now));
  l *= with;
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j] *= with;
  for (int off = lanes; off < 64; off <<= 1) {
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
  int join_lanes_log2;  // of the join: lanes to a row's strip
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
  if (c->batch > 0 && full < 4 * resident && p.blocks * (c->table_width * c->page_size / 32 + 1) < 0x40000000 &&
      (resident + p.blocks) * c->heads * kRows < 0x40000000 && rows * q_heads < 0x1000000) {
    p.parts = std::max<int64_t>(1, resident / pairs);
    p.part_rows = std::min(kRows, rows * shared);
    p.slots = p.parts + p.blocks;
    // the join: as many pieces of a row at a time as it has on average
    const int64_t pieces = p.parts * pairs / std::max<int64_t>(full, 1);
    p.join_lanes_log2 = pieces > 8 ? 2 : pieces > 4 ? 3 : pieces > 2 ? 4 : 5;
    while (p.join_lanes_log2 > 1 && (8 << (p.join_lanes_log2 - 1)) >= c->v_width) --p.join_lanes_log2;
  }
  return p;
}

template <int DT, bool kEight, int RT, int CT, int KS>
int launch_attn(const AttnArgs& a, const Plan& p, void* stream) {
  const auto kernel = paged_attn_kernel<DT, kEight, RT, CT, KS>;
  const size_t bytes = (RT * KS * 64 + p.waves * RT * 64) * sizeof(uint4) + RT * 16 * 8 * sizeof(float) + kMaxWaves * sizeof(int) + RT * 16 * sizeof(int2);
  if (bytes > 65536)
    MEGA_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)));
  hipStream_t s = static_cast<hipStream_t>(stream);
  kernel<<<dim3(static_cast<uint32_t>(p.workgroups(a.heads))), dim3(p.waves * kWave), bytes, s>>>(a);
  MEGA_CHECK_LAUNCH();
  if (p.parts > 0) {
    const int64_t strip = 8 << p.join_lanes_log2, strips = (a.v.width + strip - 1) / strip, waves = static_cast<int64_t>(a.rows) * a.heads * a.shared * strips;
    paged_join_kernel<DT><<<dim3(static_cast<uint32_t>((waves + kJoinThreads / kWave - 1) / (kJoinThreads / kWave))), dim3(kJoinThreads), 0, s>>>(
        a, p.join_lanes_log2, static_cast<uint32_t>(strips));
    MEGA_CHECK_LAUNCH();
  }
  return MEGA_OK;
}

template <int DT, bool kEight, int KS>
int launch_rows(const AttnArgs& a, const Plan& p, void* stream) {
  if (p.rt == 1 && p.ct == 16) return launch_attn<DT, kEight, 1, 16, KS>(a, p, stream);
  if (p.rt == 1) return launch_attn<DT, kEight, 1, 8, KS>(a, p, stream);
  if constexpr (KS < 16)
    if (p.rt == 4) return launch_attn<DT, kEight, 4, 8, KS>(a, p, stream);
  return launch_attn<DT, kEight, 2, 8, KS>(a, p, stream);
}

template <int DT, bool kEight>
int launch_width(const AttnArgs& a, const Plan& p, void* stream) {
  if (p.ks == 4) return launch_rows<DT, kEight, 4>(a, p, stream);
  if (p.ks == 8) return launch_rows<DT, kEight, 8>(a, p, stream);
  return launch_rows<DT, kEight, 16>(a, p, stream);
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
  a.scale = static_cast<float>(scale * 1.4426950408889634);
  const bool eight = cache->k_exponents != nullptr;
  if (dtype == MEGA_BF16) return eight ? launch_width<MEGA_BF16, true>(a, p, stream) : launch_width<MEGA_BF16, false>(a, p, stream);
  return eight ? launch_width<MEGA_F16, true>(a, p, stream) : launch_width<MEGA_F16, false>(a, p, stream);
}
