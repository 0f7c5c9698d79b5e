// What the kernels of the paged attention share: their arguments, the way from a workgroup to its rows and keys, the rows'
// way into LDS and the results' way out.
#pragma once

#include "paged.hpp"

namespace mega {

constexpr int kMaxWaves = 8;
constexpr int kMaxKeyWidth = 512;
constexpr int kCus = 256;
// A row's m stays until a score is more than 2^kSlack times above it: probabilities up to 2^kSlack are as exact as those up to 1, and the
// factor leaves p, l and o alike.  In float16 they are lifted further, to 2^15 at the most: below 2^-14 its numbers thin out, and many
// small probabilities of a long sequence weigh as much as a large one.
constexpr float kSlack = 8.f;
template <int DT>
constexpr float kLift = DT == MEGA_F16 ? 7.f : 0.f;

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
  int32_t lead;               // units in front of a block's own on the line
  int32_t clear_rest;
  int32_t chunk_shift, shared_shift;  // their logarithms where they are powers of two, else -1: a division is thirty instructions in a row
  float scale;                // |scale| log2(e), above zero: a negative scale turns the rows' signs (sign: their bits)
  uint32_t sign;
  double per_part;            // 1 / parts
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

__device__ __forceinline__ int chunk_start(const AttnArgs& a, int position) {
  if (a.chunk == 0 || position <= 0) return 0;
  return a.chunk_shift >= 0 ? position >> a.chunk_shift << a.chunk_shift : position / a.chunk * a.chunk;
}
// the new token of row r (token * shared + head)
__device__ __forceinline__ int token_of(const AttnArgs& a, int r) { return a.shared_shift >= 0 ? r >> a.shared_shift : r / a.shared; }

// A number of `cu` or `lengths`: kUniform: at an index that the wave has in common.
template <bool kUniform>
__device__ __forceinline__ int number_at(const int32_t* p, int i) {
  if constexpr (kUniform) return constant_at(p, i);
  return p[i];
}
template <bool kUniform>
__device__ __forceinline__ int bound_at(const AttnArgs& a, int i) { return min(max(number_at<kUniform>(a.cu, i), 0), a.rows); }

// Sequences, the rows behind the last one counted as one more where they are to be cleared.
__device__ __forceinline__ int sequences_of(const AttnArgs& a) { return a.view.batch + (a.clear_rest ? 1 : 0); }

// A sequence (the rows behind the last one are one more, without keys): its first packed row, new rows and positions.
struct Sequence {
  int32_t start, count, length;
};
template <bool kUniform>
__device__ __forceinline__ Sequence sequence_of(const AttnArgs& a, int b) {
  const bool rest = b >= a.view.batch;
  const int start = bound_at<kUniform>(a, b), end = rest ? a.rows : bound_at<kUniform>(a, b + 1);
  return {start, max(end - start, 0), rest ? 0 : max(number_at<kUniform>(a.lengths, b), 0)};
}
template <int kRows>
__device__ __forceinline__ int blocks_of(const AttnArgs& a, const Sequence& s) {
  return static_cast<int>((static_cast<int64_t>(s.count) * a.shared + kRows - 1) / kRows);
}
// Row block `number` of sequence b; false: it has no such block.
template <int kRows>
__device__ __forceinline__ bool block_of(const AttnArgs& a, const Sequence& s, int b, int64_t number, Block& k) {
  k.sequence = b;
  k.start = s.start;
  const int64_t row0 = number * kRows, rows = static_cast<int64_t>(s.count) * a.shared;
  if (row0 < 0 || row0 >= rows) return false;
  k.row0 = static_cast<int32_t>(row0);
  k.count = static_cast<int32_t>(min(static_cast<int64_t>(kRows), rows - row0));
  k.keys = static_cast<int32_t>(min(static_cast<int64_t>(s.length), static_cast<int64_t>(a.view.table_width) << a.view.page_shift));
  k.position0 = s.length - s.count;
  k.begin = chunk_start(a, k.position0 + token_of(a, k.row0));
  k.end = min(k.position0 + token_of(a, k.row0 + k.count - 1) + 1, k.keys);
  return true;
}

// A workgroup a block: blocks are numbered so that sequence b's begin at cu[b] shared / kRows + b, which leaves ceil(n shared / kRows)
// numbers before the next sequence's whatever the lengths are, and the host need not know these.
template <int kRows>
__device__ __forceinline__ bool find_block(const AttnArgs& a, int number, Block& k) {
  const int sequences = sequences_of(a);
  const auto first = [&](int b) { return static_cast<int64_t>(bound_at<false>(a, b)) * a.shared / kRows + b; };
  const int b = last_not_above(sequences, number, first);
  return block_of<kRows>(a, sequence_of<true>(a, b), b, number - (static_cast<int64_t>(bound_at<true>(a, b)) * a.shared / kRows + b), k);
}

// The line of units: a block has one for every 32 keys that it sees, and one if there are none, behind a.lead units for what a piece costs
// whatever its length (its rows' way in, its results' way out).  Only the units behind these are anybody's: a part that ends in a block's
// lead has nothing of the block, one that begins there has it from its first key.
__device__ __forceinline__ int units_of(const Block& k) { return max(k.end - (k.begin & ~31) + 31, 32) >> 5; }
// A place on the line: a block (its sequence, its number there), its units, and the blocks and units in front of it.
struct Mark {
  int32_t sequence, number, blocks, units;  // blocks: of the sequence; units: with the lead
  int32_t blocks_before, units_before, total;  // total: of the whole line (the host cuts no line of 2^30 units)
};
// units of a part; the parts behind the line's end are empty.  (The quotient in double is right: it is half a part away from the next one.)
__device__ __forceinline__ int part_units(const AttnArgs& a, int total) { return static_cast<int>((total + a.parts - 0.5) * a.per_part); }

// Inclusive sums over the lanes, in steps that stay in the vector unit (every lane has to be there).
template <int kControl, int kRowMask>
__device__ __forceinline__ int plus_moved(int v) { return v + __builtin_amdgcn_update_dpp(0, v, kControl, kRowMask, 0xf, false); }
__device__ __forceinline__ int sums_before_and_here(int v) {
  v = plus_moved<0x111, 0xf>(v);  // one, two, four, eight lanes up inside the rows of 16
  v = plus_moved<0x112, 0xf>(v);
  v = plus_moved<0x114, 0xf>(v);
  v = plus_moved<0x118, 0xf>(v);
  v = plus_moved<0x142, 0xa>(v);  // the last lane of rows 0 and 2 to rows 1 and 3, then lane 31 to rows 2 and 3
  return plus_moved<0x143, 0xc>(v);
}
// The units of the 64 blocks of a sequence from `number` on, one to a lane
template <int kRows>
__device__ __forceinline__ int lane_units(const AttnArgs& a, int b, int number, int blocks) {
  Block k;
  const int i = number + (static_cast<int>(threadIdx.x) & 63);
  const bool has = block_of<kRows>(a, sequence_of<true>(a, b), b, i, k);
  return i < blocks && has ? units_of(k) + a.lead : 0;
}

// The block in which part `part` begins (false: the part is empty); all lanes of a wave together, 64 sequences a round, and 64 blocks of a
// sequence that has more than one.
template <int kRows>
__device__ __forceinline__ bool find_mark(const AttnArgs& a, int part, Mark& mark, Block& block) {
  const int lane = static_cast<int>(threadIdx.x) & 63, sequences = sequences_of(a);
  int blocks = 0, units = 0, units_here = 0, blocks_here = 0;  // of the lane's sequence; inclusive sums
  Block k;                                                     // its first block
  const auto round = [&](int b0) {
    const int b = min(b0 + lane, sequences - 1);
    const Sequence q = sequence_of<false>(a, b);
    const bool has = block_of<kRows>(a, q, b, 0, k) && b0 + lane < sequences;
    blocks = has ? blocks_of<kRows>(a, q) : 0, units = has ? units_of(k) + a.lead : 0;
    for (uint64_t more = __ballot(blocks > 1); more != 0; more &= more - 1) {
      const int l = __ffsll(static_cast<unsigned long long>(more)) - 1, count = __builtin_amdgcn_readlane(blocks, l);
      int sum = 0;
      for (int i = 0; i < count; i += 64) sum += lane_units<kRows>(a, b0 + l, i, count);
      sum = __builtin_amdgcn_readlane(sums_before_and_here(sum), 63);
      if (lane == l) units = sum;
    }
    units_here = sums_before_and_here(units), blocks_here = sums_before_and_here(blocks);
  };
  mark.total = 0;
  for (int b0 = 0; b0 < sequences; b0 += 64) {
    round(b0);
    mark.total += __builtin_amdgcn_readlane(units_here, 63);
  }
  const int first = part * part_units(a, mark.total);
  if (first >= mark.total) return false;
  int units_before = 0, blocks_before = 0;
  for (int b0 = 0; b0 < sequences; b0 += 64) {
    if (sequences > 64) round(b0);
    const uint64_t which = __ballot(units_before + units_here > first);
    if (which != 0) {
      const int l = __ffsll(static_cast<unsigned long long>(which)) - 1;
      mark.sequence = b0 + l;
      mark.blocks = __builtin_amdgcn_readlane(blocks, l);
      mark.units_before = units_before + __builtin_amdgcn_readlane(units_here - units, l);
      mark.blocks_before = blocks_before + __builtin_amdgcn_readlane(blocks_here - blocks, l);
      mark.number = 0, mark.units = __builtin_amdgcn_readlane(units, l);
      if (mark.blocks == 1) {
        block = {mark.sequence, __builtin_amdgcn_readlane(k.start, l), __builtin_amdgcn_readlane(k.row0, l), __builtin_amdgcn_readlane(k.count, l),
                 __builtin_amdgcn_readlane(k.position0, l), __builtin_amdgcn_readlane(k.keys, l), __builtin_amdgcn_readlane(k.begin, l), __builtin_amdgcn_readlane(k.end, l)};
        return true;
      }
      for (int i = 0; i < mark.blocks; i += 64) {
        const int own = lane_units<kRows>(a, mark.sequence, i, mark.blocks), here = sums_before_and_here(own);
        const uint64_t found = __ballot(mark.units_before + here > first);
        if (found != 0) {
          const int f = __ffsll(static_cast<unsigned long long>(found)) - 1;
          mark.number = i + f, mark.units = __builtin_amdgcn_readlane(own, f);
          mark.units_before += __builtin_amdgcn_readlane(here - own, f);
          mark.blocks_before += mark.number;
          block_of<kRows>(a, sequence_of<true>(a, mark.sequence), mark.sequence, mark.number, block);
          return true;
        }
        mark.units_before += __builtin_amdgcn_readlane(here, 63);
      }
    }
    units_before += __builtin_amdgcn_readlane(units_here, 63);
    blocks_before += __builtin_amdgcn_readlane(blocks_here, 63);
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

// ones over those bytes of a word whose e4m3 codes times `unit` are finite numbers of the type
template <int DT>
__device__ __forceinline__ uint32_t finite_codes(uint32_t w, float unit) {
  const uint32_t low = finite_halves<DT>(widen<DT, false>(w, unit)), high = finite_halves<DT>(widen<DT, true>(w, unit));
  return __builtin_amdgcn_perm(high, low, 0x06040200);
}

// v, of which the compiler knows nothing: what is computed from it is computed where it is used, not once ahead of a loop
// and kept in registers that the loop has no room for
__device__ __forceinline__ int opaque(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

__device__ __forceinline__ float across(float v, int mask) { return __shfl_xor(v, mask, 64); }
// v's maximum and sum over the four lanes n, n + 16, n + 32, n + 48, in all of them: the swapping moves leave both halves in each place
__device__ __forceinline__ float four_max(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(t[0]), __uint_as_float(t[1]));
}
__device__ __forceinline__ float four_sum(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(t[0]) + __uint_as_float(t[1]);
}

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

// One request: lane l's 16 bytes at base + offset go to LDS bytes lds_dst + 16 l .. + 15 (lds_dst in M0, a wave's own).  Assembly, so that the
// compiler does not see a vector memory instruction that writes LDS and wait for every request in flight in front of each LDS read; the wait for
// these requests is explicit, the s_nop the wait state between a scalar write of M0 and a load to LDS.
__device__ __forceinline__ void load_to_lds16(const void* base, uint32_t offset, uint32_t lds_dst) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(offset), "s"(base), "s"(lds_dst) : "memory");
}
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const char*)(p)));
}

// Where a workgroup is on the line of units, kept in LDS while it works on a piece.
struct Progress {
  Mark mark;
  int32_t unit, unit_end, per, part;
  int32_t pieces;  // of the block, this one included if it is the first; 0 for the others
  bool alone;      // the whole block is this workgroup's
};

// The first row block of a workgroup, and its place on the line of units; false: it has none.
template <int kRows>
__device__ __forceinline__ bool first_piece(const AttnArgs& a, int id, Progress& at, Block& k) {
  if (a.parts == 0) return find_block<kRows>(a, a.blocks - 1 - id, k);
  // One sequence whose blocks see much the same number of keys (the first three quarters of the last one's): as many equal pieces of each block as
  // there are parts for, so that nobody has two.  512 tokens behind 1531: 57 us, 64 on the line; behind 256, where the first block sees 40 %:
  // 46.4, 45.5 on the line; behind 1024 (70 %): 53, 60 on the line
  if (a.view.batch == 1) {
    const Sequence s = sequence_of<true>(a, 0);
    const int blocks = blocks_of<kRows>(a, s);
    if (s.start == 0 && (s.count == a.rows || !a.clear_rest) && blocks > 0 && blocks <= a.parts) {
      Block first;
      block_of<kRows>(a, s, 0, 0, first);
      block_of<kRows>(a, s, 0, blocks - 1, k);
      if (units_of(first) * 4 >= units_of(k) * 3) {
        const int each = a.parts / blocks, number = id / each, piece = id - number * each;
        if (!block_of<kRows>(a, s, 0, number, k)) return false;
        const int units = units_of(k);
        at.per = (units + each - 1) / each, at.part = piece;
        at.unit = piece * at.per, at.unit_end = min(at.unit + at.per, units);
        at.mark = {0, number, blocks, units + a.lead, 0, -a.lead, units};
        return at.unit < units;
      }
    }
  }
  if (!find_mark<kRows>(a, id, at.mark, k)) return false;
  at.part = id;
  at.per = part_units(a, at.mark.total);
  at.unit = id * at.per, at.unit_end = min(at.unit + at.per, at.mark.total);
  // (the part's first block may be one that it has nothing of)
  return at.unit_end > at.mark.units_before + a.lead;
}
// Which of block k's keys the workgroup has, [begin, end), begin a multiple of 32; its progress goes to LDS.
template <int kRows>
__device__ __forceinline__ void take_piece(const AttnArgs& a, Progress at, Progress& progress, const Block& k, int& begin, int& end) {
  if (a.parts == 0) {
    begin = k.begin & ~31, end = k.end;
    return;
  }
  const int units = at.mark.units - a.lead, first = at.mark.units_before + a.lead, last = min(first + units, at.unit_end);
  at.unit = max(at.unit, first);
  begin = __builtin_amdgcn_readfirstlane((k.begin & ~31) + (at.unit - first) * 32);
  end = __builtin_amdgcn_readfirstlane(min((k.begin & ~31) + (last - first) * 32, k.end));
  const int part_end = (at.part + 1) * at.per;
  const bool begins_here = first >= part_end - at.per;  // (and in front of the part's end)
  at.alone = begins_here && first + units <= part_end;
  at.pieces = !begins_here ? 0 : at.alone ? 1 : 1 + (first + units - part_end + at.per - 1) / at.per;
  at.unit = last;
  if (threadIdx.x == 0) progress = at;
}
// On to the next block (there is one): behind a piece, in front of a barrier.
template <int kRows>
__device__ __forceinline__ Progress next_piece(const AttnArgs& a, const Progress& progress, Block& k) {
  const auto in_common = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
  Progress at{};
  if (a.parts == 0) return at;  // (a workgroup a block: not reached)
  const Mark& m = progress.mark;
  at.mark = {in_common(m.sequence), in_common(m.number) + 1, in_common(m.blocks), 0, in_common(m.blocks_before) + 1, in_common(m.units_before) + in_common(m.units), 0};
  at.unit = in_common(progress.unit), at.unit_end = in_common(progress.unit_end), at.per = in_common(progress.per), at.part = in_common(progress.part);
  Sequence s = sequence_of<true>(a, at.mark.sequence);
  if (at.mark.number == at.mark.blocks) {
    do s = sequence_of<true>(a, ++at.mark.sequence);
    while (s.count == 0 && at.mark.sequence + 1 < sequences_of(a));
    at.mark.blocks = blocks_of<kRows>(a, s), at.mark.number = 0;
  }
  block_of<kRows>(a, s, at.mark.sequence, at.mark.number, k);
  at.mark.units = units_of(k) + a.lead;
  return at;
}

// The block's rows to LDS, [row tile][step][lane]: the order in which the matrix instructions take them, zeros behind the rows' end and in
// rows that there are not.  Eight elements at a time: a row's are 4 KS pieces.
template <int KS>
__device__ __forceinline__ uint4 row_piece(const AttnArgs& a, const Block& k, int head, int c) {
  const int row = c / (KS * 4), d = c % (KS * 4);
  if (row >= k.count || d * 8 >= a.k.width) return make_uint4(0, 0, 0, 0);
  const int r = k.row0 + row, t = token_of(a, r), g = r - t * a.shared;
  uint4 x = *reinterpret_cast<const uint4*>(a.q + (static_cast<int64_t>(k.start) + t) * a.q_row + (static_cast<int64_t>(head) * a.shared + g) * a.q_head + d * 8);
  x.x ^= a.sign, x.y ^= a.sign, x.z ^= a.sign, x.w ^= a.sign;
  return x;
}
template <bool kEight, int KS>
__device__ __forceinline__ void row_piece_to_lds(uint4 x, int c, uint4* lds_q) {
  // (8-bit keys: a lane reads 16 codes at a time, which serve two steps)
  const int row = c / (KS * 4), d = c % (KS * 4);
  const int step = kEight ? (d >> 3) * 2 + (d & 1) : d >> 2, quarter = kEight ? (d >> 1) & 3 : d & 3;
  lds_q[((row >> 4) * KS + step) * 64 + quarter * 16 + (row & 15)] = x;
}

// The rows' visible keys of a piece to LDS: the first one and the number of further ones (none: a first one that no key reaches).
template <int kRows>
__device__ __forceinline__ void ranges_to_lds(const AttnArgs& a, const Block& k, int end, int2* lds_sees) {
  for (int row = threadIdx.x; row < kRows; row += blockDim.x) {
    const int position = k.position0 + token_of(a, k.row0 + row), low = chunk_start(a, position), high = min(position, end - 1);
    const bool none = row >= k.count || high < low;
    lds_sees[row] = none ? make_int2(0x7fffffff, 0) : make_int2(low, high - low);
  }
}
__device__ __forceinline__ bool in_range(int2 range, int key) { return static_cast<uint32_t>(key) - static_cast<uint32_t>(range.x) <= static_cast<uint32_t>(range.y); }

// Key by key, the infinities and NaN among 32 keys' values (from `first` on, slot 8 h + i as in paged_attention.hip) into the rows that see them; the
// product had zeros in their places.  An 8-bit value is what its code and exponent stand for in the rows' type, which may not hold it.
// weight(rt, slot): the bits of the probability of row rt * 16 + (lane & 15).
template <int DT, bool kEight, int kCols, int RT, int CT, typename Step, typename Weight>
__device__ __forceinline__ void add_odd_values(const AttnArgs& a, const Block& k, int end, int first, int first_column, const Step& t, const int2* lds_sees,
                                               Weight weight, f32x4 (&acc)[RT][CT]) {
  const auto number = [](uint32_t bits) { return DT == MEGA_BF16 ? bf16_bits_to_float(static_cast<uint16_t>(bits)) : f16_bits_to_float(static_cast<uint16_t>(bits)); };
#pragma unroll 1
  for (int slot = 0; slot < 32; ++slot) {
    const int l = opaque(static_cast<int>(threadIdx.x) & 63), n = l & 15, h = l >> 4;
    const int place = slot & 7, half = place >> 2, in_group = 4 * (slot >> 3) + (place & 3), key = first + 16 * half + in_group;
    if (key < k.begin || key >= end || !(half ? t.there[1] : t.there[0])) continue;
    const uint8_t* const row = (half ? t.from[1] : t.from[0]) + static_cast<int64_t>(in_group) * a.v.slot * (kEight ? 1 : 2);
    float unit = 0.f;
    if constexpr (kEight) unit = exponent_value((half ? t.exponents[1] : t.exponents[0])[static_cast<int64_t>(in_group) * a.v.eSlot]);
    float p[RT];
    bool its[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      p[rt] = number(weight(rt, slot));
      its[rt] = in_range(lds_sees[rt * 16 + n], key);
    }
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = min(first_column + 16 * kCols * (c / kCols) + kCols * (4 * h + i) + c % kCols, a.v.width - 1);
        float v;
        if constexpr (kEight)
          v = number(widen<DT, false>(row[at], unit));
        else
          v = number(reinterpret_cast<const uint16_t*>(row)[at]);
        const bool finite = fabsf(v) < __builtin_inff();
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) acc[rt][c][i] = finite || !its[rt] ? acc[rt][c][i] : fmaf(p[rt], v, acc[rt][c][i]);
        __builtin_amdgcn_sched_barrier(0);
      }
  }
}

// The sum of the first `waves` of eight numbers in LDS.
__device__ __forceinline__ float sum_of_waves(const float* p, int waves) {
  const float4 u = *reinterpret_cast<const float4*>(p), v = *reinterpret_cast<const float4*>(p + 4);
  const float x[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
  float sum = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) sum += w < waves ? x[w] : 0.f;
  return sum;
}

// Where a piece's results go.
struct Destination {
  bool alone, last;  // to out, the block is this workgroup's; this was its last piece
  bool fits;
  int32_t pieces;
  int64_t slot;      // else: its first row in the workspace
};
__device__ __forceinline__ Destination destination_of(const AttnArgs& a, const Progress& progress, int id, int head) {
  if (a.parts == 0) return {true, true, true, 0, 0};
  const int number = id + progress.mark.blocks_before;  // (more blocks than there are rows for: cu decreases somewhere)
  return {progress.alone, progress.unit + a.lead >= progress.unit_end, number < a.slots, progress.pieces,
          (static_cast<int64_t>(head) * a.slots + number) * a.part_rows};
}
// A row's number in out and, with `note`, its m and l to the workspace and the number of its pieces.
__device__ __forceinline__ int64_t place_of_row(const AttnArgs& a, const Block& k, const Destination& to, int head, int row, bool note, float m, float l) {
  const int r = k.row0 + row, t = token_of(a, r), g = r - t * a.shared;
  const int64_t at = (static_cast<int64_t>(k.start) + t) * (a.heads * a.shared) + head * a.shared + g;
  if (note && a.parts > 0 && row < k.count) {
    if (!to.alone) *reinterpret_cast<float2*>(a.stats + (to.slot + row) * 2) = make_float2(m, l);
    // (places are 32-bit numbers: the host sees to that)
    if (to.pieces > 0) a.joins[at] = make_int2(static_cast<int>(to.slot + row), to.alone ? 0 : to.pieces);
  }
  return at;
}

// Blocks of more than 32 rows (paged_attention_rows.hip).
struct RowsPlan {
  int ks, waves;  // 32-wide steps of a key row, waves of a workgroup
  int64_t workgroups;
};
int launch_paged_rows(const AttnArgs& a, const RowsPlan& p, int dtype, bool eight, void* stream);

}  // namespace mega
