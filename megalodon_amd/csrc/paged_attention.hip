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
// Few rows (single tokens, drafts): bound by the cache's bytes.  The key range of a row block is cut into equal runs
// until the launch fills the chip; their (o, m, l) go to a workspace in float32 and a second kernel joins them.
// Many rows: bound by the matrix cores and by what L2 gives for the operands.
#include "paged.hpp"

#include <algorithm>

namespace mega {
namespace {

constexpr int kMaxWaves = 8;
constexpr int kMaxKeyWidth = 512;
constexpr int kMaxRuns = 64;

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
  float *part, *stats;        // runs > 1: (runs, rows, q_heads, v_width), (runs, rows, q_heads, 2)
  int32_t rows, heads, shared, chunk, runs, slabs, blocks;
  int32_t clear_rest;
  float scale;                // times log2(e)
};

// A row block of one sequence and the keys that any of its rows sees.
struct Block {
  int32_t start, row0, count;  // first packed row of the sequence; first row (token * shared + head) and their number
  int32_t position0;           // position of the sequence's first new token
  int32_t keys;                // positions that have a place
  int32_t begin, end;          // keys that the block sees, [begin, end)
  int32_t sequence;
};

__device__ __forceinline__ int chunk_start(int position, int chunk) { return chunk > 0 && position > 0 ? position / chunk * chunk : 0; }

// Row blocks are numbered so that sequence b's begin at cu[b] shared / kRows + b: enough for ceil(n shared / kRows) of them
// before the next sequence's, whatever the lengths, and the host need not know these.  (`rest`: rows behind the last
// sequence form one more, which has no keys.)
template <int kRows>
__device__ __forceinline__ bool find_block(const AttnArgs& a, int number, Block& k) {
  const int32_t* cu = a.cu;
  const int sequences = a.view.batch + (a.clear_rest ? 1 : 0);
  if (sequences == 0) return false;
  const auto first = [&](int b) { return static_cast<int64_t>(row_bound(cu, b, a.rows)) * a.shared / kRows + b; };
  const int b = last_not_above(sequences, number, first);
  k.sequence = b;
  k.start = row_bound(cu, b, a.rows);
  const int n = (b < a.view.batch ? row_bound(cu, b + 1, a.rows) : a.rows) - k.start;
  const int64_t row0 = (number - first(b)) * kRows;
  if (row0 < 0 || row0 >= static_cast<int64_t>(n) * a.shared) return false;
  k.row0 = static_cast<int32_t>(row0);
  k.count = static_cast<int32_t>(min(static_cast<int64_t>(kRows), static_cast<int64_t>(n) * a.shared - row0));
  const int length = b < a.view.batch ? max(a.lengths[b], 0) : 0;
  k.keys = min(static_cast<int64_t>(length), static_cast<int64_t>(a.view.table_width) << a.view.page_shift);
  k.position0 = length - n;
  k.begin = chunk_start(k.position0 + k.row0 / a.shared, a.chunk);
  k.end = min(k.position0 + (k.row0 + k.count - 1) / a.shared + 1, k.keys);
  return true;
}

// Run `i` of a block's keys: [begin, end), begin a multiple of 32; empty where there are fewer runs.
__device__ __forceinline__ int run_length(const Block& k, int runs) {
  const int groups = (k.end - (k.begin & ~31) + 31) >> 5;
  return max((groups + runs - 1) / runs, 1) * 32;
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

// whether one of a word's two 16-bit numbers is infinite or NaN
template <int DT>
__device__ __forceinline__ bool not_finite(uint32_t w) {
  constexpr uint32_t top = DT == MEGA_BF16 ? 0x7f80u : 0x7c00u;
  return (w & top) == top || ((w >> 16) & top) == top;
}

__device__ __forceinline__ float across(float v, int mask) { return __shfl_xor(v, mask, 64); }

// The page of 16 keys: its number and whether there is one (0 otherwise, so that addresses stay in the pool).
struct Page {
  uint32_t number;
  bool there;
};
__device__ __forceinline__ Page page_of(const AttnArgs& a, int sequence, int key) {
  const uint32_t e = static_cast<uint32_t>(a.view.table[sequence * a.view.table_stride + (key >> a.view.page_shift)]);
  const bool there = e < static_cast<uint32_t>(a.view.pages);
  return {there ? e : 0, there};
}

template <int DT, bool kEight, int RT, int CT, int KS>  // KS: 32-wide steps of a key row
__global__ __launch_bounds__(kMaxWaves * kWave, 2) void paged_attn_kernel(AttnArgs a) {
  constexpr int kRows = 16 * RT, kGroups = CT / 8;  // column groups of 128
  extern __shared__ __align__(16) uint4 lds[];
  const int lane = static_cast<int>(threadIdx.x) & 63, n = lane & 15, h = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6), waves = static_cast<int>(blockDim.x) >> 6;
  uint4* const lds_q = lds;                       // [RT][KS][64]
  uint4* const lds_p = lds + RT * KS * 64;        // [waves][RT][64]
  float* const lds_m = reinterpret_cast<float*>(lds_p + waves * RT * 64);  // [kRows][8]

  // column slab and head fastest: workgroups that read the same keys and values share an XCD's L2 (the hardware deals
  // workgroups to the eight XCDs in turn); late row blocks, which see the most keys, first
  uint32_t id = blockIdx.x;
  const int slab = id % a.slabs;
  id /= a.slabs;
  const int head = id % a.heads;
  id /= a.heads;
  const int run = id % a.runs;
  Block k;
  if (!find_block<kRows>(a, a.blocks - 1 - static_cast<int>(id / a.runs), k)) return;
  int begin = k.begin & ~31, end = k.end;
  if (a.runs > 1) {
    const int length = run_length(k, a.runs);
    begin += run * length;
    end = min(end, begin + length);
    if (begin >= end) return;  // (the join knows as many runs as there are)
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
  __syncthreads();

  int low[RT], high[RT];  // the lane's rows see keys low .. high
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int row = rt * 16 + n, position = k.position0 + (k.row0 + row) / a.shared;
    low[rt] = chunk_start(position, a.chunk);
    high[rt] = row < k.count ? min(position, k.keys - 1) : -1;
  }
  // keys all_low .. all_high are seen by every row of the block
  const int all_low = chunk_start(k.position0 + (k.row0 + k.count - 1) / a.shared, a.chunk), all_high = min(k.position0 + k.row0 / a.shared, k.keys - 1);

  f32x4 acc[RT][CT];
  float m[RT], l[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = -__builtin_inff(), l[rt] = 0.f;
#pragma unroll
    for (int c = 0; c < CT; ++c) acc[rt][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const int page_mask = (1 << a.view.page_shift) - 1;
  const int column = (slab * waves + wave) * CT * 16 + n * 8;  // + 128 g

  for (int tile = begin; tile < end; tile += 32 * waves) {
    // ---- scores of the wave's 32 keys
    const int mine = tile + 32 * wave;
    f32x4 s[2][RT];
    if (mine < end) {
      bool whole = mine >= all_low && mine + 31 <= all_high;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int group = mine + 16 * half, held = min(group, (end - 1) & ~15);
        const Page page = page_of(a, k.sequence, held);
        whole = whole && page.there;
        const int place = (held & page_mask) + n;
        u32x4 kx[KS];
        if constexpr (kEight) {
          const uint8_t* from = static_cast<const uint8_t*>(a.k.rows) + page.number * a.k.page + static_cast<int64_t>(head) * a.k.head;
          const uint32_t at = static_cast<uint32_t>(place) * a.k.slot + h * 16;
#pragma unroll
          for (int c = 0; c < KS / 2; ++c) {
            const int d = c * 64 + h * 16;
            const u32x4 x = d < a.k.width ? *reinterpret_cast<const u32x4*>(from + at + c * 64) : u32x4{0, 0, 0, 0};
            kx[2 * c] = u32x4{widen<DT, false>(x[0], 1.f), widen<DT, true>(x[0], 1.f), widen<DT, false>(x[1], 1.f), widen<DT, true>(x[1], 1.f)};
            kx[2 * c + 1] = u32x4{widen<DT, false>(x[2], 1.f), widen<DT, true>(x[2], 1.f), widen<DT, false>(x[3], 1.f), widen<DT, true>(x[3], 1.f)};
          }
        } else {
          const uint16_t* from = static_cast<const uint16_t*>(a.k.rows) + page.number * a.k.page + static_cast<int64_t>(head) * a.k.head;
          const uint32_t at = static_cast<uint32_t>(place) * a.k.slot + h * 8;
#pragma unroll
          for (int c = 0; c < KS; ++c)
            kx[c] = c * 32 + h * 8 < a.k.width ? *reinterpret_cast<const u32x4*>(from + at + c * 32) : u32x4{0, 0, 0, 0};
        }
        f32x4 factor = {a.scale, a.scale, a.scale, a.scale};
        if constexpr (kEight) {
          const uint8_t* e = a.k.exponents + page.number * a.k.ePage + static_cast<int64_t>(head) * a.k.eHead;
#pragma unroll
          for (int i = 0; i < 4; ++i) factor[i] *= exponent_value(e[static_cast<uint32_t>((held & page_mask) + 4 * h + i) * a.k.eSlot]);
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s[half][rt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < KS; ++c)
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) s[half][rt] = mma<DT>(kx[c], __builtin_bit_cast(u32x4, lds_q[(rt * KS + c) * 64 + lane]), s[half][rt]);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s[half][rt] *= factor;
        if (!whole) {
          const int first = group + 4 * h;
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (!page.there || first + i < low[rt] || first + i > high[rt] || first + i >= end) s[half][rt][i] = -__builtin_inff();
        }
      }
    } else {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) s[0][rt] = s[1][rt] = f32x4{-__builtin_inff(), -__builtin_inff(), -__builtin_inff(), -__builtin_inff()};
    }

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
      __syncthreads();
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
        for (int w = 0; w < waves; ++w) top[rt] = fmaxf(top[rt], lds_m[(rt * 16 + n) * 8 + w]);
    }

    // ---- probabilities, in the operand order of the second product
    bool moved = false;
    float alpha[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const float now = fmaxf(m[rt], top[rt]), base = now == -__builtin_inff() ? 0.f : now;
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
    }
    if (__any(moved))
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int c = 0; c < CT; ++c) acc[rt][c] *= alpha[rt];
    __syncthreads();

    // ---- values: 32 keys a step
    for (int step = 0; step < waves; ++step) {
      const int first = tile + 32 * step;
      if (first >= end) break;
      const int held[2] = {first, min(first + 16, (end - 1) & ~15)};
      const Page page[2] = {page_of(a, k.sequence, held[0]), page_of(a, k.sequence, held[1])};
      u32x4 vt[CT];
      const bool inside = first >= k.begin && first + 32 <= end && page[0].there && page[1].there;
      float unit[8];
      if constexpr (kEight) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint8_t* e = a.v.exponents + page[half].number * a.v.ePage + static_cast<int64_t>(head) * a.v.eHead;
#pragma unroll
          for (int i = 0; i < 4; ++i) unit[4 * half + i] = exponent_value(e[static_cast<uint32_t>((held[half] & page_mask) + 4 * h + i) * a.v.eSlot]);
        }
      }
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        const int c0 = min(column + 128 * g, a.v.width - 8);  // (columns behind the last are computed from others and not written)
        u32x4 x[8];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int64_t base = page[half].number * a.v.page + static_cast<int64_t>(head) * a.v.head;
          const uint32_t at = static_cast<uint32_t>((held[half] & page_mask) + 4 * h) * a.v.slot + c0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if constexpr (kEight) {
              const uint2 c = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.v.rows) + base + (at + static_cast<uint32_t>(i) * a.v.slot));
              const float u = unit[4 * half + i];
              x[4 * half + i] = u32x4{widen<DT, false>(c.x, u), widen<DT, true>(c.x, u), widen<DT, false>(c.y, u), widen<DT, true>(c.y, u)};
            } else {
              x[4 * half + i] = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.v.rows) + base + (at + static_cast<uint32_t>(i) * a.v.slot));
            }
          }
        }
        if (!inside)  // what is not there, or not this run's, must not meet a probability of zero as NaN
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int key = first + 16 * (i >> 2) + 4 * h + (i & 3);
            if (key < k.begin || key >= end || !page[i >> 2].there) x[i] = u32x4{0, 0, 0, 0};
          }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            vt[8 * g + 2 * j][i] = __builtin_amdgcn_perm(x[2 * i + 1][j], x[2 * i][j], 0x05040100);
            vt[8 * g + 2 * j + 1][i] = __builtin_amdgcn_perm(x[2 * i + 1][j], x[2 * i][j], 0x07060302);
          }
      }
      bool plain = first >= all_low && first + 31 <= all_high;
      if (!plain) {  // some row does not see some of these keys: harmless unless a value is infinite or NaN
        bool odd = false;
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) odd = odd || not_finite<DT>(vt[c][i]);
        plain = !__any(odd);
      }
      if (plain) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const u32x4 p = __builtin_bit_cast(u32x4, lds_p[(step * RT + rt) * 64 + lane]);
#pragma unroll
          for (int c = 0; c < CT; ++c) acc[rt][c] = mma<DT>(vt[c], p, acc[rt][c]);
        }
      } else {  // key by key, each into the rows that see it
#pragma unroll 1
        for (int slot = 0; slot < 32; ++slot) {
          const int e = slot & 7, key = first + 16 * (e >> 2) + 4 * (slot >> 3) + (e & 3);
          u32x4 keep;
#pragma unroll
          for (int i = 0; i < 4; ++i) keep[i] = h == slot >> 3 && i == e >> 1 ? ((e & 1) ? 0xffff0000u : 0x0000ffffu) : 0u;
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            const u32x4 p = __builtin_bit_cast(u32x4, lds_p[(step * RT + rt) * 64 + lane]);
            const bool sees = key >= low[rt] && key <= high[rt];
#pragma unroll
            for (int c = 0; c < CT; ++c) {
              const f32x4 with = mma<DT>(vt[c] & keep, p, acc[rt][c]);
#pragma unroll
              for (int i = 0; i < 4; ++i) acc[rt][c][i] = sees ? with[i] : acc[rt][c][i];
            }
          }
        }
      }
    }
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
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int row = rt * 16 + n;
    if (row >= k.count) continue;
    const int r = k.row0 + row, t = r / a.shared, g = r - t * a.shared;
    const int64_t at = (static_cast<int64_t>(k.start) + t) * (a.heads * a.shared) + head * a.shared + g;
    const int64_t all = static_cast<int64_t>(a.rows) * a.heads * a.shared;
    const float inverse = l[rt] == 0.f ? 0.f : 1.f / l[rt];
    if (a.runs > 1 && slab == 0 && wave == 0 && h == 0) {
      a.stats[(run * all + at) * 2] = m[rt];
      a.stats[(run * all + at) * 2 + 1] = l[rt];
    }
#pragma unroll
    for (int cg = 0; cg < kGroups; ++cg)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // accumulator element i of column operand j is column 8 (4 h + i) + j of the group
        const int c = (slab * waves + wave) * CT * 16 + 128 * cg + 8 * (4 * h + i);
        if (c >= a.v.width) continue;
        float o[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = acc[rt][8 * cg + j][i];
        if (a.runs > 1) {
          float4* to = reinterpret_cast<float4*>(a.part + (run * all + at) * a.v.width + c);
          to[0] = make_float4(o[0], o[1], o[2], o[3]);
          to[1] = make_float4(o[4], o[5], o[6], o[7]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) o[j] = l[rt] == 0.f ? 0.f : o[j] * inverse;
          *reinterpret_cast<uint4*>(a.out + at * a.v.width + c) = pack8<DT>(o);
        }
      }
  }
}

// Joins a row's runs: o = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i with m = max_i m_i.  A thread has eight columns of
// a row; the runs come in their order, whatever order they were made in.
constexpr int kJoinThreads = 256;
template <int DT, int kRows>
__global__ __launch_bounds__(kJoinThreads) void paged_join_kernel(AttnArgs a) {
  const int pieces = a.v.width / 8, q_heads = a.heads * a.shared;
  const int64_t all = static_cast<int64_t>(a.rows) * q_heads, items = all * pieces;
  const int64_t item0 = static_cast<int64_t>(blockIdx.x) * kJoinThreads + (threadIdx.x & ~63u), item = item0 + (threadIdx.x & 63u);
  if (item0 >= items) return;
  int b = last_not_above(a.view.batch + 1, item0 / pieces / q_heads, [&](int i) { return static_cast<int64_t>(row_bound(a.cu, i, a.rows)); });
  if (item >= items) return;
  const int64_t row = item / pieces;
  const int token = static_cast<int>(row / q_heads), c = static_cast<int>(item - row * pieces) * 8;
  while (b < a.view.batch && row_bound(a.cu, b + 1, a.rows) <= token) ++b;
  if (b == a.view.batch && !a.clear_rest) return;
  int runs = 0;
  if (b < a.view.batch) {
    Block k;
    k.start = row_bound(a.cu, b, a.rows);
    if (token < k.start) return;
    const int n = row_bound(a.cu, b + 1, a.rows) - k.start, length = max(a.lengths[b], 0);
    const int r = (token - k.start) * a.shared + static_cast<int>(row % q_heads) % a.shared;
    k.row0 = r / kRows * kRows;
    k.count = min(static_cast<int64_t>(kRows), static_cast<int64_t>(n) * a.shared - k.row0);
    k.keys = min(static_cast<int64_t>(length), static_cast<int64_t>(a.view.table_width) << a.view.page_shift);
    k.position0 = length - n;
    k.begin = chunk_start(k.position0 + k.row0 / a.shared, a.chunk);
    k.end = min(k.position0 + (k.row0 + k.count - 1) / a.shared + 1, k.keys);
    const int from = k.begin & ~31;
    if (k.end > from) runs = (k.end - from + run_length(k, a.runs) - 1) / run_length(k, a.runs);
  }
  float m = -__builtin_inff();
  for (int i = 0; i < runs; ++i) m = fmaxf(m, a.stats[(i * all + row) * 2]);
  float l = 0.f, o[8] = {};
  if (m != -__builtin_inff())
    for (int i = 0; i < runs; ++i) {
      const float mi = a.stats[(i * all + row) * 2];
      if (mi == -__builtin_inff()) continue;
      const float w = __builtin_amdgcn_exp2f(mi - m);
      l += w * a.stats[(i * all + row) * 2 + 1];
      const float4* from = reinterpret_cast<const float4*>(a.part + (i * all + row) * a.v.width + c);
      const float4 x = from[0], y = from[1];
      const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = fmaf(w, v[j], o[j]);
    }
  const float inverse = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j] = l == 0.f ? 0.f : o[j] * inverse;
  *reinterpret_cast<uint4*>(a.out + row * a.v.width + c) = pack8<DT>(o);
}

// How a call is cut.
struct Plan {
  int rt, ct, ks, waves, slabs, runs;
  int64_t blocks;
  int64_t workgroups(int64_t heads) const { return blocks * runs * heads * slabs; }
};

Plan plan_of(const mega_paged_cache* c, int64_t rows, int64_t q_heads, int64_t chunk) {
  Plan p{};
  const int64_t shared = q_heads / c->heads, sequences = std::max<int64_t>(c->batch, 1);
  // rows of a sequence, on average: a block's rows pad to the next size
  const int64_t mean = (rows * shared + sequences - 1) / sequences;
  p.rt = mean <= 16 ? 1 : mean <= 32 ? 2 : 4;
  p.ks = c->k_width <= 128 ? 4 : c->k_width <= 256 ? 8 : 16;
  p.ct = p.rt == 1 && c->v_width > 1024 ? 16 : 8;
  const int64_t per_wave = 16 * p.ct;
  p.slabs = static_cast<int>((c->v_width + kMaxWaves * per_wave - 1) / (kMaxWaves * per_wave));
  const int64_t slab = (c->v_width + p.slabs - 1) / p.slabs;
  p.waves = static_cast<int>((slab + per_wave - 1) / per_wave);
  p.blocks = rows * shared / (16 * p.rt) + c->batch + 1;
  // runs: until the chip has its waves; none shorter than 32 keys
  const int64_t keys = std::min(c->table_width * c->page_size, chunk > 0 ? chunk : INT64_MAX);
  const int64_t full = std::max<int64_t>(1, std::max(rows * shared / (16 * p.rt), std::min(c->batch, rows))) * c->heads * p.slabs * p.waves;
  const int64_t wanted = 2048;  // eight waves to a CU
  p.runs = static_cast<int>(std::clamp<int64_t>(wanted / full, 1, std::min<int64_t>(kMaxRuns, std::max<int64_t>(1, keys / 32))));
  return p;
}

template <int DT, bool kEight, int RT, int CT, int KS>
int launch_attn(const AttnArgs& a, const Plan& p, void* stream) {
  const auto kernel = paged_attn_kernel<DT, kEight, RT, CT, KS>;
  const size_t bytes = (RT * KS * 64 + p.waves * RT * 64) * sizeof(uint4) + RT * 16 * 8 * sizeof(float);
  if (bytes > 65536)
    MEGA_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)));
  hipStream_t s = static_cast<hipStream_t>(stream);
  kernel<<<dim3(static_cast<uint32_t>(p.workgroups(a.heads))), dim3(p.waves * kWave), bytes, s>>>(a);
  MEGA_CHECK_LAUNCH();
  if (p.runs > 1) {
    const int64_t items = static_cast<int64_t>(a.rows) * a.heads * a.shared * (a.v.width / 8);
    paged_join_kernel<DT, 16 * RT><<<dim3(static_cast<uint32_t>((items + kJoinThreads - 1) / kJoinThreads)), dim3(kJoinThreads), 0, s>>>(a);
    MEGA_CHECK_LAUNCH();
  }
  return MEGA_OK;
}

template <int DT, bool kEight, int KS>
int launch_rows(const AttnArgs& a, const Plan& p, void* stream) {
  if (p.rt == 1 && p.ct == 16) return launch_attn<DT, kEight, 1, 16, KS>(a, p, stream);
  if (p.rt == 1) return launch_attn<DT, kEight, 1, 8, KS>(a, p, stream);
  if (p.rt == 2) return launch_attn<DT, kEight, 2, 8, KS>(a, p, stream);
  return launch_attn<DT, kEight, 4, 8, KS>(a, p, stream);
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
  const Plan p = plan_of(cache, rows, q_heads, chunk);
  return p.runs > 1 ? p.runs * rows * q_heads * (cache->v_width + 2) * static_cast<int64_t>(sizeof(float)) : 0;
}

extern "C" int mega_paged_attention_fwd(const mega_paged_cache* cache, int dtype, const void* q, int64_t q_row, int64_t q_head,
                                        const int32_t* lengths, const int32_t* cu, int64_t rows, int64_t q_heads, double scale,
                                        int64_t chunk, void* out, int clear_rest, void* workspace, void* stream) {
  if (const int rc = check_paged_cache(cache, dtype, "mega_paged_attention_fwd"); rc != MEGA_OK) return rc;
  MEGA_CHECK_ARG(sizes_fit(cache, rows, q_heads, chunk), "mega_paged_attention_fwd: bad sizes (q_heads has to be a multiple of the cache's heads)");
  MEGA_CHECK_ARG(cache->k_width <= kMaxKeyWidth, "mega_paged_attention_fwd: k_width must be at most 512");
  if (rows == 0) return MEGA_OK;
  MEGA_CHECK_ARG(q != nullptr && out != nullptr && (lengths != nullptr || cache->batch == 0) && cu != nullptr, "mega_paged_attention_fwd: null pointer");
  MEGA_CHECK_ARG(reinterpret_cast<uintptr_t>(q) % 16 == 0 && q_row % 8 == 0 && q_head % 8 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0,
                 "mega_paged_attention_fwd: q and out must be 16-byte aligned");
  const Plan p = plan_of(cache, rows, q_heads, chunk);
  MEGA_CHECK_ARG(p.workgroups(cache->heads) <= 0x7fffffff && rows * (q_heads / cache->heads) <= 0x7fffffff, "mega_paged_attention_fwd: too many rows for one launch");
  MEGA_CHECK_ARG(p.runs == 1 || (workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
                 "mega_paged_attention_fwd: a 16-byte aligned workspace is needed");
  AttnArgs a{};
  a.view = paged_view(cache), a.k = paged_pool(cache, false), a.v = paged_pool(cache, true);
  a.q = static_cast<const uint16_t*>(q), a.q_row = q_row, a.q_head = q_head;
  a.lengths = lengths, a.cu = cu, a.out = static_cast<uint16_t*>(out);
  a.part = static_cast<float*>(workspace);
  if (p.runs > 1) a.stats = a.part + p.runs * rows * q_heads * cache->v_width;
  a.rows = static_cast<int32_t>(rows), a.heads = static_cast<int32_t>(cache->heads), a.shared = static_cast<int32_t>(q_heads / cache->heads);
  a.chunk = static_cast<int32_t>(chunk), a.runs = p.runs, a.slabs = p.slabs, a.blocks = static_cast<int32_t>(p.blocks);
  a.clear_rest = clear_rest != 0;
  a.scale = static_cast<float>(scale * 1.4426950408889634);
  const bool eight = cache->k_exponents != nullptr;
  if (dtype == MEGA_BF16) return eight ? launch_width<MEGA_BF16, true>(a, p, stream) : launch_width<MEGA_BF16, false>(a, p, stream);
  return eight ? launch_width<MEGA_F16, true>(a, p, stream) : launch_width<MEGA_F16, false>(a, p, stream);
}
