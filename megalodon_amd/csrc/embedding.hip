// Embedding for gfx950: rows of a table by token, and the table's gradient.
//   y[r] = s W[t_r]                      (float32 / bfloat16 / float16, rounded once)
//   dW[v] = s sum over r with t_r = v of dy[r]   (float32 sums, in an order that sizes and tokens alone set)
// A token that is no row of the table gives zeros and takes no gradient; the padding token gives its row and takes none.
//
// Both are bound by the bytes they move.  The gradient sorts the positions by token (stable), cuts the sorted line into equal pieces, so that
// no frequent token keeps one workgroup, and sums each piece's runs of one token in registers.  A run that ends inside its piece is a row
// of dW; runs over a piece's ends leave float32 sums that a second kernel adds up in their order.  Rows without a token are
// zeroed by the same launch.  The only atomics count integers: the same call gives the same bits.
// Narrow rows leave a piece few threads, so that a workgroup has several pieces (bfloat16 gradients of 262144 tokens, us, one / several: 64 columns,
// 1000 rows 169 / 67, 1048576 tokens 675 / 128).  32768 tokens, 32000 rows of 4096: sums 100 us of 126, 5.3 TB/s.
#include "common.hpp"

#include <algorithm>

namespace mega {
namespace {

constexpr int kThreads = 256;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_any16 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4_any32 __attribute__((ext_vector_type(4), aligned(4)));

// 16 bytes at any element's boundary; behind the end (left < what 16 bytes hold) element by element, zeros for the rest
template <int DT> struct Row {
  static constexpr int kPer = DT == MEGA_F32 ? 4 : 8;  // elements of 16 bytes
  using T = typename Elem<DT>::type;
  using Any = std::conditional_t<DT == MEGA_F32, u32x4_any32, u32x4_any16>;
  static __device__ __forceinline__ void load(const T* p, int left, float* v) {
    if (left >= kPer) {
      unpack(__builtin_bit_cast(uint4, *reinterpret_cast<const Any*>(p)), v);
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e) v[e] = e < left ? Elem<DT>::load(p + e) : 0.f;
    }
  }
  static __device__ __forceinline__ void unpack(uint4 q, float* v) {
    if constexpr (DT == MEGA_F32) {
      v[0] = __uint_as_float(q.x), v[1] = __uint_as_float(q.y), v[2] = __uint_as_float(q.z), v[3] = __uint_as_float(q.w);
    } else {
      unpack8<DT>(q, v);
    }
  }
  // (a whole piece of what is read once)
  static __device__ __forceinline__ void load_once(const T* p, int left, float* v) {
    if (left >= kPer) unpack(__builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const Any*>(p))), v);
    else load(p, left, v);
  }
  // (streaming: whole cache lines that nobody reads here; half lines are written slowly with the hint)
  static __device__ __forceinline__ void store(T* p, int left, const float* v, bool streaming) {
    if (left >= kPer) {
      uint4 q;
      if constexpr (DT == MEGA_F32) q = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
      else q = pack8<DT>(v);
      if (streaming) __builtin_nontemporal_store(__builtin_bit_cast(Any, q), reinterpret_cast<Any*>(p));
      else *reinterpret_cast<Any*>(p) = __builtin_bit_cast(Any, q);
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (e < left) Elem<DT>::store(p + e, v[e]);
    }
  }
};

// ---- forward ------------------------------------------------------------------------------------------
// A thread has one 16-byte piece of ROWS rows, so that as many table rows are in flight behind their tokens.
template <int DT, typename Token, int ROWS>
__global__ __launch_bounds__(kThreads) void gather_kernel(const Token* tokens, const typename Elem<DT>::type* table, typename Elem<DT>::type* out,
                                                         int64_t n, int64_t vocab, int width, int64_t ld, float scale, bool streaming) {
  constexpr int kPer = Row<DT>::kPer;
  const int pieces = (width + kPer - 1) / kPer;
  const int64_t groups = (n + ROWS - 1) / ROWS;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < groups * pieces; i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t r0 = i / pieces * ROWS;
    const int k = static_cast<int>(i % pieces) * kPer;
    int64_t token[ROWS];
#pragma unroll
    for (int q = 0; q < ROWS; ++q) token[q] = tokens[min(r0 + q, n - 1)];
    float v[ROWS][kPer];
#pragma unroll
    for (int q = 0; q < ROWS; ++q) {
      const bool there = token[q] >= 0 && token[q] < vocab;
      Row<DT>::load(table + (there ? token[q] : 0) * ld + k, width - k, v[q]);
      if (!there)
#pragma unroll
        for (int e = 0; e < kPer; ++e) v[q][e] = 0.f;
    }
#pragma unroll
    for (int q = 0; q < ROWS; ++q) {
      if (r0 + q >= n) break;
#pragma unroll
      for (int e = 0; e < kPer; ++e) v[q][e] *= scale;
      Row<DT>::store(out + (r0 + q) * width + k, width - k, v[q], streaming);
    }
  }
}

// ---- positions by token -----------------------------------------------------------------------------------
// Sorting key of a token: its row, or `vocab` for what takes no gradient.
template <typename Token>
__device__ __forceinline__ uint32_t key_of(Token t, int64_t vocab, int64_t padding) {
  const int64_t v = static_cast<int64_t>(t);
  return static_cast<uint32_t>(v < 0 || v >= vocab || v == padding ? vocab : v);
}

// Up to kRankTokens positions: the place of a position is the number of keys below its own and of equal ones in front of it, n^2 comparisons
// with keys in LDS.  A workgroup has 16 positions; sixteen lanes at a time have a 64th of the keys each.
constexpr int kRankTokens = 8192, kRankWaves = 16, kRankEach = 16, kRankParts = kRankWaves * kWave / kRankEach;

template <typename Token>
__global__ __launch_bounds__(kRankWaves * kWave) void rank_kernel(const Token* tokens, int n, int64_t vocab, int64_t padding, uint32_t* keys, uint32_t* order) {
  __shared__ __align__(16) uint32_t all[kRankTokens + 4];
  __shared__ uint32_t counts[kRankParts][kRankEach];
  const int quads = (n + 3) / 4;
  for (int j = threadIdx.x; j < quads * 4; j += kRankWaves * kWave) all[j] = j < n ? key_of(tokens[j], vocab, padding) : 0xffffffffu;
  __syncthreads();
  const int own = threadIdx.x % kRankEach, part = threadIdx.x / kRankEach, first = blockIdx.x * kRankEach, i = first + own;
  const uint32_t mine = i < n ? all[i] : 0xffffffffu;
  // quads of keys in front of the workgroup's positions (equal ones count), its own, and those behind (equal ones do not)
  uint32_t count = 0;
  const int own_quad = first / 4;
  int q = part;
#pragma unroll 4
  for (; q < own_quad; q += kRankParts) {
    const uint4 k = *reinterpret_cast<const uint4*>(all + 4 * q);
    count += (k.x <= mine) + (k.y <= mine) + (k.z <= mine) + (k.w <= mine);
  }
  if (q < min(own_quad + kRankEach / 4, quads)) {
    for (int j = 4 * q; j < 4 * q + 4; ++j) count += all[j] < mine || (all[j] == mine && j < i);
    q += kRankParts;
  }
#pragma unroll 4
  for (; q < quads; q += kRankParts) {
    const uint4 k = *reinterpret_cast<const uint4*>(all + 4 * q);
    count += (k.x < mine) + (k.y < mine) + (k.z < mine) + (k.w < mine);
  }
  counts[part][own] = count;
  __syncthreads();
  if (part > 0 || i >= n) return;
#pragma unroll
  for (int p = 1; p < kRankParts; ++p) count += counts[p][own];
  keys[count] = mine;
  order[count] = static_cast<uint32_t>(i);
}

// More: digits from the lowest up, each a stable move of all positions; a workgroup has `tiles` times kSortBlock of them, one after the other.  Few
// workgroups read each other's counts where they need them, more than kSortAlone have them added up by a launch between (their reads grow with
// the square: 262144 positions, two digits, us without / with: 160 / 45).  Positions of a thread, us for all of the gradient at 1, 2, 4:
// 8193 tokens of 64 columns 37, 41, 44, 65536 49, 49, 52, 1048576 158, 158, 153.
constexpr int kSortThreads = 512, kSortWaves = kSortThreads / kWave, kSortEach = 2, kSortBlock = kSortThreads * kSortEach, kMostDigits = 2048;
constexpr int kSortAlone = 64, kSortGroups = 1024;

// what the passes move: in the first, the tokens themselves
template <typename Token>
struct Positions {
  const Token* tokens;           // first pass, else null
  const uint32_t *keys, *order;  // the others
  int64_t vocab, padding;
  __device__ __forceinline__ uint32_t key(int64_t i) const { return tokens != nullptr ? key_of(tokens[i], vocab, padding) : keys[i]; }
};

template <typename Token>
__global__ __launch_bounds__(kSortThreads) void count_kernel(const Positions<Token> from, int64_t n, int tiles, int shift, int digits, uint32_t* counts) {
  __shared__ uint32_t seen[kMostDigits];
  for (int d = threadIdx.x; d < digits; d += kSortThreads) seen[d] = 0;
  __syncthreads();
  for (int tile = 0; tile < tiles; ++tile) {
#pragma unroll
    for (int q = 0; q < kSortEach; ++q) {
      const int64_t i = (static_cast<int64_t>(blockIdx.x) * tiles + tile) * kSortBlock + q * kSortThreads + threadIdx.x;
      if (i < n) atomicAdd(&seen[from.key(i) >> shift & (digits - 1)], 1u);
    }
  }
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += kSortThreads) counts[static_cast<int64_t>(blockIdx.x) * digits + d] = seen[d];
}

// counts [group][digit] to those of the groups in front, and behind them the totals: a lane has a digit, the waves have a sixteenth of the groups each
constexpr int kScanWaves = 16;
__global__ __launch_bounds__(kScanWaves * kWave) void scan_kernel(uint32_t* counts, int groups, int digits) {
  __shared__ uint32_t sums[kScanWaves][kWave];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, d = blockIdx.x * kWave + lane;
  const int lo = groups * wave / kScanWaves, hi = groups * (wave + 1) / kScanWaves;
  uint32_t sum = 0;
  if (d < digits) {
#pragma unroll 8
    for (int g = lo; g < hi; ++g) sum += counts[static_cast<int64_t>(g) * digits + d];
  }
  sums[wave][lane] = sum;
  __syncthreads();
  if (d >= digits) return;
  uint32_t at = 0;
  for (int w = 0; w < wave; ++w) at += sums[w][lane];
#pragma unroll 8
  for (int g = lo; g < hi; ++g) {
    const uint32_t c = counts[static_cast<int64_t>(g) * digits + d];
    counts[static_cast<int64_t>(g) * digits + d] = at;
    at += c;
  }
  if (wave == kScanWaves - 1) counts[static_cast<int64_t>(groups) * digits + d] = at;
}

// A digit's first place for this workgroup: all smaller digits, and its own of the workgroups in front.  A wave has 64 kSortEach consecutive
// positions, 64 at a time: lanes of one digit find each other by ballots, one of them advances the wave's count of it.
template <typename Token>
__global__ __launch_bounds__(kSortThreads) void move_kernel(const Positions<Token> from, int64_t n, int tiles, int shift, int bits, const uint32_t* counts,
                                                           uint32_t* keys, uint32_t* order) {
  extern __shared__ uint32_t lds[];
  const int digits = 1 << bits, lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, groups = static_cast<int>(gridDim.x);
  uint32_t* const begins = lds;                  // [digits]
  uint32_t* const seen = lds + digits;           // [wave][digits]
  __shared__ uint32_t totals[kMostDigits], wave_sums[kSortWaves];
  if (groups > kSortAlone) {
    for (int d = threadIdx.x; d < digits; d += kSortThreads) {
      begins[d] = counts[static_cast<int64_t>(blockIdx.x) * digits + d];
      totals[d] = counts[static_cast<int64_t>(groups) * digits + d];
    }
  } else {
    for (int d = threadIdx.x; d < digits; d += kSortThreads) begins[d] = totals[d] = 0;
    __syncthreads();
    const int parts = max(kSortThreads / digits, 1);  // threads of a digit
    for (int i = threadIdx.x; i < digits * parts; i += kSortThreads) {
      const int d = i % digits;
      uint32_t before = 0, total = 0;
#pragma unroll 8
      for (int g = i / digits; g < groups; g += parts) {
        const uint32_t c = counts[g * digits + d];
        if (g < static_cast<int>(blockIdx.x)) before += c;
        total += c;
      }
      atomicAdd(&begins[d], before);
      atomicAdd(&totals[d], total);
    }
  }
  __syncthreads();
  // neighbouring digits a thread
  const int each = (digits + kSortThreads - 1) / kSortThreads;
  uint32_t sum = 0;
  for (int q = 0; q < each; ++q)
    if (const int d = each * threadIdx.x + q; d < digits) sum += totals[d];
  const uint32_t own = sum;
#pragma unroll
  for (int step = 1; step < kWave; step *= 2) {
    const uint32_t up = __shfl_up(sum, step);
    if (lane >= step) sum += up;
  }
  if (lane == kWave - 1) wave_sums[wave] = sum;
  __syncthreads();
  uint32_t at = sum - own;
  for (int w = 0; w < wave; ++w) at += wave_sums[w];
  for (int q = 0; q < each; ++q)
    if (const int d = each * threadIdx.x + q; d < digits) begins[d] += at, at += totals[d];
  for (int tile = 0; tile < tiles; ++tile) {
  for (int d = threadIdx.x; d < digits * kSortWaves; d += kSortThreads) seen[d] = 0;
  __syncthreads();
  uint32_t key[kSortEach], rank[kSortEach];
  volatile uint32_t* const mine = seen + wave * digits;
  const int64_t first = (static_cast<int64_t>(blockIdx.x) * tiles + tile) * kSortBlock + wave * (kWave * kSortEach) + lane;
#pragma unroll
  for (int q = 0; q < kSortEach; ++q) key[q] = first + q * kWave < n ? from.key(first + q * kWave) : 0;
#pragma unroll
  for (int q = 0; q < kSortEach; ++q) {
    const bool there = first + q * kWave < n;
    const uint32_t d = key[q] >> shift & (digits - 1);
    uint64_t same = __ballot(there);
    for (int bit = 0; bit < bits; ++bit) {
      const uint64_t set = __ballot(d >> bit & 1);
      same &= d >> bit & 1 ? set : ~set;
    }
    const int in_front = __popcll(same & ((1ull << lane) - 1));
    if (there) {
      const uint32_t old = mine[d];
      rank[q] = old + in_front;
      __builtin_amdgcn_wave_barrier();
      if (in_front == 0) mine[d] = old + __popcll(same);
    }
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += kSortThreads) {
    uint32_t place = begins[d];
    for (int w = 0; w < kSortWaves; ++w) {
      const uint32_t c = seen[w * digits + d];
      seen[w * digits + d] = place;
      place += c;
    }
    begins[d] = place;
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < kSortEach; ++q) {
    const int64_t i = first + q * kWave;
    if (i >= n) break;
    const uint32_t to = seen[wave * digits + (key[q] >> shift & (digits - 1))] + rank[q];
    if (to >= n) break;  // (tokens that somebody wrote since they were counted: no order, but nothing outside the workspace)
    keys[to] = key[q];
    order[to] = from.tokens != nullptr ? static_cast<uint32_t>(i) : from.order[i];
  }
  __syncthreads();
  }
}

// ---- sums ---------------------------------------------------------------------------------------------------
struct SumParams {
  const void* dy;
  void* dw;
  const uint32_t *keys, *order;
  float* open;      // [piece][2][width]: sums of runs that begin in front of the piece, and of those that go on behind it
  int64_t n, vocab;
  int width, per_piece, slices, threads;  // threads: of a piece (narrow rows: several pieces to a workgroup)
  int64_t pieces, groups;                 // groups: workgroups of a slice
  float scale;
  bool streaming, past_cache;  // past_cache: zeros
};
constexpr int kZeroRows = 16;  // rows of dW that a workgroup looks at
constexpr int kMostPiece = 1024;  // positions of a workgroup

template <int DT>
__global__ __launch_bounds__(kThreads) void sum_kernel(const SumParams p) {
  using R = Row<DT>;
  using T = typename Elem<DT>::type;
  constexpr int kPer = R::kPer, kAhead = 8;
  const int tid = threadIdx.x;
  if (blockIdx.x >= p.groups * p.slices) {
    // rows without a token: lanes look for 16 rows' keys, the workgroup writes
    __shared__ uint32_t empty;
    const int64_t begin = blockIdx.x - p.groups * p.slices, step = gridDim.x - p.groups * p.slices;
    for (int64_t v0 = begin * kZeroRows; v0 < p.vocab; v0 += step * kZeroRows) {
    if (tid < kWave) {
      const int64_t v = v0 + tid;
      bool none = false;
      if (tid < kZeroRows && v < p.vocab) {
        int64_t lo = 0, hi = p.n;
        while (lo < hi) {
          const int64_t mid = (lo + hi) / 2;
          if (p.keys[mid] < v) lo = mid + 1;
          else hi = mid;
        }
        none = lo == p.n || p.keys[lo] != v;
      }
      const uint64_t mask = __ballot(none);
      if (tid == 0) empty = static_cast<uint32_t>(mask);
    }
    __syncthreads();
    // (rows beside each other are one line of memory, written in whole pieces whatever their width is: 4084 tokens, 50001 rows of 1001 floats 69 us row by
    // row, 66.5 so, 64.3 past the cache, which a table of half its size and more would only pass through)
    for (uint32_t m = empty; m != 0;) {
      const int first = __builtin_ctz(m), rows = __builtin_ctz(~(m >> first));
      m &= ~(((1u << rows) - 1) << first);
      T* const line = static_cast<T*>(p.dw) + (v0 + first) * p.width;
      const int n = rows * p.width, head = min(static_cast<int>(-reinterpret_cast<uintptr_t>(line) % 16 / sizeof(T)), n), whole = (n - head) / kPer;
      if (tid < head) line[tid] = T(0);
      u32x4* const to = reinterpret_cast<u32x4*>(line + head);
      if (p.past_cache) {
        for (int i = tid; i < whole; i += kThreads) __builtin_nontemporal_store(u32x4{0, 0, 0, 0}, to + i);
      } else {
        for (int i = tid; i < whole; i += kThreads) to[i] = u32x4{0, 0, 0, 0};
      }
      if (const int at = head + whole * kPer + tid; at < n) line[at] = T(0);
    }
    __syncthreads();
    }
    return;
  }
  const int each = kThreads / p.threads, own = tid / p.threads;  // pieces of the workgroup, the thread's among them
  const int64_t piece0 = blockIdx.x / p.slices * each, first = piece0 * p.per_piece, piece = piece0 + own;
  const int k = (blockIdx.x % p.slices * kThreads + tid % p.threads) * kPer, left = p.width - k;
  const int all = static_cast<int>(min(static_cast<int64_t>(p.per_piece) * each, p.n - first));
  __shared__ uint32_t all_keys[kMostPiece + 2], all_order[kMostPiece];  // all_keys[0] and [all + 1]: the neighbours'
  for (int i = tid; i < all + 2; i += kThreads) {
    const int64_t at = first + i - 1;
    all_keys[i] = at >= 0 && at < p.n ? p.keys[at] : 0xffffffffu;
    if (i < all) all_order[i] = min(p.order[first + i], static_cast<uint32_t>(p.n - 1));  // (as above)
  }
  __syncthreads();
  const int count = min(p.per_piece, all - own * p.per_piece);
  if (own >= each || count <= 0 || left <= 0) return;
  const uint32_t *const keys = all_keys + own * p.per_piece, *const order = all_order + own * p.per_piece;  // keys[0] and keys[count + 1]: the neighbours'
  if (keys[1] >= p.vocab) return;
  const T* const dy = static_cast<const T*>(p.dy) + k;
  T* const dw = static_cast<T*>(p.dw) + k;
  float* const open = p.open + piece * 2 * p.width + k;
  float sum[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) sum[e] = 0.f;
  bool begun = keys[0] != keys[1];  // the run begins in this piece
  for (int i = 0; i < count; i += kAhead) {
    float v[kAhead][kPer];
#pragma unroll
    for (int q = 0; q < kAhead; ++q) R::load_once(dy + static_cast<int64_t>(order[min(i + q, count - 1)]) * p.width, left, v[q]);
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      if (i + q >= count) break;
      const uint32_t key = keys[1 + i + q], next = keys[2 + i + q];
      if (key >= p.vocab) return;
#pragma unroll
      for (int e = 0; e < kPer; ++e) sum[e] += v[q][e];
      const bool ends = key != next;
      if (!ends && i + q + 1 < count) continue;
      if (begun && ends) {
#pragma unroll
        for (int e = 0; e < kPer; ++e) sum[e] *= p.scale;
        R::store(dw + static_cast<int64_t>(key) * p.width, left, sum, p.streaming);
      } else {
        // (a piece inside a run: its sum counts as that of the run's part from in front)
        float* const to = open + (begun ? p.width : 0);
#pragma unroll
        for (int e = 0; e < kPer; ++e)
          if (e < left) to[e] = sum[e];
      }
      begun = true;
#pragma unroll
      for (int e = 0; e < kPer; ++e) sum[e] = 0.f;
    }
  }
}

// Runs over the end of the piece that they begin in: the parts of it and of the pieces behind, in their order.  A workgroup has `columns` columns, VEC of
// them a thread (4 in wide rows: a quarter of the workgroups, most of which find nothing to do; 32768 tokens, 4096 columns 10.6 us, 9.0 so); in narrow
// rows its threads share a column's parts.
template <int DT, int VEC>
__global__ __launch_bounds__(kThreads) void join_kernel(const SumParams p, int columns) {
  const int per = columns / VEC;  // threads of the columns
  const unsigned slices = (p.width + columns - 1) / columns, group = group_number(), piece = group / slices;
  const int tid = threadIdx.x, k = static_cast<int>(group % slices) * columns + tid % per * VEC, share = tid / per, shares = kThreads / per;
  const int64_t first = static_cast<int64_t>(piece) * p.per_piece, behind = first + p.per_piece;
  if (behind >= p.n) return;
  const uint32_t key = p.keys[behind], last = p.keys[behind - 1], head = p.keys[first], ahead = first > 0 ? p.keys[first - 1] : 0xffffffffu;
  if (key >= p.vocab || last != key) return;
  if (head == key && ahead == key) return;  // begins further in front
  // pieces behind whose first position is of the run, 256 at a time
  int parts = 0;
  for (bool more = true; more; ) {
    uint64_t in[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t at = behind + static_cast<int64_t>(parts + j * kWave + tid % kWave) * p.per_piece;
      in[j] = __ballot(at < p.n && p.keys[min(at, p.n - 1)] == key);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int run = in[j] == ~0ull ? kWave : __builtin_ctzll(~in[j]);
      if (more) parts += run;
      more = more && run == kWave;
    }
  }
  const int64_t step = 2 * static_cast<int64_t>(p.width);
  const int begin = static_cast<int>(static_cast<int64_t>(parts) * share / shares);
  int left = static_cast<int>(static_cast<int64_t>(parts) * (share + 1) / shares) - begin;
  const int columns_left = p.width - k;
  using Floats = float __attribute__((ext_vector_type(VEC), aligned(4)));
  const auto load = [&](const float* from) {
    Floats v;
    if (columns_left >= VEC) {
      v = *reinterpret_cast<const Floats*>(from);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = e < columns_left ? from[e] : 0.f;
    }
    return v;
  };
  Floats sum = 0.f;
  if (columns_left > 0) {
    const float* open = p.open + piece * step + k;
    if (share == 0) sum = load(open + p.width);
    open += begin * step;
    constexpr int kAhead = 16 / VEC * (VEC > 1 ? 2 : 1);  // parts in flight
    for (; left >= kAhead; left -= kAhead) {
      Floats v[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) v[i] = load(open += step);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) sum += v[i];
    }
    for (; left > 0; --left) sum += load(open += step);
  }
  if (shares > 1) {
    __shared__ Floats sums[kThreads];
    sums[tid] = sum;
    __syncthreads();
    if (share > 0) return;
    for (int i = 1; i < shares; ++i) sum += sums[i * per + tid];
  }
  auto* const to = static_cast<typename Elem<DT>::type*>(p.dw) + static_cast<int64_t>(key) * p.width + k;
#pragma unroll
  for (int e = 0; e < VEC; ++e)
    if (e < columns_left) Elem<DT>::store(to + e, sum[e] * p.scale);
}

// ---- host side ------------------------------------------------------------------------------------------------
// rows of whole cache lines
bool whole_lines(const void* p, int64_t width, int dtype) { return reinterpret_cast<uintptr_t>(p) % 128 == 0 && width * elem_size(dtype) % 128 == 0; }
int64_t up(int64_t n) { return (n + 255) / 256 * 256; }

struct Sizes {
  int bits, passes, tiles;  // of a sorting pass, and how many
  int slices, per_piece, threads;
  int64_t blocks, pieces, groups, bytes, keys[2], order[2], counts, open;  // (offsets into the workspace)
  Sizes(int dtype, int64_t n, int64_t vocab, int64_t width) {
    int all = 1;
    while ((vocab >> all) > 0) ++all;  // of keys up to `vocab`
    passes = (all + 10) / 11;
    bits = (all + passes - 1) / passes;
    const int64_t lines = (n + kSortBlock - 1) / kSortBlock;
    tiles = static_cast<int>((lines + kSortGroups - 1) / kSortGroups);
    blocks = tiles > 0 ? (lines + tiles - 1) / tiles : 0;
    const int per = kThreads * (dtype == MEGA_F32 ? 4 : 8);
    slices = static_cast<int>((width + per - 1) / per);
    threads = slices > 1 ? kThreads : static_cast<int>((width + per / kThreads - 1) / (per / kThreads));
    const int each = kThreads / threads;
    per_piece = each <= kMostPiece / 16 ? 16 : kMostPiece / each;
    while (2 * per_piece * each <= kMostPiece && per_piece * each * 1024ll < n * slices) per_piece *= 2;
    pieces = (n + per_piece - 1) / per_piece, groups = (pieces + each - 1) / each;
    const bool sorts = n > kRankTokens;
    bytes = 0;
    const auto take = [&](int64_t size) { const int64_t at = bytes; bytes += up(size); return at; };
    for (int i = 0; i < 2; ++i) keys[i] = i == 0 || sorts ? take(4 * n) : 0, order[i] = i == 0 || sorts ? take(4 * n) : 0;
    counts = sorts ? take(4 * ((blocks + 1) << bits)) : 0;
    open = take(4 * pieces * 2 * width);
  }
};

int check_sizes(const char* who, int dtype, int token_bits, int64_t n, int64_t vocab, int64_t width) {
  MEGA_CHECK_ARG(valid_dtype(dtype), "%s: float32, bfloat16 or float16 tables", who);
  MEGA_CHECK_ARG(token_bits == 32 || token_bits == 64, "%s: tokens of 32 or 64 bits", who);
  MEGA_CHECK_ARG(n >= 0 && n < (1ll << 31) && vocab >= 1 && vocab < (1ll << 31) && width >= 1 && width <= (1 << 20), "%s: bad sizes", who);
  return MEGA_OK;
}

template <int DT, typename Token>
int gather(const Token* tokens, const void* table, int64_t n, int64_t vocab, int64_t width, int64_t ld, float scale, void* out, hipStream_t s) {
  using T = typename Elem<DT>::type;
  const int64_t pieces = (width + Row<DT>::kPer - 1) / Row<DT>::kPer;
  const bool streaming = whole_lines(out, width, DT);
  const auto grid = [&](int64_t rows) { return static_cast<unsigned>(std::min<int64_t>(((n + rows - 1) / rows * pieces + kThreads - 1) / kThreads, 1 << 20)); };
  if (n * pieces <= (1 << 18))
    gather_kernel<DT, Token, 1><<<grid(1), kThreads, 0, s>>>(tokens, static_cast<const T*>(table), static_cast<T*>(out), n, vocab, static_cast<int>(width), ld, scale, streaming);
  else
    gather_kernel<DT, Token, 4><<<grid(4), kThreads, 0, s>>>(tokens, static_cast<const T*>(table), static_cast<T*>(out), n, vocab, static_cast<int>(width), ld, scale, streaming);
  MEGA_CHECK_LAUNCH();
  return MEGA_OK;
}

template <typename Token>
int sort_positions(const Token* tokens, int64_t n, int64_t vocab, int64_t padding, const Sizes& z, char* ws, const uint32_t** keys, const uint32_t** order, hipStream_t s) {
  const auto at = [&](int64_t offset) { return reinterpret_cast<uint32_t*>(ws + offset); };
  if (n <= kRankTokens) {
    rank_kernel<Token><<<static_cast<unsigned>((n + kRankEach - 1) / kRankEach), kRankWaves * kWave, 0, s>>>(tokens, static_cast<int>(n), vocab, padding, at(z.keys[0]), at(z.order[0]));
    MEGA_CHECK_LAUNCH();
    *keys = at(z.keys[0]), *order = at(z.order[0]);
    return MEGA_OK;
  }
  Positions<Token> from{tokens, nullptr, nullptr, vocab, padding};
  const size_t lds = sizeof(uint32_t) * ((kSortWaves + 1) << z.bits);
  MEGA_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&move_kernel<Token>), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds)));
  for (int pass = 0; pass < z.passes; ++pass) {
    uint32_t *to_keys = at(z.keys[pass & 1]), *to_order = at(z.order[pass & 1]);
    count_kernel<Token><<<static_cast<unsigned>(z.blocks), kSortThreads, 0, s>>>(from, n, z.tiles, pass * z.bits, 1 << z.bits, at(z.counts));
    MEGA_CHECK_LAUNCH();
    if (z.blocks > kSortAlone) {
      scan_kernel<<<((1 << z.bits) + kWave - 1) / kWave, kScanWaves * kWave, 0, s>>>(at(z.counts), static_cast<int>(z.blocks), 1 << z.bits);
      MEGA_CHECK_LAUNCH();
    }
    move_kernel<Token><<<static_cast<unsigned>(z.blocks), kSortThreads, lds, s>>>(from, n, z.tiles, pass * z.bits, z.bits, at(z.counts), to_keys, to_order);
    MEGA_CHECK_LAUNCH();
    from = Positions<Token>{nullptr, to_keys, to_order, vocab, padding};
  }
  *keys = from.keys, *order = from.order;
  return MEGA_OK;
}

template <int DT>
int table_grad(const void* dy, const void* tokens, int token_bits, int64_t n, int64_t vocab, int64_t width, float scale, int64_t padding, void* dw, char* ws, hipStream_t s) {
  const Sizes z(DT, n, vocab, width);
  SumParams p{};
  p.dy = dy, p.dw = dw, p.open = reinterpret_cast<float*>(ws + z.open);
  p.n = n, p.vocab = vocab, p.width = static_cast<int>(width), p.per_piece = z.per_piece, p.slices = z.slices, p.threads = z.threads, p.pieces = z.pieces, p.groups = z.groups, p.scale = scale, p.streaming = whole_lines(dw, width, DT), p.past_cache = vocab * width * elem_size(DT) >= 128ll << 20;
  if (n > 0) {
    const int rc = token_bits == 64 ? sort_positions(static_cast<const int64_t*>(tokens), n, vocab, padding, z, ws, &p.keys, &p.order, s)
                                    : sort_positions(static_cast<const int32_t*>(tokens), n, vocab, padding, z, ws, &p.keys, &p.order, s);
    if (rc != MEGA_OK) return rc;
  }
  const int64_t groups = p.groups * p.slices + std::min<int64_t>((vocab + kZeroRows - 1) / kZeroRows, 1 << 20);  // (2^32 threads are the most)
  sum_kernel<DT><<<static_cast<unsigned>(groups), kThreads, 0, s>>>(p);
  MEGA_CHECK_LAUNCH();
  if (p.pieces > 1) {
    int columns = 16;
    while (columns < kThreads && columns < width) columns *= 2;
    if (width >= 4 * kThreads) columns = 4 * kThreads;
    const dim3 grid = grid_of(p.pieces * ((width + columns - 1) / columns));  // (fewer than 2^31 for any gradient that fits a device)
    if (columns > kThreads) join_kernel<DT, 4><<<grid, kThreads, 0, s>>>(p, columns);
    else join_kernel<DT, 1><<<grid, kThreads, 0, s>>>(p, columns);
    MEGA_CHECK_LAUNCH();
  }
  return MEGA_OK;
}

}  // namespace
}  // namespace mega

using namespace mega;

extern "C" int mega_embedding_fwd(const void* tokens, int token_bits, const void* table, int dtype, int64_t n, int64_t vocab, int64_t width, int64_t ld,
                                  double scale, void* out, void* stream) {
  if (const int rc = check_sizes("mega_embedding_fwd", dtype, token_bits, n, vocab, width); rc != MEGA_OK) return rc;
  if (n == 0) return MEGA_OK;
  MEGA_CHECK_ARG(tokens && table && out && ld >= 0, "mega_embedding_fwd: null pointer or bad row pitch");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const float f = static_cast<float>(scale);
#define MEGA_GATHER(DT)                                                                                                                      \
  (token_bits == 64 ? gather<DT>(static_cast<const int64_t*>(tokens), table, n, vocab, width, ld, f, out, s)                                 \
                    : gather<DT>(static_cast<const int32_t*>(tokens), table, n, vocab, width, ld, f, out, s))
  return dtype == MEGA_F32 ? MEGA_GATHER(MEGA_F32) : dtype == MEGA_BF16 ? MEGA_GATHER(MEGA_BF16) : MEGA_GATHER(MEGA_F16);
#undef MEGA_GATHER
}

extern "C" int64_t mega_embedding_workspace_bytes(int dtype, int64_t n, int64_t vocab, int64_t width) {
  if (!valid_dtype(dtype) || n < 1 || n >= (1ll << 31) || vocab < 1 || vocab >= (1ll << 31) || width < 1 || width > (1 << 20)) return 0;
  return Sizes(dtype, n, vocab, width).bytes;
}

extern "C" int mega_embedding_bwd(const void* dy, int dtype, const void* tokens, int token_bits, int64_t n, int64_t vocab, int64_t width, double scale,
                                  int64_t padding, void* dw, void* workspace, void* stream) {
  if (const int rc = check_sizes("mega_embedding_bwd", dtype, token_bits, n, vocab, width); rc != MEGA_OK) return rc;
  MEGA_CHECK_ARG(dw && (n == 0 || (dy && tokens && workspace)) && reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "mega_embedding_bwd: null or misaligned pointer");
  hipStream_t s = static_cast<hipStream_t>(stream);
  char* const ws = static_cast<char*>(workspace);
  const float f = static_cast<float>(scale);
  switch (dtype) {
    case MEGA_F32: return table_grad<MEGA_F32>(dy, tokens, token_bits, n, vocab, width, f, padding, dw, ws, s);
    case MEGA_BF16: return table_grad<MEGA_BF16>(dy, tokens, token_bits, n, vocab, width, f, padding, dw, ws, s);
    default: return table_grad<MEGA_F16>(dy, tokens, token_bits, n, vocab, width, f, padding, dw, ws, s);
  }
}
