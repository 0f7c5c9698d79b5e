// Rows into and out of the paged key / value cache.
//
// A row is one position's key or value of one head.  16 bits: a copy.  8 bits: the row's largest finite
// magnitude a gives the exponent, e = min { e : a <= 448 2^e }, read off a's own bits (448 = 0.875 * 2^9:
// with a = f 2^x, 0.5 <= f < 1, it is x - 9 where f <= 0.875 and x - 8 above); code = e4m3(x 2^-e), to nearest,
// ties to even.  A power of two costs an e4m3 number nothing (its relative step is the same at every scale short of
// its subnormals), makes both the division and the way back exact, and takes one byte a row.
//
// Bound by HBM: a row is read once and written once.  A wave has a token, all of its heads or some of them: where the token lies is looked up
// once (four loads that wait for each other), then its values go by, then its keys.  16, 32 or 64 lanes take a row, each lane pieces of eight
// elements (one 16-byte access of 16-bit ones), which it keeps in registers between the maximum and the codes; lanes that a narrow row leaves
// take the next heads.  Measured: 8-bit rows of 32000 positions back to 16 bits, 885 MB: 185 us, 4.8 TB/s (the streaming copy: 5.9); 4096 positions
// into 8 bits, 113 MB: 24 us, 4.7 TB/s; one token a sequence: a launch (4 - 5 us).  A wave a row instead: 215 us, the look-up in front of each.
#include "paged.hpp"

#include <algorithm>

namespace mega {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / kWave;
constexpr int kPieces = kMaxCacheWidth / (8 * kWave);  // of a row of the greatest width, to a lane

struct Side {
  PagedPool pool;
  void* rows;          // packed rows: new ones (write) or those handed out (read)
  int64_t row, head;   // their strides
  int lanes, lanes_log2;     // to a row
};
struct CacheArgs {
  PagedView view;
  Side side[2];               // keys, values
  const int32_t *first, *cu;  // first: lengths (write), begins (read)
  int32_t rows, heads;
  int32_t at_once, shares;    // heads of a wave; waves of a token (twice that where `apart`: keys and values have waves of their own)
  int32_t apart;
  int clear_rest;
};

// Where a token is, the same for a wave.
struct Place {
  int32_t token, head, end;  // heads head .. end - 1 are the wave's
  uint32_t page, slot;       // in the pool
  bool there, owned;         // it has a place; a sequence has it
  bool keys, values;         // what the wave moves
};

// false: the wave has nothing to do
template <bool kWrite>
__device__ __forceinline__ bool find_place(const CacheArgs& a, Place& p) {
  int64_t item = static_cast<int64_t>(group_number()) * kWaves + __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  p.keys = !a.apart || (item & 1) != 0, p.values = !a.apart || (item & 1) == 0;
  item >>= a.apart;
  if (item >= static_cast<int64_t>(a.rows) * a.shares) return false;
  p.token = static_cast<int32_t>(item / a.shares);
  p.head = static_cast<int32_t>(item - static_cast<int64_t>(p.token) * a.shares) * a.at_once, p.end = min(p.head + a.at_once, a.heads);
  p.there = p.owned = false, p.page = p.slot = 0;
  const int b = last_not_above(a.view.batch, p.token, [&](int i) { return static_cast<int64_t>(a.cu[i]); });
  const int start = row_bound(a.cu, b, a.rows), end = row_bound(a.cu, b + 1, a.rows);
  p.owned = p.token >= start && p.token < end;
  if (!p.owned) return !kWrite && a.clear_rest;
  const int64_t position = static_cast<int64_t>(a.first[b]) + (kWrite ? p.token - end : p.token - start);
  if (position >= 0 && (position >> a.view.page_shift) < a.view.table_width) {
    p.page = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(a.view.table[b * a.view.table_stride + (position >> a.view.page_shift)]));
    p.slot = static_cast<uint32_t>(position) & ((1u << a.view.page_shift) - 1);
    p.there = p.page < static_cast<uint32_t>(a.view.pages);
  }
  return !kWrite || p.there;
}

// The rows of one side, a few heads at a time: `row(head, active)` for this lane's.
template <typename F>
__device__ __forceinline__ void each_row(const Side& s, const Place& p, F row) {
  const int lane = static_cast<int>(threadIdx.x) & 63, heads = kWave >> s.lanes_log2;
  for (int h = p.head; h < p.end; h += heads) row(h + (lane >> s.lanes_log2), h + (lane >> s.lanes_log2) < p.end);
}
__device__ __forceinline__ int64_t pool_offset(const PagedPool& pool, const Place& p, int head) {
  return p.page * pool.page + static_cast<int64_t>(p.slot) * pool.slot + static_cast<int64_t>(head) * pool.head;
}
__device__ __forceinline__ int64_t exponent_offset(const PagedPool& pool, const Place& p, int head) {
  return p.page * pool.ePage + static_cast<int64_t>(p.slot) * pool.eSlot + static_cast<int64_t>(head) * pool.eHead;
}

// the greater of each half's 16-bit magnitudes; with kFinite those of infinities and NaN count as zero
template <int DT, bool kFinite>
__device__ __forceinline__ uint32_t greater_magnitudes(uint32_t a, uint32_t w) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  w &= 0x7fff7fffu;
  if constexpr (kFinite) {
    constexpr uint32_t top = DT == MEGA_BF16 ? 0x7f80u : 0x7c00u;
    w = ((w & 0xffffu) >= top ? 0u : w & 0xffffu) | ((w >> 16) >= top ? 0u : w & 0xffff0000u);
  }
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, w)));
}
// a row's greatest magnitude, in all of its lanes (bit patterns of non-negative numbers are ordered as the numbers are)
template <int DT, bool kFinite>
__device__ __forceinline__ uint32_t row_top(const uint4 (&x)[kPieces], int lanes) {
  uint32_t both = 0;
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    both = greater_magnitudes<DT, kFinite>(greater_magnitudes<DT, kFinite>(both, x[i].x), x[i].y);
    both = greater_magnitudes<DT, kFinite>(greater_magnitudes<DT, kFinite>(both, x[i].z), x[i].w);
  }
  uint32_t top = max(both & 0xffffu, both >> 16);
  for (int off = 1; off < lanes; off <<= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), off, 64)));
  return top;
}

template <int DT, bool kEight>
__device__ __forceinline__ void write_rows(const Side& s, const Place& p) {
  const int l = (static_cast<int>(threadIdx.x) & (s.lanes - 1)) * 8, stride = s.lanes * 8, width = s.pool.width;
  each_row(s, p, [&](int head, bool active) {
    const uint16_t* from = static_cast<const uint16_t*>(s.rows) + p.token * s.row + head * s.head;
    const int mine = active ? width : 0;
    uint4 x[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      x[i] = make_uint4(0, 0, 0, 0);
      if (l + i * stride < mine) x[i] = *reinterpret_cast<const uint4*>(from + l + i * stride);
    }
    if constexpr (!kEight) {
      uint16_t* to = static_cast<uint16_t*>(s.pool.rows) + pool_offset(s.pool, p, head);
#pragma unroll
      for (int i = 0; i < kPieces; ++i)
        if (l + i * stride < mine) *reinterpret_cast<uint4*>(to + l + i * stride) = x[i];
    } else {
      uint32_t top = row_top<DT, false>(x, s.lanes);
      const bool odd = __any(top >= (DT == MEGA_BF16 ? 0x7f80u : 0x7c00u));  // (some row has an infinity or NaN)
      if (odd) top = row_top<DT, true>(x, s.lanes);
      int e = 0;
      if (top != 0) {
        int power;
        const float fraction = frexpf(DT == MEGA_BF16 ? bf16_bits_to_float(top) : f16_bits_to_float(top), &power);
        e = max(fraction > 0.875f ? power - 8 : power - 9, -126);
      }
      const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
      // 256 2^e is twice the type's greatest power of two: a magnitude that would round to it stays at 240
      const bool edge = e == (DT == MEGA_BF16 ? 120 : 8);
      const float limit = edge ? 240.f : 448.f;
      const bool plain = !odd && !__any(edge);
      uint8_t* to = static_cast<uint8_t*>(s.pool.rows) + pool_offset(s.pool, p, head);
#pragma unroll
      for (int i = 0; i < kPieces; ++i)
        if (l + i * stride < mine) {
          float v[8];
          unpack8<DT>(x[i], v);
          int code[2] = {0, 0};
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float y = v[j] * down;
            v[j] = plain ? y : fabsf(v[j]) < __builtin_inff() ? fminf(fmaxf(y, -limit), limit) : __builtin_nanf("");
          }
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            code[j] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * j], v[4 * j + 1], 0, false);
            code[j] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * j + 2], v[4 * j + 3], code[j], true);
          }
          *reinterpret_cast<uint2*>(to + l + i * stride) = make_uint2(static_cast<uint32_t>(code[0]), static_cast<uint32_t>(code[1]));
        }
      if (l == 0 && active) s.pool.exponents[exponent_offset(s.pool, p, head)] = static_cast<uint8_t>(e + 127);
    }
  });
}

template <int DT, bool kEight>
__global__ __launch_bounds__(kThreads) void paged_write_kernel(CacheArgs a) {
  Place p;
  if (!find_place<true>(a, p)) return;
  if (p.values) write_rows<DT, kEight>(a.side[1], p);
  if (p.keys) write_rows<DT, kEight>(a.side[0], p);
}

template <int DT, bool kEight>
__device__ __forceinline__ void read_rows(const Side& s, const Place& p) {
  const int l = (static_cast<int>(threadIdx.x) & (s.lanes - 1)) * 8, stride = s.lanes * 8, width = s.pool.width;
  each_row(s, p, [&](int head, bool active) {
    uint16_t* to = static_cast<uint16_t*>(s.rows) + p.token * s.row + head * s.head;
    const int mine = active ? width : 0, stored = p.there ? mine : 0;
    float scale = 0.f;
    if (kEight && stored > 0) scale = exponent_value(s.pool.exponents[exponent_offset(s.pool, p, head)]);
    uint4 x[kPieces];
    const int64_t from = pool_offset(s.pool, p, head);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      x[i] = make_uint4(0, 0, 0, 0);
      if (l + i * stride < stored) {
        if (kEight) {
          const uint2 c = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(s.pool.rows) + from + l + i * stride);
          x[i].x = c.x, x[i].y = c.y;
        } else {
          x[i] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(s.pool.rows) + from + l + i * stride);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kPieces; ++i)
      if (l + i * stride < mine) {
        if (kEight)
          x[i] = make_uint4(widen<DT, false>(x[i].x, scale), widen<DT, true>(x[i].x, scale), widen<DT, false>(x[i].y, scale),
                            widen<DT, true>(x[i].y, scale));
        *reinterpret_cast<uint4*>(to + l + i * stride) = x[i];
      }
  });
}

template <int DT, bool kEight>
__global__ __launch_bounds__(kThreads) void paged_read_kernel(CacheArgs a) {
  Place p;
  if (!find_place<false>(a, p)) return;
  if (p.values) read_rows<DT, kEight>(a.side[1], p);
  if (p.keys) read_rows<DT, kEight>(a.side[0], p);
}

// lanes to a row: as few as take it in one piece each, 16 at the least
void split_row(Side& s) {
  s.lanes = 16, s.lanes_log2 = 4;
  while (s.lanes < kWave && s.lanes * 8 < s.pool.width) s.lanes *= 2, ++s.lanes_log2;
}
// all heads of a token to a wave where that leaves waves enough (sixteen to a CU), fewer where it does not
void split_heads(CacheArgs& a) {
  constexpr int64_t kEnough = 256 * 16;
  a.shares = static_cast<int32_t>(std::clamp<int64_t>(kEnough / a.rows, 1, a.heads));
  a.at_once = (a.heads + a.shares - 1) / a.shares;
  a.shares = (a.heads + a.at_once - 1) / a.at_once;
  a.apart = static_cast<int64_t>(a.rows) * a.shares < kEnough;
}

template <typename K>
int launch(K kernel, CacheArgs& a, void* stream) {
  split_row(a.side[0]), split_row(a.side[1]);
  split_heads(a);
  const int64_t groups = ((static_cast<int64_t>(a.rows) * a.shares << a.apart) + kWaves - 1) / kWaves;
  kernel<<<grid_of(groups), dim3(kThreads), 0, static_cast<hipStream_t>(stream)>>>(a);
  MEGA_CHECK_LAUNCH();
  return MEGA_OK;
}

// A pool's places, in bytes: rows of `width` at base + i stride[0] + j stride[1] + ..., axes of one entry left out, the largest stride first.
struct Places {
  uintptr_t base;
  int64_t stride[3], count[3], width;
  int axes;
  // bytes from the first row's begin to the last one's end, over the axes behind the first `from`
  int64_t span(int from) const {
    constexpr int64_t kAll = int64_t{1} << 60;  // (more than there are addresses)
    int64_t n = width, step;
    for (int i = from; i < axes; ++i)
      if (__builtin_mul_overflow(count[i] - 1, stride[i], &step) || step >= kAll - n) return kAll;
      else n += step;
    return n;
  }
};
Places places_of(const mega_paged_cache* c, const void* base, const int64_t* stride, int64_t width, int64_t bytes) {
  Places p{reinterpret_cast<uintptr_t>(base), {}, {}, width * bytes, 0};
  const int64_t count[3] = {c->pages, c->page_size, c->heads};
  for (int i = 0; i < 3; ++i) {
    if (count[i] == 1) continue;
    int at = p.axes++;
    for (; at > 0 && p.stride[at - 1] < stride[i] * bytes; --at) p.stride[at] = p.stride[at - 1], p.count[at] = p.count[at - 1];
    p.stride[at] = stride[i] * bytes, p.count[at] = count[i];
  }
  return p;
}
// Whether two rows of a pool may share memory: an axis steps over all that lies behind it, or they may.
bool rows_meet(const Places& p) {
  for (int i = 0; i < p.axes; ++i)
    if (p.stride[i] < p.span(i + 1)) return true;
  return false;
}
// Whether a row of a and one of b, which begins `ahead` bytes behind a, may share memory: axis by axis, as long as their strides agree.
bool places_meet(const Places& a, const Places& b, int64_t ahead, int axis = 0) {
  if (ahead >= a.span(axis) || ahead + b.span(axis) <= 0) return false;
  if (axis == a.axes || axis == b.axes || a.stride[axis] != b.stride[axis]) return true;
  const int64_t stride = a.stride[axis], inner_a = a.span(axis + 1), inner_b = b.span(axis + 1);
  if (inner_a > stride || inner_b > stride) return true;
  // steps d with -inner_b < ahead + d stride < inner_a, three at the most
  const auto floor_div = [&](int64_t n) { return n / stride - (n % stride < 0); };
  const int64_t low = std::max(floor_div(-inner_b - ahead) + 1, 1 - a.count[axis]), high = std::min(floor_div(inner_a - ahead - 1), b.count[axis] - 1);
  for (int64_t d = low; d <= high; ++d)
    if (places_meet(a, b, ahead + d * stride, axis + 1)) return true;
  return false;
}
// Rows that are written at once must not share memory: not two of a pool, nor one of a pool with one of another.
bool pools_meet(const mega_paged_cache* c) {
  const bool eight = c->k_exponents != nullptr;
  const Places p[4] = {places_of(c, c->k, c->k_stride, c->k_width, eight ? 1 : 2), places_of(c, c->v, c->v_stride, c->v_width, eight ? 1 : 2),
                       places_of(c, c->k_exponents, c->ke_stride, 1, 1), places_of(c, c->v_exponents, c->ve_stride, 1, 1)};
  for (int i = 0; i < (eight ? 4 : 2); ++i) {
    if (rows_meet(p[i])) return true;
    for (int j = 0; j < i; ++j)
      if (places_meet(p[i], p[j], static_cast<int64_t>(p[j].base) - static_cast<int64_t>(p[i].base))) return true;
  }
  return false;
}

bool unaligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; }

}  // namespace

int check_paged_cache(const mega_paged_cache* c, int dtype, const char* who) {
  MEGA_CHECK_ARG(c != nullptr, "%s: null cache", who);
  MEGA_CHECK_ARG(dtype == MEGA_BF16 || dtype == MEGA_F16, "%s: dtype must be MEGA_BF16 or MEGA_F16", who);
  MEGA_CHECK_ARG(c->batch >= 0 && c->batch <= 0x7fffffff && c->heads >= 1 && c->heads <= 65536, "%s: bad batch or heads", who);
  MEGA_CHECK_ARG(c->page_size >= kMinPage && c->page_size <= kMaxPage && (c->page_size & (c->page_size - 1)) == 0,
                 "%s: page_size must be a power of two, 16 .. 65536", who);
  MEGA_CHECK_ARG(c->pages >= 1 && c->pages <= 0x7fffffff, "%s: bad number of pages", who);
  MEGA_CHECK_ARG(c->table_width >= 0 && c->table_width * c->page_size <= 0x40000000 && c->table_stride >= 0,
                 "%s: a row of the table holds up to 2^30 positions", who);
  for (const int64_t w : {c->k_width, c->v_width})
    MEGA_CHECK_ARG(w >= 16 && w <= kMaxCacheWidth && w % 16 == 0, "%s: widths must be multiples of 16, 16 .. 4096", who);
  MEGA_CHECK_ARG(c->k != nullptr && c->v != nullptr && (c->table != nullptr || c->batch == 0 || c->table_width == 0), "%s: null pointer", who);
  MEGA_CHECK_ARG((c->k_exponents == nullptr) == (c->v_exponents == nullptr), "%s: exponents of keys and values go together", who);
  MEGA_CHECK_ARG(!unaligned(c->k) && !unaligned(c->v), "%s: pools must be 16-byte aligned", who);
  // (offsets inside a page are 32-bit numbers)
  const auto fits = [&](const int64_t* st, int64_t unit) {
    for (int i = 0; i < 3; ++i)
      if (st[i] < 0 || st[i] % unit != 0 || st[i] > (int64_t{1} << 40)) return false;
    return st[1] <= 0x3fffffff / c->page_size && st[2] <= 0x7fffffff;
  };
  MEGA_CHECK_ARG(fits(c->k_stride, 16) && fits(c->v_stride, 16), "%s: pool strides must be multiples of 16 elements, a page's positions within 2^30", who);
  MEGA_CHECK_ARG(c->k_exponents == nullptr || (fits(c->ke_stride, 1) && fits(c->ve_stride, 1)), "%s: bad exponent strides", who);
  return MEGA_OK;
}

PagedView paged_view(const mega_paged_cache* c) {
  PagedView v{c->table, c->table_stride, static_cast<int32_t>(c->table_width), static_cast<int32_t>(c->batch), static_cast<int32_t>(c->pages), 0};
  while ((int64_t{1} << v.page_shift) < c->page_size) ++v.page_shift;
  return v;
}

PagedPool paged_pool(const mega_paged_cache* c, bool values) {
  const int64_t *st = values ? c->v_stride : c->k_stride, *est = values ? c->ve_stride : c->ke_stride;
  PagedPool p{values ? c->v : c->k, values ? c->v_exponents : c->k_exponents, st[0], 0, static_cast<int32_t>(st[1]), static_cast<int32_t>(st[2]), 0, 0,
              static_cast<int32_t>(values ? c->v_width : c->k_width)};
  if (p.exponents != nullptr) p.ePage = est[0], p.eSlot = static_cast<int32_t>(est[1]), p.eHead = static_cast<int32_t>(est[2]);
  return p;
}

}  // namespace mega

using namespace mega;

extern "C" int mega_paged_cache_write(const mega_paged_cache* cache, int dtype, const void* k_new, int64_t k_row, int64_t k_head,
                                      const void* v_new, int64_t v_row, int64_t v_head, const int32_t* lengths, const int32_t* cu,
                                      int64_t rows, void* stream) {
  if (const int rc = check_paged_cache(cache, dtype, "mega_paged_cache_write"); rc != MEGA_OK) return rc;
  MEGA_CHECK_ARG(rows >= 0 && rows <= 0x7fffffff, "mega_paged_cache_write: bad number of rows");
  MEGA_CHECK_ARG(!pools_meet(cache), "mega_paged_cache_write: the places of the pools must not share memory");
  if (rows == 0 || cache->batch == 0) return MEGA_OK;
  MEGA_CHECK_ARG(k_new != nullptr && v_new != nullptr && lengths != nullptr && cu != nullptr, "mega_paged_cache_write: null pointer");
  MEGA_CHECK_ARG(!unaligned(k_new) && !unaligned(v_new) && k_row % 8 == 0 && k_head % 8 == 0 && v_row % 8 == 0 && v_head % 8 == 0,
                 "mega_paged_cache_write: new rows must be 16-byte aligned");
  CacheArgs a{paged_view(cache), {{paged_pool(cache, false), const_cast<void*>(k_new), k_row, k_head, 0, 0},
                                  {paged_pool(cache, true), const_cast<void*>(v_new), v_row, v_head, 0, 0}},
              lengths, cu, static_cast<int32_t>(rows), static_cast<int32_t>(cache->heads), 0, 0, 0, 0};
  const bool eight = cache->k_exponents != nullptr;
  if (dtype == MEGA_BF16)
    return eight ? launch(paged_write_kernel<MEGA_BF16, true>, a, stream) : launch(paged_write_kernel<MEGA_BF16, false>, a, stream);
  // (a copy does not look at its elements: one kernel for both types)
  return eight ? launch(paged_write_kernel<MEGA_F16, true>, a, stream) : launch(paged_write_kernel<MEGA_BF16, false>, a, stream);
}

extern "C" int mega_paged_cache_read(const mega_paged_cache* cache, int dtype, const int32_t* begins, const int32_t* cu, int64_t rows,
                                     void* k_out, void* v_out, int clear_rest, void* stream) {
  if (const int rc = check_paged_cache(cache, dtype, "mega_paged_cache_read"); rc != MEGA_OK) return rc;
  MEGA_CHECK_ARG(rows >= 0 && rows <= 0x7fffffff, "mega_paged_cache_read: bad number of rows");
  if (rows == 0) return MEGA_OK;
  MEGA_CHECK_ARG(cache->batch >= 1, "mega_paged_cache_read: rows of no sequence");
  MEGA_CHECK_ARG(k_out != nullptr && v_out != nullptr && begins != nullptr && cu != nullptr, "mega_paged_cache_read: null pointer");
  MEGA_CHECK_ARG(!unaligned(k_out) && !unaligned(v_out), "mega_paged_cache_read: outputs must be 16-byte aligned");
  const int64_t H = cache->heads;
  CacheArgs a{paged_view(cache), {{paged_pool(cache, false), k_out, H * cache->k_width, cache->k_width, 0, 0},
                                  {paged_pool(cache, true), v_out, H * cache->v_width, cache->v_width, 0, 0}},
              begins, cu, static_cast<int32_t>(rows), static_cast<int32_t>(H), 0, 0, 0, clear_rest != 0};
  const bool eight = cache->k_exponents != nullptr;
  if (dtype == MEGA_BF16)
    return eight ? launch(paged_read_kernel<MEGA_BF16, true>, a, stream) : launch(paged_read_kernel<MEGA_BF16, false>, a, stream);
  return eight ? launch(paged_read_kernel<MEGA_F16, true>, a, stream) : launch(paged_read_kernel<MEGA_BF16, false>, a, stream);
}
