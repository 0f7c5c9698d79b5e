// What the kernels of the paged key / value cache share: the pool's layout, the way from a row to its
// sequence and from a position to its page, and the host's checks.
#pragma once

#include "common.hpp"

namespace mega {

constexpr int kMinPage = 16, kMaxPage = 65536;  // (16: a lane group of the attention's key tile never leaves its page)
constexpr int kMaxCacheWidth = 4096;

// The pool as a kernel sees it.  Strides in elements.
struct PagedView {
  const int32_t* table;
  int64_t table_stride;
  int32_t table_width, batch, pages, page_shift;
};
struct PagedPool {
  void* rows;
  uint8_t* exponents;  // null: 16 bits
  int64_t page, ePage;
  int32_t slot, head, eSlot, eHead;
  int32_t width;
};

// The largest i of 0 .. n - 1 with f(i) <= x, for a non-decreasing f with f(0) <= x, found by all lanes of a wave
// together: 64 probes a round, so one load for up to 64 sequences and two for up to 4096.
template <typename F>
__device__ __forceinline__ int last_not_above(int n, int64_t x, F f) {
  const int lane = static_cast<int>(threadIdx.x) & 63;
  int low = 0;
  while (n > 1) {
    const int step = (n + 63) >> 6, i = lane * step;
    const uint64_t below = __ballot(i < n && f(low + i) <= x);
    const int c = below == 0 ? 0 : static_cast<int>(__popcll(below)) - 1;
    low += c * step;
    n = min(step, n - c * step);
  }
  return __builtin_amdgcn_readfirstlane(low);
}

// A launch has fewer than 2^32 threads along an axis (of more, those past a multiple of 2^32 run and no error says so): groups in lines of 2^22,
// of up to 512 threads each.  The last line has numbers behind the last group's.
constexpr int64_t kLine = 1 << 22;
inline dim3 grid_of(int64_t groups) { return dim3(static_cast<uint32_t>(groups < kLine ? groups : kLine), static_cast<uint32_t>((groups + kLine - 1) / kLine)); }
__device__ __forceinline__ uint32_t group_number() { return blockIdx.y * static_cast<uint32_t>(kLine) + blockIdx.x; }

// row numbers that `cu` gives, kept inside the operand whatever it holds
__device__ __forceinline__ int row_bound(const int32_t* cu, int i, int rows) { return min(max(cu[i], 0), rows); }

// 2^(e - 127) of an exponent byte 1 .. 254
__device__ __forceinline__ float exponent_value(uint32_t e) { return __uint_as_float(e << 23); }
// two e4m3 codes of a word's lower or upper half times a power of two, as 16-bit numbers
template <int DT, bool kUpper>
__device__ __forceinline__ uint32_t widen(uint32_t codes, float scale) {
  if constexpr (DT == MEGA_BF16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, kUpper));
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, kUpper));
}

// The host's half: MEGA_OK, or the error with its message.
int check_paged_cache(const mega_paged_cache* c, int dtype, const char* who);
PagedView paged_view(const mega_paged_cache* c);
PagedPool paged_pool(const mega_paged_cache* c, bool values);

}  // namespace mega
