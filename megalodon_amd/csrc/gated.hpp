// The gated product between its entry points (gated_linear.hip) and the tiles that it runs in (gated_tiles.hip, attention.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mega {

#ifdef __HIP_DEVICE_COMPILE__
// 1 / (1 + exp(-a)) in two transcendental instructions (each within a unit in the last place; 2^x of a product: |a| 2^-24 more), where the
// IEEE division and the scaled exponential take eighteen instructions an element (8192 tokens, 4096 -> 11008 1105 -> 1084 us).
// exp(-a) that overflows gives 0, one that vanishes 1.
__device__ __forceinline__ float fast_sigmoid(float a) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504088896340736f * a));
}
#else
__device__ float fast_sigmoid(float a);
#endif

// h = silu(x w1^T) o (x w3^T), and the two products where they are kept (a and b; null: they are not); tokens * n_in and n_out * n_in
// below 2^30, n_in a multiple of 64, rows of x, w1 and w3 on 16-byte boundaries.
// Rows of a and b are `pitch` elements apart, n_out rounded up to 8; what lies behind n_out is of no meaning.
// Tiles 0 .. tiles - 1 of 256 tokens x 128 features, in bands of eight columns of tiles, row by row in each.
struct GatedTiles {
  const uint16_t *x, *w1, *w3;
  uint16_t* h;
  void *a, *b;
  int tokens, n_in, n_out, pitch, row_tiles, col_tiles, tiles;
};
int gated_tiles(int dtype, int keep, const GatedTiles& p, int grid, hipStream_t s);

// parts: gated_parts_bytes, or null; wide: a and b in float32
int gated_product(int dtype, const uint16_t* x, const uint16_t* w1, const uint16_t* w3, int64_t tokens, int64_t n_in, int64_t n_out,
                  uint16_t* h, void* a, void* b, bool wide, float* parts, hipStream_t s);
__host__ __device__ inline int64_t gated_pitch(int64_t n_out) { return (n_out + 7) / 8 * 8; }
int64_t gated_parts_bytes(int64_t tokens, int64_t n_in, int64_t n_out);

}  // namespace mega
