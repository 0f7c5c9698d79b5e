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

// A launch of gated_tiles.hip: C (m, n) of operands A and B along k, as its modes read them.
struct GatedTiles {
  const uint16_t *a, *b, *b2;
  uint32_t a_bytes, b_bytes;  // where the operands end
  int m, n, k, lda, ldb;
  int seg;                    // kInput: slabs of 64 features of b, those behind them are b2's
  uint16_t *c, *c2;           // (kWeight: the gradient of w1 or of the only matrix, of w3)
  void *kept_a, *kept_b;      // kGate: rows of `pitch` elements, n rounded up to 8; what lies behind n is of no meaning
  int pitch;
  int cols, half, n_out;      // kInput, kWeight: columns of c; kWeight: columns of a half of A, rows of c
  float* sum;                 // kWeight of more tokens than a launch takes: the sums so far, rows of c, then of c2; null: one launch
  int first, last;            // kWeight: of the launches: nothing is in the sums yet; c is written, and not the sums
  int row_tiles, col_tiles;
  int full, left, cut;        // tiles as a whole, then some whose slabs are cut into `cut` pieces, which go to parts
  float* parts;
};
// Operands of fewer than 2^30 elements on 16-byte boundaries; parts: gated_tiles_bytes (kind: 0, 1, 2 as they stand here), or null for none.
// h = silu(x w1^T) o (x w3^T); a and b may be null; n_in a multiple of 8
int gated_tiles(int dtype, const uint16_t* x, const uint16_t* w1, const uint16_t* w3, int64_t tokens, int64_t n_in, int64_t n_out,
                uint16_t* h, void* a, void* b, bool wide, float* parts, hipStream_t s);
// g (tokens, terms, 2 half), half n_out rounded up to 64: the gradients of a and, from column half on, of b, zeros behind n_out, as sums of one or two
// terms (two: up to 64 tokens); for dw each row of x stands there `terms` times.  Rows of x, w1, w3 `ld` elements apart, a multiple of 8.
// dx (tokens, n_in), dw1 and dw3 (n_out, n_in), one of them or both, of any pitch; sums: of more tokens than a launch takes, (1 or 2, n_out, n_in)
// numbers that go from the first launch to the last, which writes dw1 and dw3; or null
int gated_tiles_input(int dtype, const uint16_t* g, const uint16_t* w1, const uint16_t* w3, int64_t tokens, int64_t n_in, int64_t n_out, int64_t ld,
                      int terms, uint16_t* dx, float* parts, hipStream_t s);
int gated_tiles_weight(int dtype, const uint16_t* g, const uint16_t* x, int64_t tokens, int64_t n_in, int64_t n_out, int64_t ld,
                       int terms, uint16_t* dw1, uint16_t* dw3, float* sums, bool first, bool last, float* parts, hipStream_t s);
int64_t gated_tiles_bytes(int kind, int64_t tokens, int64_t n_in, int64_t n_out, int matrices = 2, int terms = 1);

// parts: gated_parts_bytes, or null; wide: a and b in float32
int gated_product(int dtype, const uint16_t* x, const uint16_t* w1, const uint16_t* w3, int64_t tokens, int64_t n_in, int64_t n_out,
                  uint16_t* h, void* a, void* b, bool wide, float* parts, hipStream_t s);
__host__ __device__ inline int64_t gated_pitch(int64_t n_out) { return (n_out + 7) / 8 * 8; }
int64_t gated_parts_bytes(int64_t tokens, int64_t n_in, int64_t n_out);

}  // namespace mega
