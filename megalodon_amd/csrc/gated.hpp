// The gated product between its entry points (gated_linear.hip) and the tiles that it runs in (attention.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mega {

// h = silu(x w1^T) o (x w3^T) in tiles, and the two products where a and b are given; tokens * n_in and n_out * n_in below 2^30, n_in a
// multiple of 64, rows of x, w1 and w3 on 16-byte boundaries.  parts: gated_parts_bytes, or null
int gated_product(int dtype, const uint16_t* x, const uint16_t* w1, const uint16_t* w3, int64_t tokens, int64_t n_in, int64_t n_out,
                  uint16_t* h, uint16_t* a, uint16_t* b, float* parts, hipStream_t s);
int64_t gated_parts_bytes(int64_t tokens, int64_t n_in, int64_t n_out);

}  // namespace mega
