// The gated half of a feed-forward network for gfx950 (bfloat16 / float16 rows, float32 inside):
//   a = x w1^T, b = x w3^T, h = a sigma(a) b                       (x: tokens x n_in, w1, w3: n_out x n_in)
//   da = dh b sigma(a) (1 + a (1 - sigma(a))), db = dh a sigma(a)
//   dx = da w1 + db w3, dw1 = da^T x, dw3 = db^T x
// One kernel has both projections: a wave's accumulators hold a and b of the same elements, and the gate is taken from them
// in float32, so that neither product goes through memory (training keeps both, rounded, for the backward: 4 bytes an element
// where float32 would be 8; the gradients that come of them are rounded to 16 bits for the matrix cores anyway).
//
// Many tokens: the product kernels of attention.hip with a gate for an epilogue (gated_product).  Few: the weights' stream from memory is all
// the time there is, and the kernel below reads them once, straight into the operand registers of the matrix cores.
#include "common.hpp"
#include "gated.hpp"

#include <algorithm>

namespace mega {

// dw (n_out, n_in) = dy^T x + add; sizes as mega_linear_weight_grads takes them (attention.hip)
int weight_grad_onto(int dtype, const uint16_t* dy, const uint16_t* x, int64_t tokens, int64_t n_in, int64_t n_out, const uint16_t* add,
                     uint16_t* dw, float* parts, hipStream_t s);

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <int DT>
__device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (DT == MEGA_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ float sigmoidf(float a) { return 1.f / (1.f + __expf(-a)); }

// ---- few tokens -------------------------------------------------------------------------------------
// A workgroup has 16 features of both matrices and all of the tokens (NT blocks of 16); its waves have equal runs of k and meet in
// LDS, in their order.  A product of 16 features x 16 tokens x 32 k: lane l holds 8 k of feature l % 16 and 8 k of token l % 16,
// k = 32 step + 8 (l / 16), so that both come from memory as they are, 64 bytes of a row to four lanes.  It gives lane l
// token l % 16 of features 4 (l / 16) .. + 3.
// Rows behind the last feature or token are the last one again, never stored.  WHOLE: rows are whole 16-byte pieces.
constexpr int kFewTokens = 64, kFewWaves = 8;

struct FewParams {
  const uint16_t *x, *w1, *w3;
  uint16_t *h, *a, *b;
  int tokens, n_in, n_out;
};

template <bool WHOLE>
__device__ __forceinline__ u32x4 eight(const uint16_t* row, int k, int n) {
  if (k + 8 <= n) {
    if constexpr (WHOLE) return *reinterpret_cast<const u32x4*>(row + k);
    else return __builtin_bit_cast(u32x4, *reinterpret_cast<const u32x4_any*>(row + k));
  }
  uint32_t e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = k + i < n ? row[k + i] : 0u;
  return u32x4{e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16};
}

template <int DT, int NT, bool WHOLE>
__global__ __launch_bounds__(kFewWaves * kWave) void gated_few_kernel(const FewParams p) {
  __shared__ f32x4 sums[kFewWaves][2 * NT][kWave];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, r = lane % 16, g = lane / 16;
  const int f0 = blockIdx.x * 16;
  const int64_t feature = static_cast<int64_t>(min(f0 + r, p.n_out - 1)) * p.n_in;
  const uint16_t *w1 = p.w1 + feature, *w3 = p.w3 + feature;
  const uint16_t* x[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) x[t] = p.x + static_cast<int64_t>(min(16 * t + r, p.tokens - 1)) * p.n_in;
  f32x4 acc[2][NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[0][t] = acc[1][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int steps = (p.n_in + 31) / 32, lo = steps * wave / kFewWaves, hi = steps * (wave + 1) / kFewWaves;
  constexpr int U = NT > 2 ? 2 : 4;  // steps whose operands are asked for together
  int s = lo;
  for (; s + U <= hi && 32 * (s + U) <= p.n_in; s += U) {
    u32x4 a[U], b[U], v[U][NT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = 32 * (s + u) + 8 * g;
      a[u] = eight<WHOLE>(w1, k, 0x7fffffff);
      b[u] = eight<WHOLE>(w3, k, 0x7fffffff);
#pragma unroll
      for (int t = 0; t < NT; ++t) v[u][t] = eight<WHOLE>(x[t], k, 0x7fffffff);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        acc[0][t] = mma16<DT>(a[u], v[u][t], acc[0][t]);
        acc[1][t] = mma16<DT>(b[u], v[u][t], acc[1][t]);
      }
  }
  for (; s < hi; ++s) {
    const int k = 32 * s + 8 * g;
    const u32x4 a = eight<WHOLE>(w1, k, p.n_in), b = eight<WHOLE>(w3, k, p.n_in);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const u32x4 v = eight<WHOLE>(x[t], k, p.n_in);
      acc[0][t] = mma16<DT>(a, v, acc[0][t]);
      acc[1][t] = mma16<DT>(b, v, acc[1][t]);
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) sums[wave][t][lane] = acc[0][t], sums[wave][NT + t][lane] = acc[1][t];
  __syncthreads();
  if (wave >= NT) return;
  const int token = 16 * wave + r, f = f0 + 4 * g;
  f32x4 a = sums[0][wave][lane], b = sums[0][NT + wave][lane];
#pragma unroll
  for (int w = 1; w < kFewWaves; ++w) a += sums[w][wave][lane], b += sums[w][NT + wave][lane];
  if (token >= p.tokens) return;
  const int64_t at = static_cast<int64_t>(token) * p.n_out + f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (f + e >= p.n_out) break;
    Elem<DT>::store(p.h + at + e, a[e] * sigmoidf(a[e]) * b[e]);
    if (p.a != nullptr) Elem<DT>::store(p.a + at + e, a[e]), Elem<DT>::store(p.b + at + e, b[e]);
  }
}

template <int DT>
int launch_few(const FewParams& p, hipStream_t s) {
  const dim3 grid((p.n_out + 15) / 16), block(kFewWaves * kWave);
  const bool whole = p.n_in % 8 == 0;
#define MEGA_FEW(NT)                                                              \
  (whole ? gated_few_kernel<DT, NT, true><<<grid, block, 0, s>>>(p) : gated_few_kernel<DT, NT, false><<<grid, block, 0, s>>>(p))
  if (p.tokens <= 16) MEGA_FEW(1);
  else if (p.tokens <= 32) MEGA_FEW(2);
  else MEGA_FEW(4);
#undef MEGA_FEW
  MEGA_CHECK_LAUNCH();
  return MEGA_OK;
}

// ---- rows of whole 16-byte pieces, and back -----------------------------------------------------------
constexpr int kThreads = 256;

// dst (rows, to) = src (rows, from), zeros behind column `from`; `to` a multiple of 8, dst on 16-byte boundaries
__global__ __launch_bounds__(kThreads) void widen_kernel(const uint16_t* src, uint16_t* dst, int64_t rows, int from, int to) {
  const int64_t pieces = rows * (to / 8);
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < pieces; i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t row = i / (to / 8);
    const int k = static_cast<int>(i % (to / 8)) * 8;
    *reinterpret_cast<u32x4*>(dst + 8 * i) = eight<false>(src + row * from, k, from);
  }
}
// dst (rows, to) = the first columns of src (rows, from); `from` a multiple of 8
__global__ __launch_bounds__(kThreads) void narrow_kernel(const uint16_t* src, uint16_t* dst, int64_t rows, int from, int to) {
  const int64_t pieces = rows * (from / 8);
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < pieces; i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t row = i / (from / 8);
    const int k = static_cast<int>(i % (from / 8)) * 8;
    const u32x4 v = *reinterpret_cast<const u32x4*>(src + 8 * i);
    uint16_t* const to_row = dst + row * to;
    if (k + 8 <= to) {
      *reinterpret_cast<u32x4_any*>(to_row + k) = __builtin_bit_cast(u32x4_any, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (k + e < to) to_row[k + e] = static_cast<uint16_t>(v[e / 2] >> (16 * (e % 2)));
    }
  }
}
unsigned pieces_grid(int64_t pieces) { return static_cast<unsigned>(std::min<int64_t>((pieces + kThreads - 1) / kThreads, 16384)); }
int widen(const uint16_t* src, uint16_t* dst, int64_t rows, int64_t from, int64_t to, hipStream_t s) {
  widen_kernel<<<pieces_grid(rows * (to / 8)), kThreads, 0, s>>>(src, dst, rows, static_cast<int>(from), static_cast<int>(to));
  MEGA_CHECK_LAUNCH();
  return MEGA_OK;
}
int narrow(const uint16_t* src, uint16_t* dst, int64_t rows, int64_t from, int64_t to, hipStream_t s) {
  narrow_kernel<<<pieces_grid(rows * (from / 8)), kThreads, 0, s>>>(src, dst, rows, static_cast<int>(from), static_cast<int>(to));
  MEGA_CHECK_LAUNCH();
  return MEGA_OK;
}

// ---- the gate's backward --------------------------------------------------------------------------------
// da, db (tokens, ld) from dh, a, b (tokens, n): 8 elements a thread, zeros from column n to `to`
template <int DT>
__global__ __launch_bounds__(kThreads) void gate_grad_kernel(const uint16_t* dh, const uint16_t* a, const uint16_t* b, uint16_t* da, uint16_t* db,
                                                            int64_t tokens, int n, int to, int64_t ld) {
  const int64_t pieces = tokens * (to / 8);
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < pieces; i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t row = i / (to / 8);
    const int k = static_cast<int>(i % (to / 8)) * 8;
    float g[8], u[8], v[8], du[8], dv[8];
    unpack8<DT>(__builtin_bit_cast(uint4, eight<false>(dh + row * n, k, n)), g);
    unpack8<DT>(__builtin_bit_cast(uint4, eight<false>(a + row * n, k, n)), u);
    unpack8<DT>(__builtin_bit_cast(uint4, eight<false>(b + row * n, k, n)), v);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float s = sigmoidf(u[e]);
      dv[e] = g[e] * u[e] * s;
      du[e] = g[e] * v[e] * s * (1.f + u[e] * (1.f - s));
    }
    *reinterpret_cast<uint4*>(da + row * ld + k) = pack8<DT>(du);
    *reinterpret_cast<uint4*>(db + row * ld + k) = pack8<DT>(dv);
  }
}

// ---- sizes ----------------------------------------------------------------------------------------------
int64_t up(int64_t n, int64_t step) { return (n + step - 1) / step * step; }
constexpr int64_t kMost = 1ll << 30;  // elements of an operand: the product kernels' byte offsets have 32 bits

// What a call lays out in its workspace, in bytes from its start (0 bytes where a piece is not needed).
struct Room {
  int64_t bytes = 0;
  int64_t take(int64_t n) {
    const int64_t at = bytes;
    bytes += up(n, 256);
    return at;
  }
};
struct Forward {
  int64_t k, rows;  // n_in with its padding, tokens of a launch
  int64_t x, w1, w3, parts, bytes;
  Forward(int64_t tokens, int64_t n_in, int64_t n_out) {
    Room room;
    k = n_in, rows = tokens, x = w1 = w3 = parts = 0;
    if (tokens > kFewTokens) {
      k = up(n_in, 64);
      rows = std::min(tokens, std::max<int64_t>((kMost - 1) / k / 256 * 256, 256));
      if (k != n_in) {
        x = room.take(2 * rows * k);
        w1 = room.take(2 * n_out * k);
        w3 = room.take(2 * n_out * k);
      }
      parts = room.take(std::max(gated_parts_bytes(rows, k, n_out), gated_parts_bytes(std::max<int64_t>(tokens % rows, 1), k, n_out)));
    }
    bytes = room.bytes;
  }
};
// Backward: the gradients of a and b beside each other, (tokens, 2 h), are one operand of both products, w1 on w3 (2 h, k) the
// other of dx.  Few enough products, and weights whose rows the products take as they are: apart (the weights are not copied).
struct Backward {
  bool apart;
  int64_t h, k, rows;  // n_out and n_in with their padding, tokens of a launch
  int64_t g, w, x, dx, dw, parts, bytes;
  Backward(int64_t tokens, int64_t n_in, int64_t n_out, int what) {
    Room room;
    apart = n_out % 64 == 0 && n_in % 8 == 0 && static_cast<double>(tokens) * n_in * n_out <= 0x1p33;
    h = apart ? n_out : up(n_out, 32), k = up(n_in, 8);
    rows = std::min(tokens, std::max<int64_t>((kMost - 1) / std::max(2 * h, k) / 256 * 256, 256));
    g = room.take(2 * rows * 2 * h);
    w = (what & 1) && !apart ? room.take(2 * 2 * h * k) : 0;
    x = (what & 2) && k != n_in ? room.take(2 * rows * k) : 0;
    dx = (what & 1) && k != n_in ? room.take(2 * rows * k) : 0;
    dw = (what & 2) && (k != n_in || h != n_out) ? room.take(2 * 2 * h * k) : 0;
    parts = 0;
    if (what & 2) {
      const int64_t both = 2 * h, one[2] = {h, h}, rest = std::max<int64_t>(tokens % rows, 1);
      const auto want = [&](int64_t n) { return mega_linear_workspace_bytes(2, n, k, apart ? 2 : 1, apart ? one : &both); };
      parts = room.take(std::max(want(rows), want(rest)));
    }
    bytes = room.bytes;
  }
};

int check(const char* who, int dtype, int64_t tokens, int64_t n_in, int64_t n_out) {
  MEGA_CHECK_ARG(dtype == MEGA_BF16 || dtype == MEGA_F16, "%s: bfloat16 or float16 tensors", who);
  MEGA_CHECK_ARG(tokens >= 1 && n_in >= 1 && n_out >= 1 && tokens < (1ll << 31) && n_in <= (1 << 20) && n_out <= (1 << 20) &&
                     up(n_in, 64) * 2 * up(n_out, 32) < kMost,
                 "%s: bad sizes", who);
  return MEGA_OK;
}
bool aligned16(const void* q) { return reinterpret_cast<uintptr_t>(q) % 16 == 0; }

}  // namespace
}  // namespace mega

using namespace mega;

extern "C" int64_t mega_gated_linear_workspace_bytes(int64_t tokens, int64_t n_in, int64_t n_out, int backward) {
  if (tokens < 1 || n_in < 1 || n_out < 1 || n_in > (1 << 20) || n_out > (1 << 20) || tokens >= (1ll << 31) || up(n_in, 64) * 2 * up(n_out, 32) >= kMost) return 0;
  return backward == 0 ? Forward(tokens, n_in, n_out).bytes : Backward(tokens, n_in, n_out, backward).bytes;
}

extern "C" int mega_gated_linear_fwd(const void* x_, const void* w1_, const void* w3_, int dtype, int64_t tokens, int64_t n_in, int64_t n_out,
                                     void* h_, void* a_, void* b_, void* workspace, void* stream) {
  if (const int rc = check("mega_gated_linear_fwd", dtype, tokens, n_in, n_out); rc != MEGA_OK) return rc;
  MEGA_CHECK_ARG(x_ && w1_ && w3_ && h_ && (a_ == nullptr) == (b_ == nullptr), "mega_gated_linear_fwd: null pointer");
  for (const void* q : {x_, w1_, w3_, static_cast<const void*>(workspace)}) MEGA_CHECK_ARG(aligned16(q), "mega_gated_linear_fwd: misaligned pointer");
  const uint16_t *x = static_cast<const uint16_t*>(x_), *w1 = static_cast<const uint16_t*>(w1_), *w3 = static_cast<const uint16_t*>(w3_);
  uint16_t *h = static_cast<uint16_t*>(h_), *a = static_cast<uint16_t*>(a_), *b = static_cast<uint16_t*>(b_);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (tokens <= kFewTokens) {
    const FewParams p{x, w1, w3, h, a, b, static_cast<int>(tokens), static_cast<int>(n_in), static_cast<int>(n_out)};
    return dtype == MEGA_BF16 ? launch_few<MEGA_BF16>(p, s) : launch_few<MEGA_F16>(p, s);
  }
  const Forward f(tokens, n_in, n_out);
  MEGA_CHECK_ARG(workspace != nullptr || f.bytes == 0, "mega_gated_linear_fwd: null workspace");
  char* const ws = static_cast<char*>(workspace);
  const auto at = [&](int64_t offset) { return reinterpret_cast<uint16_t*>(ws + offset); };
  const bool padded = f.k != n_in;
  if (padded) {
    if (const int rc = widen(w1, at(f.w1), n_out, n_in, f.k, s); rc != MEGA_OK) return rc;
    if (const int rc = widen(w3, at(f.w3), n_out, n_in, f.k, s); rc != MEGA_OK) return rc;
    w1 = at(f.w1), w3 = at(f.w3);
  }
  for (int64_t t = 0; t < tokens; t += f.rows) {
    const int64_t n = std::min(f.rows, tokens - t);
    const uint16_t* rows = x + t * n_in;
    if (padded) {
      if (const int rc = widen(rows, at(f.x), n, n_in, f.k, s); rc != MEGA_OK) return rc;
      rows = at(f.x);
    }
    const bool cut = gated_parts_bytes(n, f.k, n_out) > 0;
    if (const int rc = gated_product(dtype, rows, w1, w3, n, f.k, n_out, h + t * n_out, a ? a + t * n_out : nullptr, b ? b + t * n_out : nullptr,
                                     cut ? reinterpret_cast<float*>(ws + f.parts) : nullptr, s);
        rc != MEGA_OK)
      return rc;
  }
  return MEGA_OK;
}

extern "C" int mega_gated_linear_bwd(const void* dh_, const void* x_, const void* w1_, const void* w3_, const void* a_, const void* b_, int dtype,
                                     int64_t tokens, int64_t n_in, int64_t n_out, void* dx_, void* dw_, void* workspace, void* stream) {
  if (const int rc = check("mega_gated_linear_bwd", dtype, tokens, n_in, n_out); rc != MEGA_OK) return rc;
  MEGA_CHECK_ARG(dh_ && x_ && w1_ && w3_ && a_ && b_ && workspace, "mega_gated_linear_bwd: null pointer");
  for (const void* q : {x_, w1_, w3_, static_cast<const void*>(dx_), static_cast<const void*>(dw_), static_cast<const void*>(workspace)})
    MEGA_CHECK_ARG(aligned16(q), "mega_gated_linear_bwd: misaligned pointer");
  const auto u = [](const void* q) { return static_cast<const uint16_t*>(q); };
  const uint16_t *dh = u(dh_), *x = u(x_), *w1 = u(w1_), *w3 = u(w3_), *a = u(a_), *b = u(b_);
  uint16_t *dx = static_cast<uint16_t*>(dx_), *dw = static_cast<uint16_t*>(dw_);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int what = (dx != nullptr) + 2 * (dw != nullptr);
  if (what == 0) return MEGA_OK;
  const Backward f(tokens, n_in, n_out, what);
  char* const ws = static_cast<char*>(workspace);
  const auto at = [&](int64_t offset) { return reinterpret_cast<uint16_t*>(ws + offset); };
  const int64_t h = f.h, k = f.k;
  if (dx != nullptr && !f.apart) {
    if (const int rc = widen(w1, at(f.w), n_out, n_in, k, s); rc != MEGA_OK) return rc;
    if (const int rc = widen(w3, at(f.w) + h * k, n_out, n_in, k, s); rc != MEGA_OK) return rc;
    // (features behind the last meet gradients that are zero: they have to be finite)
    if (h != n_out) {
      MEGA_CHECK_ARG(h - n_out < 32, "mega_gated_linear_bwd: padding");
      if (const int rc = widen(w1, at(f.w) + n_out * k, h - n_out, 0, k, s); rc != MEGA_OK) return rc;
      if (const int rc = widen(w3, at(f.w) + (h + n_out) * k, h - n_out, 0, k, s); rc != MEGA_OK) return rc;
    }
  }
  uint16_t* const dw_at = dw != nullptr && (k != n_in || h != n_out) ? at(f.dw) : dw;
  for (int64_t t = 0; t < tokens; t += f.rows) {
    const int64_t n = std::min(f.rows, tokens - t);
    uint16_t *da = at(f.g), *db = f.apart ? da + n * h : da + h;
    const int64_t ld = f.apart ? h : 2 * h, at0 = t * n_out;
    const unsigned grid = pieces_grid(n * (h / 8));
    if (dtype == MEGA_BF16) gate_grad_kernel<MEGA_BF16><<<grid, kThreads, 0, s>>>(dh + at0, a + at0, b + at0, da, db, n, (int)n_out, (int)h, ld);
    else gate_grad_kernel<MEGA_F16><<<grid, kThreads, 0, s>>>(dh + at0, a + at0, b + at0, da, db, n, (int)n_out, (int)h, ld);
    MEGA_CHECK_LAUNCH();
    const int64_t both = 2 * h, one[2] = {h, h};
    const void *gs[2] = {da, db}, *wide = at(f.w);
    if (dx != nullptr) {
      uint16_t* const to = k != n_in ? at(f.dx) : dx + t * n_in;
      const void* ws2[2] = {w1, w3};
      const int rc = f.apart ? mega_linear_input_grad(gs, ws2, nullptr, dtype, n, k, 2, one, to, stream)
                             : mega_linear_input_grad(gs, &wide, nullptr, dtype, n, k, 1, &both, to, stream);
      if (rc != MEGA_OK) return rc;
      if (k != n_in)
        if (const int rc2 = narrow(to, dx + t * n_in, n, k, n_in, s); rc2 != MEGA_OK) return rc2;
    }
    if (dw != nullptr) {
      const uint16_t* rows = x + t * n_in;
      if (k != n_in) {
        if (const int rc = widen(rows, at(f.x), n, n_in, k, s); rc != MEGA_OK) return rc;
        rows = at(f.x);
      }
      const bool cut = mega_linear_workspace_bytes(2, n, k, f.apart ? 2 : 1, f.apart ? one : &both) > 0;
      float* const parts = cut ? reinterpret_cast<float*>(ws + f.parts) : nullptr;
      void* to[2] = {dw_at, dw_at + h * k};
      // (apart: all of the tokens in one launch)
      const int rc = f.apart ? mega_linear_weight_grads(gs, rows, dtype, n, k, 2, one, to, parts, stream)
                             : weight_grad_onto(dtype, da, rows, n, k, both, t > 0 ? dw_at : nullptr, dw_at, parts, s);
      if (rc != MEGA_OK) return rc;
    }
  }
  if (dw != nullptr && dw_at != dw) {
    if (const int rc = narrow(dw_at, dw, n_out, k, n_in, s); rc != MEGA_OK) return rc;
    return narrow(dw_at + h * k, dw + n_out * n_in, n_out, k, n_in, s);
  }
  return MEGA_OK;
}
