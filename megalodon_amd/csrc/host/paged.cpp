// The paged key / value cache: writing to it, reading it back, attention over it (csrc/paged_*.hip).
#include "host.hpp"

#include <ATen/core/grad_mode.h>

#include <tuple>

namespace mega_host {
namespace {

using Optional = std::optional<Tensor>;

// [first, last) byte of what a strided tensor can touch
std::pair<uintptr_t, uintptr_t> span(const Tensor& t) {
  const auto first = reinterpret_cast<uintptr_t>(t.data_ptr());
  if (t.numel() == 0) return {first, first};
  int64_t last = 0;
  for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
  return {first, first + (last + 1) * t.element_size()};
}
bool overlap(const Tensor& a, const Tensor& b) {
  const auto [a0, a1] = span(a);
  const auto [b0, b1] = span(b);
  return a0 < b1 && b0 < a1;
}

// serving operators: nothing is recorded, so a gradient that is asked for is refused, not dropped
void no_gradient(std::initializer_list<const Tensor*> ts, const char* who) {
  const bool on = at::GradMode::is_enabled();
  for (const Tensor* t : ts)
    if ((on && t->requires_grad()) || has_tangent(*t)) fail(std::string(who) + " has no gradient: call it under torch.no_grad()");
}

struct Cache {
  mega_paged_cache c{};
  at::ScalarType type;  // of the pool's elements
  const Tensor *k, *v;
};

void no_repeats(const Tensor& t, const char* name) {
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1 && t.stride(i) <= 0) fail(std::string(name) + " must not be an expanded tensor");
}

Cache cache_of(const Tensor& k, const Tensor& v, const Tensor& table, const Optional& ke, const Optional& ve) {
  Cache r;
  r.k = &k, r.v = &v;
  require(k.is_cuda() && v.is_cuda() && table.is_cuda(), "megalodon_amd ops need GPU (HIP) tensors; there is no CPU fallback");
  require(k.device() == v.device() && k.device() == table.device(), "all tensors must be on the same device");
  require(k.dim() == 4 && v.dim() == 4 && k.sizes().slice(0, 3) == v.sizes().slice(0, 3),
          "paged cache: k_pages and v_pages must be (pages, page_size, heads, width) with the same pages, page_size and heads");
  require(!lazy(k) && !lazy(v), "paged cache: pools must not be lazily negated views");
  r.type = k.scalar_type();
  require(v.scalar_type() == r.type, "paged cache: k_pages and v_pages must have the same dtype");
  const bool eight = r.type == at::kFloat8_e4m3fn;
  require(eight || r.type == at::kBFloat16 || r.type == at::kHalf, "paged cache: pools must be bfloat16, float16 or float8_e4m3fn");
  for (const Tensor* t : {&k, &v}) {
    require(t->stride(3) == 1, "paged cache: the last axis of a pool must be contiguous");
    no_repeats(*t, "paged cache: a pool");
  }
  require(table.dim() == 2 && table.scalar_type() == at::kInt && (table.size(1) <= 1 || table.stride(1) == 1),
          "paged cache: block_table must be int32 (sequences, pages of one) with a contiguous last axis");
  require(table.size(0) <= 1 || table.stride(0) >= 0, "paged cache: bad block_table strides");
  require(ke.has_value() == eight && ve.has_value() == eight, "paged cache: exponents belong to float8_e4m3fn pools, and to both of them");
  mega_paged_cache& c = r.c;
  if (eight)
    for (const auto& [e, to, stride] : {std::tuple<const Optional&, uint8_t**, int64_t*>{ke, &c.k_exponents, c.ke_stride}, {ve, &c.v_exponents, c.ve_stride}}) {
      require((*e).is_cuda() && (*e).device() == k.device(), "all tensors must be on the same device");
      require((*e).scalar_type() == at::kByte && (*e).sizes() == k.sizes().slice(0, 3), "paged cache: exponents must be uint8 (pages, page_size, heads)");
      no_repeats(*e, "paged cache: exponents");
      *to = static_cast<uint8_t*>((*e).data_ptr());
      for (int i = 0; i < 3; ++i) stride[i] = (*e).stride(i);
    }
  c.k = k.data_ptr(), c.v = v.data_ptr();
  for (int i = 0; i < 3; ++i) c.k_stride[i] = k.size(i) > 1 ? k.stride(i) : 0, c.v_stride[i] = v.size(i) > 1 ? v.stride(i) : 0;
  c.pages = k.size(0), c.page_size = k.size(1), c.heads = k.size(2), c.k_width = k.size(3), c.v_width = v.size(3);
  c.table = static_cast<const int32_t*>(table.data_ptr()), c.table_stride = table.size(0) > 1 ? table.stride(0) : 0;
  c.table_width = table.size(1), c.batch = table.size(0);
  return r;
}

const int32_t* counts(const Tensor& t, const Cache& cache, int64_t n, const char* what) {
  require(t.is_cuda() && t.device() == cache.k->device(), "all tensors must be on the same device");
  if (t.dim() != 1 || t.scalar_type() != at::kInt || t.size(0) != n || !t.is_contiguous()) fail(std::string("paged cache: ") + what);
  return static_cast<const int32_t*>(t.data_ptr());
}
const char* const kPerSequence = "lengths and begins must be contiguous int32 with one number for each row of block_table";
const char* const kBounds = "the packed rows' bounds must be contiguous int32 with one number more than block_table has rows";

// packed rows (rows, heads, width) as the kernels take them: a contiguous last axis, 16-byte steps
Tensor packed(const Tensor& t, const Cache& cache, const char* what) {
  require(t.is_cuda(), "megalodon_amd ops need GPU (HIP) tensors; there is no CPU fallback");
  require(t.device() == cache.k->device(), "all tensors must be on the same device");
  if (t.dim() != 3) fail(std::string(what) + " must be (rows, heads, width)");
  require(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, "paged cache: rows must be bfloat16 or float16");
  if (cache.type != at::kFloat8_e4m3fn) require(t.scalar_type() == cache.type, "paged cache: rows must have the pools' dtype");
  const Tensor s = stored(t);
  const auto step = [&](int64_t i) { return s.size(i) <= 1 || (s.stride(i) >= 0 && s.stride(i) % 8 == 0); };
  if (s.numel() == 0 || ((s.size(2) <= 1 || s.stride(2) == 1) && step(0) && step(1) && reinterpret_cast<uintptr_t>(s.data_ptr()) % 16 == 0)) return s;
  const Tensor c = s.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone(at::MemoryFormat::Contiguous);
}
int64_t step_of(const Tensor& t, int64_t i) { return t.size(i) > 1 ? t.stride(i) : 0; }

void wrote(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

void paged_cache_write(const Tensor& k, const Tensor& v, const Tensor& k_pages, const Tensor& v_pages, const Tensor& table, const Tensor& lengths,
                       const Tensor& cu, const Optional& ke, const Optional& ve) {
  const Cache cache = cache_of(k_pages, v_pages, table, ke, ve);
  no_gradient({&k, &v, &k_pages, &v_pages}, "paged_cache_write");
  c10::DeviceGuard guard(k_pages.device());
  const Tensor kr = packed(k, cache, "paged_cache_write: k"), vr = packed(v, cache, "paged_cache_write: v");
  const mega_paged_cache& c = cache.c;
  require(kr.scalar_type() == vr.scalar_type() && kr.size(0) == vr.size(0), "paged_cache_write: k and v must have the same dtype and number of rows");
  require(kr.size(1) == c.heads && vr.size(1) == c.heads && kr.size(2) == c.k_width && vr.size(2) == c.v_width,
          "paged_cache_write: k and v must have the pools' heads and widths");
  for (const Tensor* from : {&kr, &vr})
    for (const Tensor* to : {&k_pages, &v_pages, ke.has_value() ? &*ke : &k_pages, ve.has_value() ? &*ve : &v_pages})
      require(!overlap(*from, *to), "paged_cache_write: new rows must not lie in the pools");
  const int32_t *n = counts(lengths, cache, c.batch, kPerSequence), *bounds = counts(cu, cache, c.batch + 1, kBounds);
  check(mega_paged_cache_write(&c, code_of(kr.scalar_type()), kr.data_ptr(), step_of(kr, 0), step_of(kr, 1), vr.data_ptr(), step_of(vr, 0), step_of(vr, 1),
                               n, bounds, kr.size(0), stream_of(k_pages)), "mega_paged_cache_write");
  wrote(k_pages), wrote(v_pages);
  if (ke.has_value()) wrote(*ke), wrote(*ve);
}

std::tuple<Tensor, Tensor> paged_cache_read(const Tensor& k_pages, const Tensor& v_pages, const Tensor& table, const Tensor& begins, const Tensor& cu,
                                            int64_t rows, const Optional& ke, const Optional& ve, std::optional<at::ScalarType> dtype) {
  const Cache cache = cache_of(k_pages, v_pages, table, ke, ve);
  no_gradient({&k_pages, &v_pages}, "paged_cache_read");
  const mega_paged_cache& c = cache.c;
  const bool eight = cache.type == at::kFloat8_e4m3fn;
  const auto type = dtype.value_or(eight ? at::kBFloat16 : cache.type);
  require(type == at::kBFloat16 || type == at::kHalf, "paged_cache_read: dtype must be bfloat16 or float16");
  require(eight || type == cache.type, "paged_cache_read: a 16-bit cache is read in its own dtype");
  require(rows >= 0, "paged_cache_read: rows must not be negative");
  c10::DeviceGuard guard(k_pages.device());
  const int32_t *n = counts(begins, cache, c.batch, kPerSequence), *bounds = counts(cu, cache, c.batch + 1, kBounds);
  const auto options = k_pages.options().dtype(type);
  if (c.batch == 0) return {at::zeros({rows, c.heads, c.k_width}, options), at::zeros({rows, c.heads, c.v_width}, options)};
  Tensor k = at::empty({rows, c.heads, c.k_width}, options), v = at::empty({rows, c.heads, c.v_width}, options);
  check(mega_paged_cache_read(&c, code_of(type), n, bounds, rows, k.data_ptr(), v.data_ptr(), 1, stream_of(k_pages)), "mega_paged_cache_read");
  return {k, v};
}

Tensor paged_attention(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& table, const Tensor& lengths, const Tensor& cu,
                       double scale, int64_t chunk, const Optional& ke, const Optional& ve, const Optional& out) {
  const Cache cache = cache_of(k_pages, v_pages, table, ke, ve);
  no_gradient({&q, &k_pages, &v_pages}, "paged_attention");
  const mega_paged_cache& c = cache.c;
  c10::DeviceGuard guard(k_pages.device());
  const Tensor qr = packed(q, cache, "paged_attention: q");
  require(qr.size(2) == c.k_width, "paged_attention: q must have the keys' width");
  require(c.heads >= 1 && qr.size(1) >= 1 && qr.size(1) % c.heads == 0, "paged_attention: the number of query heads must be a multiple of the cache's");
  require(chunk >= 0, "paged_attention: chunk_size must not be negative (0: no chunks)");
  const int32_t *n = counts(lengths, cache, c.batch, kPerSequence), *bounds = counts(cu, cache, c.batch + 1, kBounds);
  const int64_t rows = qr.size(0), heads = qr.size(1);
  Tensor y;
  if (out.has_value()) {
    y = *out;
    no_gradient({&y}, "paged_attention");
    require(y.is_cuda() && y.device() == qr.device() && y.scalar_type() == qr.scalar_type() && y.is_contiguous() && !lazy(y) &&
                y.sizes() == at::IntArrayRef({rows, heads, c.v_width}),
            "paged_attention: out must be contiguous (rows, query heads, v width) of q's dtype and device");
    for (const Tensor* t : {&qr, &k_pages, &v_pages, ke.has_value() ? &*ke : &k_pages, ve.has_value() ? &*ve : &v_pages})
      require(!overlap(y, *t), "paged_attention: out must not overlap q or the pools");
  } else {
    y = at::empty({rows, heads, c.v_width}, qr.options());
  }
  const int code = code_of(qr.scalar_type());
  const int64_t ws_bytes = mega_paged_attention_workspace_bytes(&c, rows, heads, chunk);
  Tensor ws;
  if (ws_bytes > 0) ws = at::empty({ws_bytes}, qr.options().dtype(at::kByte));
  check(mega_paged_attention_fwd(&c, code, qr.data_ptr(), step_of(qr, 0), step_of(qr, 1), n, bounds, rows, heads, scale, chunk, y.data_ptr(),
                                 !out.has_value(), ws.defined() ? ws.data_ptr() : nullptr, stream_of(k_pages)), "mega_paged_attention_fwd");
  if (out.has_value()) wrote(y);
  return y;
}

}  // namespace

void bind_paged(py::module_& m) {
  using free = py::call_guard<py::gil_scoped_release>;
  m.def("paged_cache_write", &paged_cache_write, free());
  m.def("paged_cache_read", &paged_cache_read, free());
  m.def("paged_attention", &paged_attention, free());
}

}  // namespace mega_host
