// The norm of many tensors and clipping by it (csrc/clip.hip).
#include "host.hpp"

#include <ATen/core/grad_mode.h>

#include <algorithm>
#include <cmath>
#include <tuple>
#include <vector>

namespace mega_host {
namespace {

// what the C interface takes, and the arrays that it points to
struct List {
  std::vector<const void*> from;
  std::vector<void*> to;
  std::vector<int64_t> size;
  std::vector<int32_t> dtype;
  mega_tensors c() const { return {static_cast<int64_t>(from.size()), from.data(), to.data(), size.data(), dtype.data()}; }
};

int kind_of(double norm_type) {
  if (norm_type == 2.0) return MEGA_NORM_2;
  if (std::isinf(norm_type) && norm_type > 0) return MEGA_NORM_MAX;
  fail("the gradients' norm is offered for norm_type 2 and infinity");
}

List list_of(const std::vector<Tensor>& tensors, bool detached, const char* who) {
  List list;
  const bool on = at::GradMode::is_enabled() && !detached;
  for (const Tensor& t : tensors) {
    require(t.layout() == at::kStrided, "the gradients' norm: sparse tensors are not supported");
    require(t.is_cuda(), "megalodon_amd ops need GPU (HIP) tensors; there is no CPU fallback");
    require(t.device() == tensors[0].device(), "all tensors must be on the same device");
    if ((on && t.requires_grad()) || has_tangent(t)) fail(std::string(who) + " has no gradient: call it under torch.no_grad()");
    require(code_of(t.scalar_type()) >= 0, "the gradients' norm: tensors must be float32, bfloat16 or float16");
    require(!lazy(t), "the gradients' norm: tensors must not be lazily negated views");
    require(t.numel() == 0 || t.is_non_overlapping_and_dense(), "the gradients' norm: tensors must fill their memory without gaps (any order of the axes)");
    list.from.push_back(t.data_ptr());
    list.size.push_back(t.numel());
    list.dtype.push_back(code_of(t.scalar_type()));
  }
  return list;
}

// Nothing that is written may be anything else's memory but its own source's.
void no_overlap(const List& list) {
  struct Span {
    uintptr_t first, last;
    bool written;
  };
  std::vector<Span> spans;
  spans.reserve(2 * list.from.size());
  for (size_t i = 0; i < list.from.size(); ++i) {
    const auto from = reinterpret_cast<uintptr_t>(list.from[i]), to = reinterpret_cast<uintptr_t>(list.to[i]);
    const uintptr_t bytes = list.size[i] * (list.dtype[i] == MEGA_F32 ? 4 : 2);
    if (bytes == 0) continue;
    spans.push_back({to, to + bytes, true});
    if (from != to) spans.push_back({from, from + bytes, false});
  }
  std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.first < b.first; });
  uintptr_t last = 0, last_written = 0;  // the furthest ends so far
  for (const Span& s : spans) {
    require(s.first >= (s.written ? last : last_written), "clip_grads: what is written must not overlap another tensor");
    last = std::max(last, s.last);
    if (s.written) last_written = std::max(last_written, s.last);
  }
}

Tensor norm_raw(const std::vector<Tensor>& tensors, const List& list, int kind, Tensor& workspace) {
  const mega_tensors c = list.c();
  workspace = at::empty({mega_tensors_workspace_bytes(&c)}, tensors[0].options().dtype(at::kByte));
  Tensor out = at::empty({}, tensors[0].options().dtype(at::kFloat));
  check(mega_tensors_norm(&c, kind, out.data_ptr<float>(), workspace.data_ptr(), stream_of(tensors[0])), "mega_tensors_norm");
  return out;
}

Tensor grad_norm(const std::vector<Tensor>& tensors, double norm_type, bool detached) {
  const int kind = kind_of(norm_type);
  require(!tensors.empty(), "grad_norm: no tensors");
  const List list = list_of(tensors, detached, "grad_norm");
  c10::DeviceGuard guard(tensors[0].device());
  at::NoGradGuard none;
  Tensor workspace;
  return norm_raw(tensors, list, kind, workspace);
}

Tensor clip_grads(const std::vector<Tensor>& tensors, const std::vector<Tensor>& out, double max_norm, double norm_type, bool detached) {
  const int kind = kind_of(norm_type);
  require(!tensors.empty(), "clip_grads: no tensors");
  require(max_norm >= 0, "clip_grads: max_norm must not be negative");
  require(out.size() == tensors.size(), "clip_grads: out must have a tensor for each one");
  List list = list_of(tensors, detached, "clip_grads");
  for (size_t i = 0; i < out.size(); ++i) {
    const Tensor &t = tensors[i], &o = out[i];
    require(o.is_cuda() && o.device() == t.device() && o.scalar_type() == t.scalar_type() && o.layout() == at::kStrided && !lazy(o) && o.sizes() == t.sizes() &&
                (o.strides() == t.strides() || (o.is_contiguous() && t.is_contiguous())),
            "clip_grads: out must have the tensors' shapes, strides, dtypes and device");
    if ((at::GradMode::is_enabled() && !detached && o.requires_grad()) || has_tangent(o)) fail("clip_grads has no gradient: call it under torch.no_grad()");
    list.to.push_back(o.data_ptr());
  }
  no_overlap(list);
  c10::DeviceGuard guard(tensors[0].device());
  at::NoGradGuard none;
  Tensor workspace;
  Tensor norm = norm_raw(tensors, list, kind, workspace);
  const mega_tensors c = list.c();
  check(mega_tensors_clip(&c, max_norm, workspace.data_ptr(), stream_of(tensors[0])), "mega_tensors_clip");
  for (const Tensor& o : out)
    if (!o.is_inference()) o.unsafeGetTensorImpl()->bump_version();
  return norm;
}

}  // namespace

void bind_clip(py::module_& m) {
  using free = py::call_guard<py::gil_scoped_release>;
  m.def("grad_norm", &grad_norm, free());
  m.def("clip_grads", &clip_grads, free());
}

}  // namespace mega_host
