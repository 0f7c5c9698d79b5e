// Embedding as a C++ autograd node (csrc/embedding.hip).
#include "host.hpp"

#include <torch/csrc/autograd/custom_function.h>

namespace mega_host {
namespace {

using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

// (autocast leaves rows of a table in their type)
bool shown() { return watched(c10::autocast_dispatch_keyset); }

Tensor gather(const Tensor& tokens, const Tensor& table, double scale) {
  const int64_t n = tokens.numel(), width = table.size(1);
  auto shape = tokens.sizes().vec();
  shape.push_back(width);
  Tensor out = at::empty(shape, table.options());
  const Tensor rows = width <= 1 || table.stride(1) == 1 ? table : table.contiguous();
  check(mega_embedding_fwd(tokens.data_ptr(), tokens.scalar_type() == at::kLong ? 64 : 32, rows.data_ptr(), code_of(table.scalar_type()), n, table.size(0), width,
                           rows.size(0) > 1 ? rows.stride(0) : width, scale, out.data_ptr(), stream_of(table)), "mega_embedding_fwd");
  return out;
}

// dW of (..., width) gradients by their tokens
Tensor table_grad(const Tensor& dy_, const Tensor& tokens, int64_t vocab, double scale, int64_t padding) {
  const Tensor dy = stored(dy_).contiguous();
  const int64_t width = dy.size(-1), n = tokens.numel();
  const int code = code_of(dy.scalar_type());
  Tensor dw = at::empty({vocab, width}, dy.options());
  const Tensor ws = at::empty({mega_embedding_workspace_bytes(code, n, vocab, width)}, dy.options().dtype(at::kByte));
  check(mega_embedding_bwd(dy.data_ptr(), code, tokens.data_ptr(), tokens.scalar_type() == at::kLong ? 64 : 32, n, vocab, width, scale, padding, dw.data_ptr(),
                           n > 0 ? ws.data_ptr() : nullptr, stream_of(dy)), "mega_embedding_bwd");
  return dw;
}

Tensor embedding(const Tensor& tokens, const Tensor& table, double scale, std::optional<int64_t> padding);

// The table's gradient where it is differentiated again: the same kernel, so that the gradient is the same; it is linear in dy, and its own gradient the
// rows of tokens that have one.
struct TableGradFn : Function<TableGradFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& dy, const Tensor& tokens, int64_t vocab, double scale, int64_t padding) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({tokens});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    return table_grad(dy, tokens, vocab, scale, padding);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const Tensor tokens = ctx->get_saved_variables()[0];
    const int64_t padding = ctx->saved_data["padding"].toInt();
    c10::DeviceGuard guard(g[0].device());
    return {embedding(padding < 0 ? tokens : tokens.masked_fill(tokens.eq(padding), -1), g[0], ctx->saved_data["scale"].toDouble(), std::nullopt), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

struct EmbeddingFn : Function<EmbeddingFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& table, const Tensor& tokens, double scale, int64_t padding) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({tokens});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    ctx->saved_data["vocab"] = table.size(0);
    return gather(tokens, table, scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const Tensor tokens = stored(ctx->get_saved_variables()[0]).contiguous();  // (saved-tensor hooks may hand back anything)
    require((tokens.scalar_type() == at::kLong || tokens.scalar_type() == at::kInt) && tokens.device() == g[0].device() && tokens.numel() * g[0].size(-1) == g[0].numel(),
            "embedding: the saved tokens have another type, device or number than they were saved with");
    const double scale = ctx->saved_data["scale"].toDouble();
    const int64_t padding = ctx->saved_data["padding"].toInt(), vocab = ctx->saved_data["vocab"].toInt();
    c10::DeviceGuard guard(g[0].device());
    if (shown() || !plain(stored(g[0]))) {  // (several gradients at once)
      const int64_t width = g[0].size(-1);
      const Tensor t = tokens.reshape({-1}).to(at::kLong), counts = at::logical_and(at::logical_and(t.ge(0), t.lt(vocab)), t.ne(padding));
      const Tensor rows = at::where(counts.unsqueeze(1), g[0].reshape({-1, width}).to(at::kFloat), at::zeros({}, g[0].options().dtype(at::kFloat)));
      return {at::embedding_dense_backward(rows, t.clamp(0, vocab - 1), vocab, -1, false).mul(scale).to(g[0].scalar_type()), Tensor(), Tensor(), Tensor()};
    }
    if (at::GradMode::is_enabled()) return {TableGradFn::apply(g[0], tokens, vocab, scale, padding), Tensor(), Tensor(), Tensor()};
    at::AutoDispatchBelowADInplaceOrView below;
    return {table_grad(g[0], tokens, vocab, scale, padding), Tensor(), Tensor(), Tensor()};
  }
};

// The same by the library's operations.
Tensor recorded(const Tensor& tokens, const Tensor& table, double scale, int64_t padding) {
  const int64_t vocab = table.size(0);
  const Tensor there = at::logical_and(tokens.ge(0), tokens.lt(vocab)).unsqueeze(-1);
  const Tensor rows = at::embedding(table, tokens.clamp(0, vocab - 1), padding);
  return at::where(there, scale == 1 ? rows : rows.to(at::kFloat).mul(scale).to(table.scalar_type()), at::zeros({}, table.options()));
}

Tensor embedding(const Tensor& tokens_, const Tensor& table_, double scale, std::optional<int64_t> padding_) {
  require(tokens_.is_cuda() && table_.is_cuda(), "megalodon_amd ops need GPU (HIP) tensors; there is no CPU fallback");
  require(tokens_.device() == table_.device(), "all tensors must be on the same device");
  require(tokens_.scalar_type() == at::kLong || tokens_.scalar_type() == at::kInt, "embedding: tokens must be int64 or int32");
  require(table_.dim() == 2 && code_of(table_.scalar_type()) >= 0, "embedding: weight must be (vocabulary, width), float32, bfloat16 or float16");
  const int64_t vocab = table_.size(0);
  require(vocab >= 1 && table_.size(1) >= 1, "embedding: weight must not be empty");
  int64_t padding = -1;
  if (padding_.has_value()) {
    require(*padding_ >= -vocab && *padding_ < vocab, "embedding: padding_idx must be a row of weight");
    padding = *padding_ < 0 ? *padding_ + vocab : *padding_;
  }
  // what watches the thread's operations is shown operations
  const Tensor given = stored(tokens_), table = stored(table_);
  if (shown() || !plain(given) || !plain(table)) return recorded(given, table, scale, padding);
  c10::DeviceGuard guard(table.device());
  const Tensor tokens = given.contiguous();
  if ((at::GradMode::is_enabled() && table.requires_grad()) || has_tangent(table)) return EmbeddingFn::apply(table, tokens, scale, padding);
  return gather(tokens, table, scale);
}

}  // namespace

void bind_embedding(py::module_& m) { m.def("embedding", &embedding, py::call_guard<py::gil_scoped_release>()); }

}  // namespace mega_host
