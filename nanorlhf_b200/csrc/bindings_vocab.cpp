// Tensors in, launches out: the kernels over rows of logits.
#include "bindings_vocab.h"

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/extension.h>

#include <limits>
#include <tuple>

#include "vocab_rows.h"

namespace {

inline cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }
inline void check(cudaError_t e, const char* what) { TORCH_CHECK(e == cudaSuccess, what, ": ", cudaGetErrorString(e)); }

// [rows, V], bf16 or float, the elements of a row side by side
void check_logits(const torch::Tensor& t, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.dim() == 2 && (t.scalar_type() == torch::kBFloat16 || t.scalar_type() == torch::kFloat32), what,
              ": logits must be a CUDA tensor [rows, V], bf16 or float32");
  TORCH_CHECK(t.size(1) > 0 && t.size(1) <= std::numeric_limits<int>::max() - 64 && t.size(0) <= std::numeric_limits<int>::max(), what,
              ": logits have no columns, or too many rows or columns");
  TORCH_CHECK(t.size(1) == 1 || t.stride(1) == 1, what, ": the elements of a row of logits must be side by side");
}
// contiguous, on the logits' device
void check_beside(const torch::Tensor& t, const torch::Tensor& logits, torch::ScalarType type, at::IntArrayRef sizes, const char* what, const char* name) {
  TORCH_CHECK(t.device() == logits.device() && t.scalar_type() == type && t.sizes() == sizes && t.is_contiguous(), what, ": ", name, " must be a contiguous ",
              type, " tensor of shape ", sizes, " on the logits' device");
}
// a call's scratch memory: of the current stream, on 512 bytes
torch::Tensor scratch_of(size_t bytes, const torch::Tensor& logits) {
  return bytes > 0 ? torch::empty({static_cast<int64_t>(bytes)}, logits.options().dtype(torch::kUInt8)) : torch::Tensor();
}
inline void* ptr_of(const torch::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
inline bool is_bf16(const torch::Tensor& t) { return t.scalar_type() == torch::kBFloat16; }

std::tuple<torch::Tensor, torch::Tensor> top_logprobs(const torch::Tensor& logits, int64_t k, double inv_temp) {
  check_logits(logits, "top_logprobs");
  TORCH_CHECK(k >= 1 && k <= kTopMax && k <= logits.size(1), "top_logprobs: k must be between 1 and the smaller of ", kTopMax, " and the columns");
  c10::cuda::CUDAGuard guard(logits.device());
  torch::Tensor logp = torch::empty({logits.size(0), k}, logits.options().dtype(torch::kFloat32));
  torch::Tensor idx = torch::empty({logits.size(0), k}, logits.options().dtype(torch::kInt32));
  const torch::Tensor scratch = scratch_of(nrl_top_scratch(is_bf16(logits), logits.size(0), logits.size(1), k), logits);
  check(nrl_top_logprobs(logits.data_ptr(), is_bf16(logits), logits.stride(0), logits.size(0), logits.size(1), k, inv_temp, logp.data_ptr<float>(),
                         idx.data_ptr<int>(), ptr_of(scratch), cur_stream()), "top_logprobs");
  return {logp, idx};
}

// token losses, their weighted sum (with_loss) and its gradient (undefined unless wanted), of the logits' type or, of float logits, bf16
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> distill_loss(const torch::Tensor& logits, const torch::Tensor& top_logp, const torch::Tensor& top_idx,
                                                                     const c10::optional<torch::Tensor>& weights, double inv_temp, double beta, bool tail,
                                                                     bool want_grad, bool bf16_grad, bool with_loss) {
  check_logits(logits, "distill_loss");
  const int64_t rows = logits.size(0), V = logits.size(1);
  TORCH_CHECK(V <= kDistillVocabMax, "distill_loss: more than ", kDistillVocabMax, " columns");
  TORCH_CHECK(top_logp.dim() == 2 && top_logp.size(1) >= 1 && top_logp.size(1) <= kTopMax, "distill_loss: between 1 and ", kTopMax, " entries of the teacher a row");
  const int64_t k = top_logp.size(1);
  check_beside(top_logp, logits, torch::kFloat32, {rows, k}, "distill_loss", "top_logp");
  check_beside(top_idx, logits, torch::kInt32, {rows, k}, "distill_loss", "top_idx");
  if (weights.has_value()) check_beside(*weights, logits, torch::kFloat32, {rows}, "distill_loss", "weights");
  c10::cuda::CUDAGuard guard(logits.device());
  const auto f32 = logits.options().dtype(torch::kFloat32);
  torch::Tensor token = torch::empty({rows}, f32), loss, grad;
  if (with_loss) loss = torch::empty({}, f32);
  if (want_grad) grad = torch::empty({rows, V}, logits.options().dtype(bf16_grad || is_bf16(logits) ? torch::kBFloat16 : torch::kFloat32));
  const torch::Tensor scratch = scratch_of(nrl_distill_scratch(is_bf16(logits), rows, V, want_grad), logits);
  check(nrl_distill_loss(logits.data_ptr(), is_bf16(logits), logits.stride(0), rows, V, top_logp.data_ptr<float>(), top_idx.data_ptr<int>(), k,
                         weights.has_value() ? weights->data_ptr<float>() : nullptr, inv_temp, beta, tail, token.data_ptr<float>(),
                         with_loss ? loss.data_ptr<float>() : nullptr, ptr_of(grad), want_grad && is_bf16(grad), ptr_of(scratch), cur_stream()),
        "distill_loss");
  return {loss, token, grad};
}

torch::Tensor weighted_sum(const torch::Tensor& token_loss, const torch::Tensor& weights) {
  TORCH_CHECK(token_loss.is_cuda() && token_loss.dim() == 1, "weighted_sum: token_loss must be a CUDA tensor [rows]");
  check_beside(token_loss, token_loss, torch::kFloat32, token_loss.sizes(), "weighted_sum", "token_loss");
  check_beside(weights, token_loss, torch::kFloat32, token_loss.sizes(), "weighted_sum", "weights");
  c10::cuda::CUDAGuard guard(token_loss.device());
  torch::Tensor loss = torch::empty({}, token_loss.options());
  check(nrl_weighted_sum(token_loss.data_ptr<float>(), weights.data_ptr<float>(), token_loss.numel(), loss.data_ptr<float>(), cur_stream()), "weighted_sum");
  return loss;
}

// x *= g (a scalar on the device), in place; nothing is touched where g is 1
void scale_(torch::Tensor x, const torch::Tensor& g) {
  TORCH_CHECK(x.is_cuda() && x.is_contiguous() && (is_bf16(x) || x.scalar_type() == torch::kFloat32) && g.device() == x.device() &&
              g.scalar_type() == torch::kFloat32 && g.numel() == 1, "scale_: a contiguous bf16 or float32 CUDA tensor and a float32 scalar beside it");
  c10::cuda::CUDAGuard guard(x.device());
  check(nrl_scale(x.data_ptr(), is_bf16(x), x.numel(), g.data_ptr<float>(), cur_stream()), "scale_");
}

// which graph the current stream is being captured into (0: none)
int64_t capture_id() {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  check(cudaStreamGetCaptureInfo(cur_stream(), &status, &id), "capture_id");
  return status == cudaStreamCaptureStatusActive ? static_cast<int64_t>(id) : 0;
}

// A gradient of the running backward, where it may be differentiated again: its own derivative with respect to that backward's inputs is refused, for it was formed in the
// forward and is a constant here.
torch::Tensor refuse_second(const torch::Tensor& grad) {
  const auto node = torch::autograd::get_current_node();
  if (!at::GradMode::is_enabled() || !node) return grad;
  torch::Tensor out = grad.detach();
  torch::autograd::edge_list inputs = node->next_edges();
  torch::autograd::create_gradient_edge(out, std::make_shared<torch::autograd::Error>("distillation: there is no second derivative", std::move(inputs)));
  return out;
}

// grads times g, in place where this backward is the graph's only one, which frees them, and every replay of a captured one forms them again
torch::Tensor scaled(torch::Tensor grad, const torch::Tensor& g, int64_t capture) {
  if (!grad.defined()) return grad;
  grad = refuse_second(grad);
  if (at::GradMode::is_enabled() || torch::autograd::get_current_graph_task_keep_graph() || g.scalar_type() != torch::kFloat32 || capture_id() != capture)
    return grad.scalar_type() == g.scalar_type() ? grad * g : (grad.to(torch::kFloat32) * g).to(grad.scalar_type());
  scale_(grad, g);
  return grad;
}

// what a call gives of the teacher, as the kernels take it
std::tuple<torch::Tensor, torch::Tensor, c10::optional<torch::Tensor>> teacher_entries(const torch::Tensor& top_logp, const torch::Tensor& top_idx,
                                                                                       const c10::optional<torch::Tensor>& weights, int64_t columns) {
  torch::Tensor idx = top_idx.scalar_type() == torch::kInt32 ? top_idx : top_idx.clamp(-1, columns).to(torch::kInt32);        // what is no token stays none
  c10::optional<torch::Tensor> w;
  if (weights.has_value()) w = weights->detach().to(torch::kFloat32).contiguous();
  return {top_logp.detach().to(torch::kFloat32).contiguous(), idx.contiguous(), w};
}

// The loss as an autograd function of the logits, in C++ for the same reason as the policy's: of 48 x 32 000 the kernels take 13 us and a Python function 100.
struct DistillFn : torch::autograd::Function<DistillFn> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, torch::Tensor logits, torch::Tensor top_logp, torch::Tensor top_idx,
                                                c10::optional<torch::Tensor> weights, double inv_temp, double beta, bool tail, bool want_grad) {
    auto [loss, token, grad] = distill_loss(logits, top_logp, top_idx, weights, inv_temp, beta, tail, want_grad, false, true);
    if (want_grad) {
      ctx->save_for_backward({grad});
      ctx->saved_data["capture"] = capture_id();
    }
    ctx->mark_non_differentiable({token});
    return {loss, token};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list g) {
    return {scaled(ctx->get_saved_variables()[0], g[0], ctx->saved_data["capture"].toInt()), {}, {}, {}, {}, {}, {}, {}};
  }
};
std::tuple<torch::Tensor, torch::Tensor> distill_loss_fn(const torch::Tensor& logits, const torch::Tensor& top_logp, const torch::Tensor& top_idx,
                                                         const c10::optional<torch::Tensor>& weights, double inv_temp, double beta, bool tail) {
  auto [logp, idx, w] = teacher_entries(top_logp, top_idx, weights, logits.size(1));
  const torch::Tensor rows = logits.stride(1) == 1 || logits.size(1) == 1 ? logits : logits.contiguous();
  auto out = DistillFn::apply(rows, logp, idx, w, inv_temp, beta, tail, at::GradMode::is_enabled() && logits.requires_grad());
  return {out[0], out[1]};
}

std::tuple<torch::Tensor, torch::Tensor> sample_filtered(const torch::Tensor& logits, const torch::Tensor& uniforms, const c10::optional<torch::Tensor>& temperature,
                                                         double temperature_all, const c10::optional<torch::Tensor>& top_k, int64_t top_k_all,
                                                         const c10::optional<torch::Tensor>& top_p, double top_p_all,
                                                         const c10::optional<torch::Tensor>& min_p, double min_p_all) {
  check_logits(logits, "sample_filtered");
  const int64_t rows = logits.size(0);
  check_beside(uniforms, logits, torch::kFloat32, {rows}, "sample_filtered", "uniforms");
  const auto floats = [&](const c10::optional<torch::Tensor>& t, const char* name) -> const float* {
    if (!t.has_value()) return nullptr;
    check_beside(*t, logits, torch::kFloat32, {rows}, "sample_filtered", name);
    return t->data_ptr<float>();
  };
  SampleFilters f{};
  f.temperature = floats(temperature, "temperature");
  f.top_p = floats(top_p, "top_p");
  f.min_p = floats(min_p, "min_p");
  if (top_k.has_value()) {
    check_beside(*top_k, logits, torch::kInt32, {rows}, "sample_filtered", "top_k");
    f.top_k = top_k->data_ptr<int>();
  }
  f.temperature_all = temperature_all;
  f.top_p_all = top_p_all;
  f.min_p_all = min_p_all;
  f.top_k_all = static_cast<int>(std::min<int64_t>(top_k_all, logits.size(1)));
  c10::cuda::CUDAGuard guard(logits.device());
  torch::Tensor tokens = torch::empty({rows}, logits.options().dtype(torch::kInt32)), logp = torch::empty({rows}, logits.options().dtype(torch::kFloat32));
  torch::Tensor top;
  if (!nrl_sample_is_short(&f, logits.size(1))) top = torch::empty({rows}, logp.options());
  const torch::Tensor scratch = scratch_of(nrl_sample_scratch(is_bf16(logits), rows, logits.size(1), &f), logits);
  check(nrl_sample_filtered(logits.data_ptr(), is_bf16(logits), logits.stride(0), rows, logits.size(1), uniforms.data_ptr<float>(), &f, tokens.data_ptr<int>(),
                            logp.data_ptr<float>(), static_cast<float*>(ptr_of(top)), ptr_of(scratch), cur_stream()), "sample_filtered");
  return {tokens, logp};
}

torch::Tensor row_uniforms(int64_t seed, int64_t step, const torch::Tensor& row_ids, const c10::optional<torch::Tensor>& row_steps) {
  TORCH_CHECK(row_ids.is_cuda() && row_ids.dim() == 1, "row_uniforms: row_ids must be a CUDA tensor [rows]");
  check_beside(row_ids, row_ids, torch::kInt32, row_ids.sizes(), "row_uniforms", "row_ids");
  if (row_steps.has_value()) check_beside(*row_steps, row_ids, torch::kInt32, row_ids.sizes(), "row_uniforms", "row_steps");
  c10::cuda::CUDAGuard guard(row_ids.device());
  torch::Tensor out = torch::empty(row_ids.sizes(), row_ids.options().dtype(torch::kFloat32));
  check(nrl_row_uniforms(static_cast<unsigned long long>(seed), static_cast<unsigned long long>(step), row_ids.data_ptr<int>(),
                         row_steps.has_value() ? row_steps->data_ptr<int>() : nullptr, row_ids.numel(), out.data_ptr<float>(), cur_stream()), "row_uniforms");
  return out;
}

}  // namespace

namespace nrl {

void bind_vocab(pybind11::module_& m) {
  namespace py = pybind11;
  m.def("top_logprobs", &top_logprobs, py::arg("logits"), py::arg("k"), py::arg("inv_temp"));
  m.def("distill_loss", &distill_loss_fn);
  m.def("teacher_entries", &teacher_entries);
  m.def("scaled", &scaled);
  m.def("refuse_second", &refuse_second);
  m.def("distill_loss_parts", &distill_loss, py::arg("logits"), py::arg("top_logp"), py::arg("top_idx"), py::arg("weights"), py::arg("inv_temp"), py::arg("beta"),
        py::arg("tail"), py::arg("want_grad"), py::arg("bf16_grad"), py::arg("with_loss"));
  m.def("weighted_sum", &weighted_sum);
  m.def("capture_id", &capture_id);
  m.def("sample_filtered", &sample_filtered);
  m.def("row_uniforms", &row_uniforms, py::arg("seed"), py::arg("step"), py::arg("row_ids"), py::arg("row_steps") = py::none());
}

}  // namespace nrl
