// Torch-facing shim of the token log probabilities: argument checks (TypeError / ValueError), the row geometry of
// strided logits, output tensors; raw pointers and torch's current stream go to the C ABI.  No arithmetic here.
#include "bindings.h"

#include <limits>
#include <vector>

#include "argument_checks.h"
#include "metadata_ticket.h"

namespace {

using namespace frwkv_bindings;
using Optional = std::optional<torch::Tensor>;

struct RowsShape {
  int64_t outer, inner, stride_outer, stride_inner, vocab;
};

// The rows of [..., V] logits as two nested loops: dimensions that lie behind one another are joined, which leaves two
// for a slice such as logits[:, :-1].
RowsShape row_shape(const torch::Tensor& logits) {
  const int64_t last = logits.dim() - 1;
  std::vector<std::pair<int64_t, int64_t>> dims;  // size, stride
  for (int64_t d = 0; d < last; ++d) {
    if (logits.size(d) == 1) continue;
    if (!dims.empty() && dims.back().second == logits.size(d) * logits.stride(d))
      dims.back() = {dims.back().first * logits.size(d), logits.stride(d)};
    else
      dims.emplace_back(logits.size(d), logits.stride(d));
  }
  need_value(dims.size() <= 2, "logits must have rows that two strides describe (make them contiguous)");
  while (dims.size() < 2) dims.insert(dims.begin(), {1, 0});
  return RowsShape{dims[0].first, dims[1].first, dims[0].second, dims[1].second, logits.size(last)};
}

RowsShape check_logits(const torch::Tensor& logits, const torch::Tensor& token_ids, double temperature) {
  need_value(logits.dim() >= 1 && logits.size(logits.dim() - 1) > 0, "logits must have shape [...,V] with V > 0");
  need_type(logits.scalar_type() == torch::kBFloat16 || logits.scalar_type() == torch::kFloat16 ||
                logits.scalar_type() == torch::kFloat32,
            "logits must be bfloat16, float16 or float32");
  need_type(token_ids.scalar_type() == torch::kInt64 || token_ids.scalar_type() == torch::kInt32,
            "token_ids must be int64 or int32");
  need_value(token_ids.sizes() == logits.sizes().slice(0, logits.dim() - 1),
             "token_ids must have the shape of logits without the vocabulary");
  const float t = static_cast<float>(temperature);
  need_value(t >= FRWKV_TEMPERATURE_MIN && t <= FRWKV_TEMPERATURE_MAX, "temperature must be in 1e-30..1e30");
  need_value(logits.size(logits.dim() - 1) <= std::numeric_limits<int>::max() &&
                 token_ids.numel() <= std::numeric_limits<int>::max(),
             "row and vocabulary counts must fit in int32");
  need_value(logits.stride(logits.dim() - 1) == 1 || logits.size(logits.dim() - 1) == 1,
             "logits must have unit stride along the vocabulary");
  const RowsShape s = token_ids.numel() > 0 ? row_shape(logits) : RowsShape{0, 0, 0, 0, logits.size(logits.dim() - 1)};
  need_value(logits.is_cuda(), "logits must be CUDA");
  need_value(token_ids.device() == logits.device(), "token_ids must share the device of logits");
  return s;
}

struct Forward {
  torch::Tensor logprobs, entropy, stats;
  Optional top_ids, top_logprobs;
};

Forward rows_forward(const torch::Tensor& logits, const torch::Tensor& token_ids, double temperature, int64_t top_k,
                     int64_t ignore_index) {
  need_value(top_k >= 0 && top_k <= FRWKV_TOP_K_MAX, "top_k must be in 0.." + std::to_string(FRWKV_TOP_K_MAX));
  const RowsShape s = check_logits(logits, token_ids, temperature);
  need_value(top_k <= s.vocab, "top_k must not exceed the vocabulary");
  const c10::cuda::CUDAGuard guard(logits.device());
  const auto ids = token_ids.contiguous();
  const auto fp32 = logits.options().dtype(torch::kFloat32);
  auto logprobs = torch::empty(token_ids.sizes(), fp32), entropy = torch::empty(token_ids.sizes(), fp32);
  auto stats = torch::empty({token_ids.numel(), 2}, fp32);
  Optional top_ids, top_logprobs;
  if (top_k > 0) {
    auto shape = token_ids.sizes().vec();
    shape.push_back(top_k);
    top_ids = torch::empty(shape, logits.options().dtype(torch::kInt64));
    top_logprobs = torch::empty(shape, fp32);
  }
  if (token_ids.numel() > 0)
    check_abi(frwkv_sm100_token_logprobs(
        logits.data_ptr(), s.outer, s.inner, s.stride_outer, s.stride_inner, ids.data_ptr(),
        ids.scalar_type() == torch::kInt64, ignore_index, static_cast<int>(s.vocab), io_code(logits),
        static_cast<float>(temperature), static_cast<int>(top_k), logprobs.data_ptr<float>(), entropy.data_ptr<float>(),
        stats.data_ptr<float>(), top_k > 0 ? top_ids->data_ptr<int64_t>() : nullptr,
        top_k > 0 ? top_logprobs->data_ptr<float>() : nullptr,
        at::cuda::getCurrentCUDAStream(logits.device().index()).stream()));
  return Forward{logprobs, entropy, stats, top_ids, top_logprobs};
}

torch::Tensor rows_backward(const torch::Tensor& logits, const torch::Tensor& token_ids, double temperature, int64_t ignore_index,
                            const torch::Tensor& stats, const torch::Tensor& entropy, const torch::Tensor& grad_logprobs,
                            const torch::Tensor& grad_entropy) {
  const RowsShape s = check_logits(logits, token_ids, temperature);
  const c10::cuda::CUDAGuard guard(logits.device());
  const auto ids = token_ids.contiguous();
  const auto row_gradient = [](const torch::Tensor& g) { return g.defined() ? g.contiguous() : g; };
  const auto dlp = row_gradient(grad_logprobs), dent = row_gradient(grad_entropy);
  auto dlogits = torch::empty(logits.sizes(), logits.options());
  if (token_ids.numel() > 0)
    check_abi(frwkv_sm100_token_logprobs_backward(
        logits.data_ptr(), s.outer, s.inner, s.stride_outer, s.stride_inner, ids.data_ptr(),
        ids.scalar_type() == torch::kInt64, ignore_index, static_cast<int>(s.vocab), io_code(logits),
        static_cast<float>(temperature), stats.data_ptr<float>(), entropy.data_ptr<float>(),
        dlp.defined() ? dlp.data_ptr<float>() : nullptr, dent.defined() ? dent.data_ptr<float>() : nullptr,
        dlogits.data_ptr(), at::cuda::getCurrentCUDAStream(logits.device().index()).stream()));
  return dlogits;
}

class RowsFunction : public torch::autograd::Function<RowsFunction> {
 public:
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const torch::Tensor& logits,
                                                const torch::Tensor& token_ids, double temperature, int64_t top_k,
                                                int64_t ignore_index) {
    const Forward f = rows_forward(logits, token_ids, temperature, top_k, ignore_index);
    ctx->save_for_backward({logits, token_ids, f.stats, f.entropy});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["ignore_index"] = ignore_index;
    ctx->set_materialize_grads(false);
    if (!f.top_ids.has_value()) return {f.logprobs, f.entropy};
    ctx->mark_non_differentiable({*f.top_ids, *f.top_logprobs});
    return {f.logprobs, f.entropy, *f.top_ids, *f.top_logprobs};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    torch::autograd::variable_list out{rows_backward(saved[0], saved[1], ctx->saved_data["temperature"].toDouble(),
                                                     ctx->saved_data["ignore_index"].toInt(), saved[2], saved[3], grads[0], grads[1])};
    out.resize(5);
    return differentiable_once(std::move(out), "the token log probabilities operator");
  }
};

// (logprobs, entropy, top_ids or None, top_logprobs or None), the first two differentiable in logits.
std::tuple<torch::Tensor, torch::Tensor, Optional, Optional> head_token_logprobs(const torch::Tensor& logits,
                                                                                 const torch::Tensor& token_ids, double temperature,
                                                                                 int64_t top_k, int64_t ignore_index) {
  if (!(torch::GradMode::is_enabled() && logits.requires_grad())) {
    const Forward f = rows_forward(logits, token_ids, temperature, top_k, ignore_index);
    return {f.logprobs, f.entropy, f.top_ids, f.top_logprobs};
  }
  const auto out = RowsFunction::apply(logits, token_ids, temperature, top_k, ignore_index);
  const bool top = out.size() > 2;
  return {out[0], out[1], top ? Optional(out[2]) : std::nullopt, top ? Optional(out[3]) : std::nullopt};
}

}  // namespace

void register_rl_infctx_head_token_logprobs_bindings(py::module_& module) {
  module.def("head_token_logprobs", &head_token_logprobs, "Log probabilities of given tokens, entropy and top alternatives",
             py::arg("logits"), py::arg("token_ids"), py::arg("temperature") = 1.0, py::arg("top_k") = 0,
             py::arg("ignore_index") = -100);
}
