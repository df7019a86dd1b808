// Torch-facing shim of the gated scan: argument checks (TypeError / ValueError), output tensors, the
// metadata ticket of the packed forms; raw pointers and torch's current stream go to the C ABI.  No arithmetic here.
#include "bindings.h"

#include <limits>

#include "argument_checks.h"
#include "metadata_ticket.h"

namespace {

using namespace frwkv_bindings;

int input_code(const std::string& input_mode) {
  need_value(input_mode == "unit" || input_mode == "complement", "input_mode must be 'unit' or 'complement'");
  return input_mode == "unit" ? FRWKV_INPUT_UNIT : FRWKV_INPUT_COMPLEMENT;
}

int decay_code_checked(const std::string& decay_mode) {
  need_value(decay_mode == "logits" || decay_mode == "retention", "decay_mode must be 'logits' or 'retention'");
  return decay_code(decay_mode);
}

struct RowsShape {
  int64_t sequences;  // dense: the batch; packed: 0
  int64_t total, channels, x_stride, decay_stride;
};

// Distance between the rows of a [T, C] or [B, T, C] tensor whose rows lie at one regular distance.
int64_t row_stride(const torch::Tensor& t, const char* name) {
  const int64_t c = t.dim() - 1;
  need_value(t.stride(c) == 1 || t.size(c) == 1, std::string(name) + " must have unit stride along its channels");
  if (t.dim() == 3 && t.size(0) > 1 && t.size(1) > 1)
    need_value(t.stride(0) == t.size(1) * t.stride(1),
               std::string(name) + " must have its rows at one regular distance (make it contiguous)");
  if (t.dim() == 3 && t.size(1) == 1) return t.size(0) > 1 ? t.stride(0) : t.size(2);
  return t.size(c - 1) > 1 ? t.stride(c - 1) : t.size(c);
}

RowsShape check_tokens(const torch::Tensor& x, const torch::Tensor& decay, bool packed) {
  need_value(x.dim() == (packed ? 2 : 3), packed ? "x must have packed shape [total_tokens,C]" : "x must have shape [B,T,C]");
  need_value(x.numel() > 0, "x must have nonzero dimensions");
  need_type(x.scalar_type() == torch::kBFloat16 || x.scalar_type() == torch::kFloat16 || x.scalar_type() == torch::kFloat32,
            "x must be bfloat16, float16 or float32");
  need_type(decay.scalar_type() == x.scalar_type(), "decay_logits must have x's dtype");
  need_value(decay.sizes() == x.sizes(), "decay_logits must have x's shape");
  const int64_t channels = x.size(x.dim() - 1);
  const int64_t total = x.numel() / channels;
  need_value(total <= std::numeric_limits<int>::max() && channels <= std::numeric_limits<int>::max(),
             "token and channel counts must fit in int32");
  RowsShape s{packed ? 0 : x.size(0), total, channels, row_stride(x, "x"), row_stride(decay, "decay_logits")};
  need_value(packed || s.sequences <= 65535, "the batch must hold at most 65535 sequences");
  return s;
}

void check_token_devices(const torch::Tensor& x, const torch::Tensor& decay) {
  need_value(x.is_cuda(), "x must be CUDA");
  need_value(decay.device() == x.device(), "decay_logits must share x's device");
}

void check_fp32(const torch::Tensor& t, at::IntArrayRef shape, const char* name,
                const char* shape_text) {
  need_type(t.scalar_type() == torch::kFloat32, std::string(name) + " must have dtype float32");
  need_value(t.sizes() == shape, std::string(name) + " must have shape " + shape_text);
  need_value(t.is_contiguous(), std::string(name) + " must be contiguous");
}

void* optional_pointer(const std::optional<torch::Tensor>& t) { return t.has_value() ? t->data_ptr() : nullptr; }

struct Serving {
  int mode, input;
  RowsShape rows;
};

// Everything that can be said of a serving call without its metadata's values.
Serving check_serving(const torch::Tensor& query_start_loc, const torch::Tensor& state_indices, const torch::Tensor& state,
                      const torch::Tensor& x, const torch::Tensor& decay_logits, const std::optional<torch::Tensor>& decay_bias,
                      const TicketPtr& validated_metadata, const std::string& decay_mode, const std::string& input_mode) {
  const int mode = decay_code_checked(decay_mode), input = input_code(input_mode);
  need_value(query_start_loc.dim() == 1 && state_indices.dim() == 1 && state_indices.numel() > 0 &&
                 state_indices.numel() <= 65535 && query_start_loc.numel() == state_indices.numel() + 1,
             "cu_seqlens must have shape [N+1] and state_indices shape [N], with 1..65535 sequences");
  need_type(query_start_loc.scalar_type() == torch::kInt32 && state_indices.scalar_type() == torch::kInt32,
            "cu_seqlens and state_indices must be int32");
  need_value(query_start_loc.is_contiguous() && state_indices.is_contiguous(),
             "cu_seqlens and state_indices must be contiguous");
  need_value(x.dim() == 2, "x must have packed shape [total_tokens,C]");
  need_value(state.dim() == 2 && state.size(0) > 0 && state.size(0) <= std::numeric_limits<int>::max() &&
                 state.size(1) == x.size(1),
             "state_pool must have shape [slots,C] with x's channels");
  need_type(state.scalar_type() == torch::kFloat32, "state_pool must have dtype float32");
  need_value(state.is_contiguous(), "state_pool must be contiguous");
  if (decay_bias.has_value()) {
    need_value(mode == FRWKV_DECAY_LOGITS, "decay_bias only applies to decay logits");
    need_value(decay_bias->dim() == 1 && decay_bias->numel() == x.size(1) && decay_bias->is_contiguous(),
               "decay_bias must be contiguous with shape [C]");
    need_type(decay_bias->scalar_type() == x.scalar_type(), "decay_bias must have x's dtype");
  }
  const RowsShape s = check_tokens(x, decay_logits, true);
  // (a capacity ticket may have room for more sequences than tokens: those beyond are not active)
  need_value(s.total >= state_indices.numel() || (validated_metadata && validated_metadata->graph_mode()),
             "every sequence needs a token");
  check_token_devices(x, decay_logits);
  need_value(state.device() == x.device() && query_start_loc.device() == x.device() &&
                 state_indices.device() == x.device() && (!decay_bias.has_value() || decay_bias->device() == x.device()),
             "state_pool, cu_seqlens, state_indices and decay_bias must share x's device");
  return Serving{mode, input, s};
}

// For a caller that has the metadata of a call validated before it makes it: refusals come first.
void check_tmix_gated_scan_fp32(const torch::Tensor& query_start_loc, const torch::Tensor& state_indices,
                                const torch::Tensor& state, const torch::Tensor& x, const torch::Tensor& decay_logits,
                                const std::optional<torch::Tensor>& decay_bias, const TicketPtr& validated_metadata,
                                int64_t, const std::string& decay_mode, const std::string& input_mode) {
  check_serving(query_start_loc, state_indices, state, x, decay_logits, decay_bias, validated_metadata, decay_mode, input_mode);
}

torch::Tensor tmix_gated_scan_fp32(const torch::Tensor& query_start_loc, const torch::Tensor& state_indices,
                                   const torch::Tensor& state, const torch::Tensor& x, const torch::Tensor& decay_logits,
                                   const std::optional<torch::Tensor>& decay_bias, const TicketPtr& validated_metadata,
                                   int64_t max_seqlen, const std::string& decay_mode, const std::string& input_mode) {
  const auto [mode, input, s] = check_serving(query_start_loc, state_indices, state, x, decay_logits, decay_bias,
                                              validated_metadata, decay_mode, input_mode);
  const c10::cuda::CUDAGuard guard(x.device());
  const auto meta = resolve_metadata(query_start_loc, state_indices, state, x, validated_metadata, max_seqlen);
  auto y = torch::empty(x.sizes(), x.options());
  check_abi(frwkv_sm100_gated_scan(
      meta.cu.data_ptr<int>(), meta.slots.data_ptr<int>(), meta.status.data_ptr<int>(), state.data_ptr<float>(),
      x.data_ptr(), s.x_stride, decay_logits.data_ptr(), s.decay_stride, optional_pointer(decay_bias), y.data_ptr(),
      static_cast<int>(state_indices.numel()), static_cast<int>(s.total), static_cast<int>(s.channels), io_code(x), mode,
      input, static_cast<int>(meta.max_seqlen),
      at::cuda::getCurrentCUDAStream(x.device().index()).stream()));
  return y;
}

using Optional = std::optional<torch::Tensor>;

// Sequence count of a training call, and for packed rows the validated copy of cu_seqlens with its status word.
// The validation runs on the device and nothing waits for it: bad bounds make every output NaN.
std::tuple<int64_t, Optional, Optional> resolve_rows(const RowsShape& s, const torch::Tensor& x, const Optional& cu_seqlens) {
  if (!cu_seqlens.has_value()) return {s.sequences, std::nullopt, std::nullopt};
  const int64_t n = cu_seqlens->numel() - 1;
  const auto slots = torch::arange(n, cu_seqlens->options());
  const auto prepared = launch_validation(*cu_seqlens, slots, torch::Tensor(), torch::Tensor(), s.total, n, n, s.total, true);
  return {n, prepared.cu, prepared.status};
}

struct Forward {
  torch::Tensor y, final_state, boundary;
  Optional cu, status;
};

Forward train_forward(const torch::Tensor& x, const torch::Tensor& decay_logits,
                      const Optional& initial_state, const Optional& cu_seqlens, const std::string& decay_mode,
                      const std::string& input_mode) {
  const int mode = decay_code_checked(decay_mode), input = input_code(input_mode);
  if (cu_seqlens.has_value()) {
    need_type(cu_seqlens->scalar_type() == torch::kInt32, "cu_seqlens must have dtype int32");
    need_value(cu_seqlens->dim() == 1 && cu_seqlens->numel() >= 2 && cu_seqlens->numel() <= 65536 &&
                   cu_seqlens->is_contiguous(),
               "cu_seqlens must be contiguous with shape [N+1], 1..65535 sequences");
  }
  const RowsShape s = check_tokens(x, decay_logits, cu_seqlens.has_value());
  const int64_t n_given = cu_seqlens.has_value() ? cu_seqlens->numel() - 1 : s.sequences;
  need_value(s.total >= n_given, "every sequence needs a token");
  if (initial_state.has_value()) check_fp32(*initial_state, {n_given, s.channels}, "initial_state", "[N,C]");
  check_token_devices(x, decay_logits);
  if (initial_state.has_value()) need_value(initial_state->device() == x.device(), "initial_state must share x's device");
  if (cu_seqlens.has_value()) need_value(cu_seqlens->device() == x.device(), "cu_seqlens must share x's device");
  const c10::cuda::CUDAGuard guard(x.device());
  const auto [n, cu, status] = resolve_rows(s, x, cu_seqlens);
  auto y = torch::empty(x.sizes(), x.options());
  const auto fp32 = x.options().dtype(torch::kFloat32);
  auto final_state = torch::empty({n, s.channels}, fp32);
  auto boundary = torch::empty({s.total / FRWKV_GATED_SCAN_SAVED_ROWS + n, s.channels}, fp32);
  check_abi(frwkv_sm100_gated_scan_train_forward(
      static_cast<const int32_t*>(optional_pointer(cu)), static_cast<const int32_t*>(optional_pointer(status)),
      x.data_ptr(), s.x_stride, decay_logits.data_ptr(), s.decay_stride,
      static_cast<const float*>(optional_pointer(initial_state)), y.data_ptr(), final_state.data_ptr<float>(),
      boundary.data_ptr<float>(), static_cast<int>(n), static_cast<int>(s.total), static_cast<int>(s.channels),
      io_code(x), mode, input, -1, at::cuda::getCurrentCUDAStream(x.device().index()).stream()));
  return Forward{y, final_state, boundary, cu, status};
}

torch::autograd::variable_list train_backward(const torch::Tensor& x, const torch::Tensor& decay_logits, const Optional& initial_state, const Optional& cu, const Optional& status,
                                            const torch::Tensor& boundary, const torch::Tensor& grad_output,
                                            const Optional& grad_final, const std::string& decay_mode,
                                            const std::string& input_mode) {
  const int mode = decay_code_checked(decay_mode), input = input_code(input_mode);
  const RowsShape s = check_tokens(x, decay_logits, cu.has_value());
  const int64_t n = cu.has_value() ? cu->numel() - 1 : s.sequences;
  check_token_devices(x, decay_logits);
  need_type(grad_output.scalar_type() == x.scalar_type(), "grad_output must have x's dtype");
  need_value(grad_output.sizes() == x.sizes() && grad_output.is_contiguous() && grad_output.device() == x.device(),
             "grad_output must be contiguous with x's shape and device");
  check_fp32(boundary, {s.total / FRWKV_GATED_SCAN_SAVED_ROWS + n, s.channels}, "boundary", "[saved rows,C]");
  if (initial_state.has_value()) check_fp32(*initial_state, {n, s.channels}, "initial_state", "[N,C]");
  if (grad_final.has_value()) check_fp32(*grad_final, {n, s.channels}, "grad_final", "[N,C]");
  const c10::cuda::CUDAGuard guard(x.device());
  auto dx = torch::empty(x.sizes(), x.options());
  auto ddecay = torch::empty(x.sizes(), x.options());
  Optional dinitial;
  if (initial_state.has_value()) dinitial = torch::empty_like(*initial_state);
  check_abi(frwkv_sm100_gated_scan_train_backward(
      static_cast<const int32_t*>(optional_pointer(cu)), static_cast<const int32_t*>(optional_pointer(status)),
      x.data_ptr(), s.x_stride, decay_logits.data_ptr(), s.decay_stride,
      static_cast<const float*>(optional_pointer(initial_state)), boundary.data_ptr<float>(), grad_output.data_ptr(),
      static_cast<const float*>(optional_pointer(grad_final)), dx.data_ptr(), ddecay.data_ptr(),
      static_cast<float*>(optional_pointer(dinitial)), static_cast<int>(n), static_cast<int>(s.total),
      static_cast<int>(s.channels), io_code(x), mode, input, -1,
      at::cuda::getCurrentCUDAStream(x.device().index()).stream()));
  return {dx, ddecay, dinitial.value_or(torch::Tensor())};
}

Optional defined(const torch::Tensor& t) { return t.defined() ? Optional(t) : std::nullopt; }

class TrainFunction : public torch::autograd::Function<TrainFunction> {
 public:
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const torch::Tensor& x,
                                                const torch::Tensor& decay_logits, const Optional& initial_state,
                                                const Optional& cu_seqlens, const std::string& decay_mode,
                                                const std::string& input_mode) {
    const Forward f = train_forward(x, decay_logits, initial_state, cu_seqlens, decay_mode, input_mode);
    ctx->save_for_backward({x, decay_logits, initial_state.value_or(torch::Tensor()), f.cu.value_or(torch::Tensor()), f.status.value_or(torch::Tensor()), f.boundary});
    ctx->saved_data["decay_mode"] = decay_mode;
    ctx->saved_data["input_mode"] = input_mode;
    ctx->set_materialize_grads(false);
    return {f.y, f.final_state};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto& x = saved[0];
    const auto grad_output = grads[0].defined() ? grads[0].contiguous() : torch::zeros(x.sizes(), x.options());
    const auto grad_final = grads[1].defined() ? Optional(grads[1].contiguous()) : std::nullopt;
    auto out = train_backward(x, saved[1], defined(saved[2]), defined(saved[3]), defined(saved[4]), saved[5], grad_output, grad_final,
                              ctx->saved_data["decay_mode"].toStringRef(), ctx->saved_data["input_mode"].toStringRef());
    out.resize(6);
    return differentiable_once(std::move(out), "the gated scan");
  }
};

// (y, final_state), differentiable in x, decay_logits and initial_state.
std::tuple<torch::Tensor, torch::Tensor> pretrain_tmix_gated_scan(const torch::Tensor& x, const torch::Tensor& decay_logits,
                                                                  const Optional& initial_state, const Optional& cu_seqlens,
                                                                  const std::string& decay_mode, const std::string& input_mode) {
  const bool differentiable = torch::GradMode::is_enabled() && (x.requires_grad() || decay_logits.requires_grad() ||
                                                               (initial_state.has_value() && initial_state->requires_grad()));
  if (!differentiable) {
    const Forward f = train_forward(x, decay_logits, initial_state, cu_seqlens, decay_mode, input_mode);
    return {f.y, f.final_state};
  }
  const auto out = TrainFunction::apply(x, decay_logits, initial_state, cu_seqlens, decay_mode, input_mode);
  return {out[0], out[1]};
}

}  // namespace

void register_tmix_gated_scan_bindings(py::module_& module) {
  const auto serving = [&](const char* name, auto function, const char* what) {
    module.def(name, function, what, py::arg("query_start_loc"), py::arg("state_indices"), py::arg("state"), py::arg("x"),
               py::arg("decay_logits"), py::arg("decay_bias") = py::none(), py::arg("validated_metadata") = py::none(),
               py::arg("max_seqlen") = -1, py::arg("decay_mode") = "logits", py::arg("input_mode") = "unit");
  };
  serving("tmix_gated_scan_fp32", &tmix_gated_scan_fp32, "Gated scan over packed rows, fp32 state in place");
  serving("check_tmix_gated_scan_fp32", &check_tmix_gated_scan_fp32, "The refusals of tmix_gated_scan_fp32 alone");
  module.def("pretrain_tmix_gated_scan", &pretrain_tmix_gated_scan, "Differentiable gated scan: (y, final_state)",
             py::arg("x"), py::arg("decay_logits"), py::arg("initial_state") = py::none(), py::arg("cu_seqlens") = py::none(),
             py::arg("decay_mode") = "logits", py::arg("input_mode") = "unit");
}
