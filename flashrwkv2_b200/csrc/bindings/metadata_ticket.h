// Pieces that every binding over packed sequences shares: elementary tensor checks, the metadata ticket and its
// resolution into what a launch needs.
#pragma once

#include "bindings.h"

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <memory>
#include <optional>
#include <string>
#include <utility>
#include <vector>

#include "frwkv_sm100.h"

namespace frwkv_bindings {

inline void check_abi(int rc) { TORCH_CHECK(rc == 0, frwkv_sm100_last_error()); }

inline void check_cuda_contiguous(const torch::Tensor& tensor, const char* name) {
  TORCH_CHECK(tensor.is_cuda(), name, " must be CUDA");
  TORCH_CHECK(tensor.is_contiguous(), name, " must be contiguous");
}

inline void check_same_device(const torch::Tensor& reference, const torch::Tensor& tensor, const char* name) {
  TORCH_CHECK(tensor.device() == reference.device(), name, " must be on the same device as state");
}

inline int io_code(const torch::Tensor& tokens) {
  switch (tokens.scalar_type()) {
    case torch::kBFloat16: return FRWKV_IO_BF16;
    case torch::kFloat16: return FRWKV_IO_FP16;
    default: return FRWKV_IO_FP32;
  }
}

inline int decay_code(const std::string& decay_mode) {
  TORCH_CHECK(decay_mode == "logits" || decay_mode == "retention", "decay_mode must be 'logits' or 'retention'");
  return decay_mode == "logits" ? FRWKV_DECAY_LOGITS : FRWKV_DECAY_RETENTION;
}

inline std::optional<uint32_t> tensor_version(const torch::Tensor& tensor) {
  if (tensor.unsafeGetTensorImpl()->is_inference()) return std::nullopt;
  return tensor.unsafeGetTensorImpl()->version_counter().current_version();
}

struct Prepared {
  torch::Tensor cu, slots, status, workspace;
};

// One launch of the validation kernel on the current stream of the metadata's device.
inline Prepared launch_validation(const torch::Tensor& query_start_loc, const torch::Tensor& state_indices,
                           const torch::Tensor& num_active_tokens, const torch::Tensor& num_active_sequences,
                           int64_t token_capacity, int64_t sequence_capacity, int64_t state_pool_size,
                           int64_t max_seqlen, bool snapshot) {
  const c10::cuda::CUDAGuard guard(query_start_loc.device());
  auto status = torch::empty({3}, query_start_loc.options());
  auto seen = torch::empty({state_pool_size}, query_start_loc.options());
  auto cu_snap = snapshot ? torch::empty_like(query_start_loc) : query_start_loc;
  auto slots_snap = snapshot ? torch::empty_like(state_indices) : state_indices;
  check_abi(frwkv_sm100_wkv7_validate_metadata(
      query_start_loc.data_ptr<int>(), state_indices.data_ptr<int>(), static_cast<int>(sequence_capacity),
      static_cast<int>(token_capacity), static_cast<int>(state_pool_size), static_cast<int>(max_seqlen),
      num_active_tokens.defined() ? num_active_tokens.data_ptr<int>() : nullptr,
      num_active_sequences.defined() ? num_active_sequences.data_ptr<int>() : nullptr, status.data_ptr<int>(),
      seen.data_ptr<int>(), snapshot ? cu_snap.data_ptr<int>() : nullptr,
      snapshot ? slots_snap.data_ptr<int>() : nullptr,
      at::cuda::getCurrentCUDAStream(query_start_loc.device().index()).stream()));
  return Prepared{std::move(cu_snap), std::move(slots_snap), std::move(status), std::move(seen)};
}

// Validated packed-sequence metadata bound to one stream (counterpart of the reference's
// RecurrentMetadataTicket, infer_recurrent_fp32io16_forward_varlen.cpp:89-225).
class RecurrentMetadataTicket final {
 public:
  RecurrentMetadataTicket(torch::Tensor query_start_loc, torch::Tensor state_indices, Prepared prepared,
                          torch::Tensor num_active_tokens, torch::Tensor num_active_sequences, int64_t total_tokens,
                          int64_t state_pool_size, int64_t max_seqlen, bool graph_mode, cudaStream_t stream)
      : cu_(std::move(query_start_loc)), slots_(std::move(state_indices)), prepared_(std::move(prepared)),
        n_tok_(std::move(num_active_tokens)), n_seq_(std::move(num_active_sequences)),
        cu_version_(tensor_version(cu_)), slots_version_(tensor_version(slots_)), cu_data_(cu_.data_ptr()),
        slots_data_(slots_.data_ptr()), cu_sizes_(cu_.sizes().vec()), slots_sizes_(slots_.sizes().vec()),
        cu_strides_(cu_.strides().vec()), slots_strides_(slots_.strides().vec()), total_tokens_(total_tokens),
        state_pool_size_(state_pool_size), max_seqlen_(max_seqlen), graph_mode_(graph_mode), device_(cu_.device()),
        stream_(stream) {}

  void check_compatible(const torch::Tensor& query_start_loc, const torch::Tensor& state_indices,
                        int64_t total_tokens, int64_t state_pool_size, int64_t max_seqlen) const {
    TORCH_CHECK(query_start_loc.is_same(cu_), "validated_metadata query_start_loc identity mismatch");
    TORCH_CHECK(state_indices.is_same(slots_), "validated_metadata state_indices identity mismatch");
    TORCH_CHECK(query_start_loc.data_ptr() == cu_data_ && state_indices.data_ptr() == slots_data_,
                "validated_metadata metadata data_ptr mismatch");
    TORCH_CHECK(query_start_loc.sizes().vec() == cu_sizes_ && state_indices.sizes().vec() == slots_sizes_ &&
                    query_start_loc.strides().vec() == cu_strides_ && state_indices.strides().vec() == slots_strides_,
                "validated_metadata metadata shape or stride mismatch");
    if (!graph_mode_ && cu_version_.has_value())
      TORCH_CHECK(tensor_version(query_start_loc) == cu_version_, "validated_metadata query_start_loc version mismatch");
    if (!graph_mode_ && slots_version_.has_value())
      TORCH_CHECK(tensor_version(state_indices) == slots_version_, "validated_metadata state_indices version mismatch");
    TORCH_CHECK(query_start_loc.device() == device_ && state_indices.device() == device_,
                "validated_metadata device mismatch");
    TORCH_CHECK(total_tokens == total_tokens_, "validated_metadata total_tokens mismatch");
    TORCH_CHECK(state_pool_size == state_pool_size_, "validated_metadata state_pool_size mismatch");
    if (max_seqlen > 0) TORCH_CHECK(max_seqlen == max_seqlen_, "validated_metadata max_seqlen mismatch");
    TORCH_CHECK(at::cuda::getCurrentCUDAStream(device_.index()).stream() == stream_,
                "validated_metadata stream mismatch; prepare and consume the ticket on the same CUDA stream");
  }

  const torch::Tensor& cu_snapshot() const { return prepared_.cu; }
  const torch::Tensor& slots_snapshot() const { return prepared_.slots; }
  const torch::Tensor& status() const { return prepared_.status; }
  int64_t max_seqlen() const { return max_seqlen_; }
  bool graph_mode() const { return graph_mode_; }
  const torch::Tensor& num_active_tokens() const { return n_tok_; }
  const torch::Tensor& num_active_sequences() const { return n_seq_; }

 private:
  torch::Tensor cu_, slots_;
  Prepared prepared_;
  torch::Tensor n_tok_, n_seq_;
  std::optional<uint32_t> cu_version_, slots_version_;
  void* cu_data_;
  void* slots_data_;
  std::vector<int64_t> cu_sizes_, slots_sizes_, cu_strides_, slots_strides_;
  int64_t total_tokens_, state_pool_size_, max_seqlen_;
  bool graph_mode_;
  c10::Device device_;
  cudaStream_t stream_;
};

using TicketPtr = std::shared_ptr<RecurrentMetadataTicket>;

struct Resolved {
  torch::Tensor cu, slots, status;
  int64_t max_seqlen;
  torch::Tensor keep;  // scratch of an un-ticketed validation, kept alive until the launch is enqueued
};

inline Resolved resolve_metadata(const torch::Tensor& query_start_loc, const torch::Tensor& state_indices,
                          const torch::Tensor& state, const torch::Tensor& r, const TicketPtr& ticket,
                          int64_t max_seqlen) {
  if (ticket) {
    ticket->check_compatible(query_start_loc, state_indices, r.size(0), state.size(0), max_seqlen);
    return Resolved{ticket->cu_snapshot(), ticket->slots_snapshot(), ticket->status(), ticket->max_seqlen(),
                    torch::Tensor()};
  }
  // un-ticketed native call: device validation only (the raising host check belongs to the static
  // prepare entry, as in the reference binding :375-381)
  auto prepared = launch_validation(query_start_loc, state_indices, torch::Tensor(), torch::Tensor(), r.size(0),
                                    state_indices.numel(), state.size(0), r.size(0), true);
  return Resolved{prepared.cu, prepared.slots, prepared.status, max_seqlen, prepared.workspace};
}

}  // namespace frwkv_bindings
