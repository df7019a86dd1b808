// Arithmetic that the gated scan's kernels share.
//
//   h_t = rho_t * h_{t-1} + i_t * x_t,   rho = exp(-s), s = exp(-1/2) * sigmoid(logit + bias)   or rho itself.
// From logits the kernels work with delta = 1 - rho and write rho * h as h - delta * h: a slow channel has delta of
// 1e-4 and less, and rho rounded to fp32 would then be off by 2^-25 / delta of the decay it stands for, at every token
// with the same sign.  A retention that the caller gives is used as it is (1 - rho loses a small rho instead).
#pragma once

#include "../../common.cuh"

namespace frwkv {

struct GatedScanParams {
  const int* cu;      // [n_seq + 1], or null: sequences of `seq_len` rows each
  const int* slots;   // [n_seq], or null: sequence i has state row i
  const int* status;  // {error, active tokens, active sequences}, or null: all of them
  const void *x, *decay, *bias;
  long long x_stride, decay_stride;
  const float* initial;  // read at the first token of a sequence; null: zeros
  float* final_state;    // written behind the last token (the pool itself for the in-place operator)
  float* boundary;       // training: the state before every FRWKV_GATED_SCAN_TILE-th row
  void* y;
  int n_seq, total, channels, seq_len;
};

template <bool LOGITS> struct Decay {
  float rho, delta;  // LOGITS: only delta is used by step()
  float slope;       // d(1 - rho) / d logit = s (1 - sigmoid) rho
  __device__ __forceinline__ void set(float d) {
    if constexpr (LOGITS) {
      const float gate = 1.0f / (1.0f + exp2f(-kLog2e * d));
      delta = -expm1f(-kRate * gate);
      rho = 1.0f - delta;
      slope = kRate * gate * (1.0f - gate) * rho;
    } else {
      rho = d;
      delta = 1.0f - d;
      slope = -1.0f;
    }
  }
  __device__ __forceinline__ float step(float h, float u) const {
    if constexpr (LOGITS) return h + fmaf(-delta, h, u);
    else return fmaf(rho, h, u);
  }
};

}  // namespace frwkv
