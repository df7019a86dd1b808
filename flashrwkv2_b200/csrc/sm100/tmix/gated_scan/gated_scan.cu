// Gated scan: in-place serving operator and training forward / backward (see gated_scan.cuh for the arithmetic).
//
// One thread walks one channel of one sequence token by token.
#include "gated_scan.cuh"

namespace frwkv {
namespace {

constexpr int kThreads = 128;
constexpr int kTile = FRWKV_GATED_SCAN_TILE;

struct Span {
  int begin, end;
};

__device__ __forceinline__ Span sequence_span(const GatedScanParams& p, int seq) {
  if (p.cu == nullptr) return Span{seq * p.seq_len, (seq + 1) * p.seq_len};
  return Span{p.cu[seq], p.cu[seq + 1]};
}

template <typename io_t, bool LOGITS, bool COMPLEMENT>
__global__ void __launch_bounds__(kThreads) gated_scan_forward_kernel(const GatedScanParams p) {
  const long long channel = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x;
  const int seq = blockIdx.y;
  io_t* y = static_cast<io_t*>(p.y);
  if (p.status != nullptr && p.status[0] != 0) {
    const long long threads = static_cast<long long>(gridDim.x) * gridDim.y * kThreads;
    const long long self = (static_cast<long long>(seq) * gridDim.x + blockIdx.x) * kThreads + threadIdx.x;
    fill_output_nan(y, nullptr, static_cast<long long>(p.total) * p.channels, self, threads);
    if (p.boundary != nullptr && channel < p.channels) p.final_state[seq * static_cast<long long>(p.channels) + channel] = __int_as_float(0x7fffffff);
    return;
  }
  if (channel >= p.channels || (p.status != nullptr && seq >= p.status[2])) return;
  const io_t* x = static_cast<const io_t*>(p.x) + channel;
  const io_t* decay = static_cast<const io_t*>(p.decay) + channel;
  const float bias = p.bias != nullptr ? to_f32(static_cast<const io_t*>(p.bias)[channel]) : 0.f;
  const Span span = sequence_span(p, seq);
  const long long state = static_cast<long long>(p.slots != nullptr ? p.slots[seq] : seq) * p.channels + channel;
  float h = p.initial != nullptr ? p.initial[state] : 0.f;
  for (long long t = span.begin; t < span.end; ++t) {
    if (p.boundary != nullptr && t % kTile == 0) p.boundary[t / kTile * p.channels + channel] = h;
    Decay<LOGITS> d;
    d.set(to_f32(decay[t * p.decay_stride]) + bias);
    const float value = to_f32(x[t * p.x_stride]);
    h = d.step(h, COMPLEMENT ? d.delta * value : value);
    y[t * p.channels + channel] = from_f32<io_t>(h);
  }
  p.final_state[state] = h;
}

struct GatedScanGrads {
  const void* dy;
  const float* dfinal;
  void *dx, *ddecay;
  float* dinitial;
};

template <typename io_t, bool LOGITS, bool COMPLEMENT>
__global__ void __launch_bounds__(kThreads) gated_scan_backward_kernel(const GatedScanParams p, const GatedScanGrads g) {
  const long long channel = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x;
  const int seq = blockIdx.y;
  if (channel >= p.channels) return;
  io_t* dx = static_cast<io_t*>(g.dx) + channel;
  io_t* dd = static_cast<io_t*>(g.ddecay) + channel;
  const long long state = static_cast<long long>(seq) * p.channels + channel;
  if (p.status != nullptr && p.status[0] != 0) {
    const float qnan = __int_as_float(0x7fffffff);
    for (long long t = seq; t < p.total; t += gridDim.y) dx[t * p.channels] = dd[t * p.channels] = from_f32<io_t>(qnan);
    if (g.dinitial != nullptr) g.dinitial[state] = qnan;
    return;
  }
  const io_t* x = static_cast<const io_t*>(p.x) + channel;
  const io_t* decay = static_cast<const io_t*>(p.decay) + channel;
  const io_t* dy = static_cast<const io_t*>(g.dy) + channel;
  const Span span = sequence_span(p, seq);
  float carry = g.dfinal != nullptr ? g.dfinal[state] : 0.f;
  float before[kTile];
  for (int tile = (span.end - 1) / kTile; tile >= span.begin / kTile; --tile) {
    const int first = max(span.begin, tile * kTile), last = min(span.end, (tile + 1) * kTile);
    float h = first > span.begin || span.begin % kTile == 0 ? p.boundary[static_cast<long long>(tile) * p.channels + channel]
              : p.initial != nullptr                        ? p.initial[state]
                                                            : 0.f;
    for (long long t = first; t < last; ++t) {
      before[t - first] = h;
      Decay<LOGITS> d;
      d.set(to_f32(decay[t * p.decay_stride]));
      const float value = to_f32(x[t * p.x_stride]);
      h = d.step(h, COMPLEMENT ? d.delta * value : value);
    }
    for (long long t = last - 1; t >= first; --t) {
      Decay<LOGITS> d;
      d.set(to_f32(decay[t * p.decay_stride]));
      const float grad = to_f32(dy[t * p.channels]) + carry;
      const float h0 = before[t - first];
      dx[t * p.channels] = from_f32<io_t>(COMPLEMENT ? d.delta * grad : grad);
      const float ddelta = grad * ((COMPLEMENT ? to_f32(x[t * p.x_stride]) : 0.f) - h0);
      dd[t * p.channels] = from_f32<io_t>(ddelta * d.slope);
      carry = d.step(grad, 0.f);
    }
  }
  if (g.dinitial != nullptr) g.dinitial[state] = carry;
}

template <typename io_t> void launch_forward(const GatedScanParams& p, int decay_mode, int input_mode, cudaStream_t s) {
  const dim3 grid((p.channels + kThreads - 1) / kThreads, p.n_seq);
  if (decay_mode == FRWKV_DECAY_LOGITS) {
    if (input_mode == FRWKV_INPUT_UNIT) gated_scan_forward_kernel<io_t, true, false><<<grid, kThreads, 0, s>>>(p);
    else gated_scan_forward_kernel<io_t, true, true><<<grid, kThreads, 0, s>>>(p);
  } else {
    if (input_mode == FRWKV_INPUT_UNIT) gated_scan_forward_kernel<io_t, false, false><<<grid, kThreads, 0, s>>>(p);
    else gated_scan_forward_kernel<io_t, false, true><<<grid, kThreads, 0, s>>>(p);
  }
}

template <typename io_t>
void launch_backward(const GatedScanParams& p, const GatedScanGrads& g, int decay_mode, int input_mode, cudaStream_t s) {
  const dim3 grid((p.channels + kThreads - 1) / kThreads, p.n_seq);
  if (decay_mode == FRWKV_DECAY_LOGITS) {
    if (input_mode == FRWKV_INPUT_UNIT) gated_scan_backward_kernel<io_t, true, false><<<grid, kThreads, 0, s>>>(p, g);
    else gated_scan_backward_kernel<io_t, true, true><<<grid, kThreads, 0, s>>>(p, g);
  } else {
    if (input_mode == FRWKV_INPUT_UNIT) gated_scan_backward_kernel<io_t, false, false><<<grid, kThreads, 0, s>>>(p, g);
    else gated_scan_backward_kernel<io_t, false, true><<<grid, kThreads, 0, s>>>(p, g);
  }
}

int check_sizes(const char* what, int n_seq, int total, int channels, int io_dtype, int decay_mode, int input_mode,
                const void* workspace, size_t workspace_bytes) {
  if (n_seq <= 0 || n_seq > 65535) return fail(FRWKV_ERR_ARGUMENT, "%s: sequence count must be in 1..65535, got %d", what, n_seq);
  if (total < n_seq || channels <= 0)
    return fail(FRWKV_ERR_ARGUMENT, "%s: every sequence needs a token and there must be a channel", what);
  if (io_dtype < FRWKV_IO_BF16 || io_dtype > FRWKV_IO_FP32) return fail(FRWKV_ERR_UNSUPPORTED, "%s: unknown token dtype", what);
  if ((decay_mode != FRWKV_DECAY_LOGITS && decay_mode != FRWKV_DECAY_RETENTION) ||
      (input_mode != FRWKV_INPUT_UNIT && input_mode != FRWKV_INPUT_COMPLEMENT))
    return fail(FRWKV_ERR_ARGUMENT, "%s: unknown decay or input mode", what);
  if (workspace_bytes < frwkv_sm100_gated_scan_workspace_bytes(total, channels) ||
      (workspace == nullptr && workspace_bytes > 0) || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0)
    return fail(FRWKV_ERR_WORKSPACE, "%s: the workspace must be 16-byte aligned and hold %zu bytes", what,
                frwkv_sm100_gated_scan_workspace_bytes(total, channels));
  return FRWKV_OK;
}

int run_forward(const GatedScanParams& p, int io_dtype, int decay_mode, int input_mode, void* stream) {
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (io_dtype == FRWKV_IO_BF16) launch_forward<__nv_bfloat16>(p, decay_mode, input_mode, s);
  else if (io_dtype == FRWKV_IO_FP16) launch_forward<__half>(p, decay_mode, input_mode, s);
  else launch_forward<float>(p, decay_mode, input_mode, s);
  return check_launch("gated_scan_forward_kernel");
}

}  // namespace
}  // namespace frwkv

extern "C" size_t frwkv_sm100_gated_scan_workspace_bytes(int total_tokens, int channels) {
  (void)total_tokens;
  (void)channels;
  return 0;
}

extern "C" int frwkv_sm100_gated_scan(
    const int32_t* cu_seqlens, const int32_t* slots, const int32_t* status, float* state_pool, const void* x,
    long long x_row_stride, const void* decay, long long decay_row_stride, const void* decay_bias, void* y, int n_seq,
    int total_tokens, int channels, int io_dtype, int decay_mode, int input_mode, int max_seqlen, void* workspace,
    size_t workspace_bytes, void* stream) {
  using namespace frwkv;
  (void)max_seqlen;
  if (!cu_seqlens || !slots || !state_pool || !x || !decay || !y)
    return fail(FRWKV_ERR_ARGUMENT, "gated_scan: cu_seqlens, slots, state_pool, x, decay and y must be non-null");
  if (decay_bias != nullptr && decay_mode != FRWKV_DECAY_LOGITS)
    return fail(FRWKV_ERR_ARGUMENT, "gated_scan: decay_bias only applies to decay logits");
  const int bad = check_sizes("gated_scan", n_seq, total_tokens, channels, io_dtype, decay_mode, input_mode, workspace,
                              workspace_bytes);
  if (bad != FRWKV_OK) return bad;
  const GatedScanParams p{cu_seqlens, slots, status, x, decay, decay_bias, x_row_stride, decay_row_stride, state_pool,
                          state_pool, nullptr, y, n_seq, total_tokens, channels, 0};
  return run_forward(p, io_dtype, decay_mode, input_mode, stream);
}

extern "C" int frwkv_sm100_gated_scan_train_forward(
    const int32_t* cu_seqlens, const int32_t* status, const void* x, long long x_row_stride, const void* decay,
    long long decay_row_stride, const float* initial, void* y, float* final_state, float* boundary, int n_seq,
    int total_tokens, int channels, int io_dtype, int decay_mode, int input_mode, void* workspace,
    size_t workspace_bytes, void* stream) {
  using namespace frwkv;
  if (!x || !decay || !y || !final_state || !boundary)
    return fail(FRWKV_ERR_ARGUMENT, "gated_scan training: x, decay, y, final_state and boundary must be non-null");
  const int bad = check_sizes("gated_scan training", n_seq, total_tokens, channels, io_dtype, decay_mode, input_mode,
                              workspace, workspace_bytes);
  if (bad != FRWKV_OK) return bad;
  if (cu_seqlens == nullptr && total_tokens % n_seq != 0)
    return fail(FRWKV_ERR_ARGUMENT, "gated_scan training: dense rows must be a multiple of the sequence count");
  const GatedScanParams p{cu_seqlens, nullptr, status, x, decay, nullptr, x_row_stride, decay_row_stride, initial,
                          final_state, boundary, y, n_seq, total_tokens, channels, total_tokens / n_seq};
  return run_forward(p, io_dtype, decay_mode, input_mode, stream);
}

extern "C" int frwkv_sm100_gated_scan_train_backward(
    const int32_t* cu_seqlens, const int32_t* status, const void* x, long long x_row_stride, const void* decay,
    long long decay_row_stride, const float* initial, const float* boundary, const void* dy, const float* dfinal,
    void* dx, void* ddecay, float* dinitial, int n_seq, int total_tokens, int channels, int io_dtype, int decay_mode,
    int input_mode, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace frwkv;
  if (!x || !decay || !boundary || !dy || !dx || !ddecay)
    return fail(FRWKV_ERR_ARGUMENT, "gated_scan backward: x, decay, boundary, dy, dx and ddecay must be non-null");
  const int bad = check_sizes("gated_scan backward", n_seq, total_tokens, channels, io_dtype, decay_mode, input_mode,
                              workspace, workspace_bytes);
  if (bad != FRWKV_OK) return bad;
  if (cu_seqlens == nullptr && total_tokens % n_seq != 0)
    return fail(FRWKV_ERR_ARGUMENT, "gated_scan backward: dense rows must be a multiple of the sequence count");
  const GatedScanParams p{cu_seqlens, nullptr, status, x, decay, nullptr, x_row_stride, decay_row_stride, initial,
                          nullptr, const_cast<float*>(boundary), nullptr, n_seq, total_tokens, channels,
                          total_tokens / n_seq};
  const GatedScanGrads g{dy, dfinal, dx, ddecay, dinitial};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (io_dtype == FRWKV_IO_BF16) launch_backward<__nv_bfloat16>(p, g, decay_mode, input_mode, s);
  else if (io_dtype == FRWKV_IO_FP16) launch_backward<__half>(p, g, decay_mode, input_mode, s);
  else launch_backward<float>(p, g, decay_mode, input_mode, s);
  return check_launch("gated_scan_backward_kernel");
}
