// Log probabilities of given tokens, entropy and top alternatives of rows of vocabulary logits; gradient.
//
// With m the largest logit of a row and e_j = exp((x_j - m) / T):  S = sum e_j,  W = sum e_j (x_j - m) / T,
//   logprob = (x_id - m) / T - log S,   entropy = log S - W / S.
// Differences to m are formed before anything is scaled, so a common offset of a row costs no precision.
// One CTA per row.
#include "../common.cuh"

namespace frwkv {
namespace {

constexpr int kThreads = 256;

struct Rows {
  const void* logits;
  long long rows, inner, stride_outer, stride_inner;
  const void* ids;
  int ids_are_int64;
  long long ignore_index;
  int vocab;
  float inv_temperature;
};

template <typename io_t> __device__ __forceinline__ const io_t* row_start(const Rows& p, long long row) {
  return static_cast<const io_t*>(p.logits) + row / p.inner * p.stride_outer + row % p.inner * p.stride_inner;
}

__device__ __forceinline__ long long row_id(const Rows& p, long long row) {
  return p.ids_are_int64 ? static_cast<const long long*>(p.ids)[row] : static_cast<const int*>(p.ids)[row];
}

// exp((x - m) / T); rows of -inf alone have m = -inf and are dealt with by the callers
__device__ __forceinline__ float scaled(float x, float m, float inv_temperature) { return (x - m) * inv_temperature; }

// Total order of logits, larger first: monotone in the value, -0 equal to +0, NaN above everything.
__device__ __forceinline__ unsigned order_of(float x) {
  if (x != x) return 0xfffffffeu;  // not the largest number: that one means "no bound yet"
  const unsigned bits = __float_as_uint(x + 0.0f);
  return (bits & 0x80000000u) ? ~bits : bits | 0x80000000u;
}

template <typename T, typename F> __device__ T block_reduce(T value, F join, T* scratch) {
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) value = join(value, __shfl_xor_sync(0xffffffffu, value, m));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = value;
  __syncthreads();
  value = scratch[0];
  for (int w = 1; w < kThreads / 32; ++w) value = join(value, scratch[w]);
  return value;
}

template <typename io_t>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(const Rows p, int top_k, float* logprobs, float* entropy,
                                                                  float* stats, int64_t* top_ids, float* top_logprobs) {
  __shared__ float scratch[kThreads / 32];
  __shared__ unsigned long long key_scratch[kThreads / 32];
  const long long row = blockIdx.x;
  const long long id = row_id(p, row);
  if (id == p.ignore_index) {
    if (threadIdx.x == 0) {
      logprobs[row] = entropy[row] = 0.f;
      stats[2 * row] = stats[2 * row + 1] = 0.f;
    }
    for (int k = threadIdx.x; k < top_k; k += kThreads) {
      top_ids[row * top_k + k] = -1;
      top_logprobs[row * top_k + k] = -INFINITY;
    }
    return;
  }
  const io_t* x = row_start<io_t>(p, row);
  float m = -INFINITY;
  for (int j = threadIdx.x; j < p.vocab; j += kThreads) m = fmaxf(m, to_f32(x[j]));
  m = block_reduce(m, [](float a, float b) { return fmaxf(a, b); }, scratch);
  float s = 0.f, w = 0.f;
  if (m != -INFINITY) {
    for (int j = threadIdx.x; j < p.vocab; j += kThreads) {
      const float z = scaled(to_f32(x[j]), m, p.inv_temperature);
      const float e = exp2f(z * kLog2e);
      s += e;
      if (e != 0.f) w = fmaf(e, z, w);
    }
  }
  const auto add = [](float a, float b) { return a + b; };
  s = block_reduce(s, add, scratch);
  w = block_reduce(w, add, scratch);
  // a row of NaN alone leaves m at -inf as well
  float any = 0.f;
  if (m == -INFINITY) {
    for (int j = threadIdx.x; j < p.vocab; j += kThreads) any += to_f32(x[j]) != to_f32(x[j]) ? 1.f : 0.f;
    any = block_reduce(any, add, scratch);
    if (any > 0.f) m = __int_as_float(0x7fffffff);
  }
  const bool empty = m == -INFINITY;
  const float log_s = empty ? 0.f : m != m ? m : logf(s);
  if (threadIdx.x == 0) {
    const bool known = id >= 0 && id < p.vocab;
    logprobs[row] = !known ? __int_as_float(0x7fffffff) : empty ? -INFINITY : scaled(to_f32(x[id]), m, p.inv_temperature) - log_s;
    entropy[row] = empty ? 0.f : log_s - w / s;
    stats[2 * row] = m;
    stats[2 * row + 1] = log_s;
  }
  unsigned long long below = ~0ull;
  for (int k = 0; k < top_k; ++k) {
    unsigned long long best = 0;
    for (int j = threadIdx.x; j < p.vocab; j += kThreads) {
      const unsigned long long key = static_cast<unsigned long long>(order_of(to_f32(x[j]))) << 32 | (0xffffffffu - j);
      if (key < below && key > best) best = key;
    }
    best = block_reduce(best, [](unsigned long long a, unsigned long long b) { return a > b ? a : b; }, key_scratch);
    below = best;
    if (threadIdx.x == 0) {
      const unsigned j = 0xffffffffu - static_cast<unsigned>(best);
      top_ids[row * top_k + k] = j;
      top_logprobs[row * top_k + k] = empty ? -INFINITY : scaled(to_f32(x[j]), m, p.inv_temperature) - log_s;
    }
  }
}

template <typename io_t>
__global__ void __launch_bounds__(kThreads) token_logprobs_backward_kernel(const Rows p, const float* stats,
                                                                           const float* entropy, const float* dlogprobs,
                                                                           const float* dentropy, io_t* dlogits) {
  const long long row = blockIdx.x;
  const long long id = row_id(p, row);
  io_t* out = dlogits + row * p.vocab;
  const float m = stats[2 * row], log_s = stats[2 * row + 1];
  if (id == p.ignore_index || m == -INFINITY) {
    for (int j = threadIdx.x; j < p.vocab; j += kThreads) out[j] = from_f32<io_t>(0.f);
    return;
  }
  const io_t* x = row_start<io_t>(p, row);
  const float a = id < 0 || id >= p.vocab ? __int_as_float(0x7fffffff) : dlogprobs != nullptr ? dlogprobs[row] : 0.f;
  const float b = dentropy != nullptr ? dentropy[row] : 0.f;
  const float h = entropy[row];
  for (int j = threadIdx.x; j < p.vocab; j += kThreads) {
    const float logp = scaled(to_f32(x[j]), m, p.inv_temperature) - log_s;
    const float prob = exp2f(logp * kLog2e);
    float grad = prob != 0.f ? -prob * fmaf(b, logp + h, a) : -0.f * a;
    if (j == id) grad += a;
    out[j] = from_f32<io_t>(grad * p.inv_temperature);
  }
}

int check_rows(const char* what, const void* logits, long long outer, long long inner, const void* ids, int vocab,
               int io_dtype, float temperature) {
  if (!logits || !ids) return fail(FRWKV_ERR_ARGUMENT, "%s: logits and ids must be non-null", what);
  if (outer <= 0 || inner <= 0 || outer > 0x7fffffffLL / inner)
    return fail(FRWKV_ERR_ARGUMENT, "%s: the row count must be positive and fit in int32", what);
  if (vocab <= 0) return fail(FRWKV_ERR_ARGUMENT, "%s: vocab must be positive", what);
  if (io_dtype < FRWKV_IO_BF16 || io_dtype > FRWKV_IO_FP32) return fail(FRWKV_ERR_UNSUPPORTED, "%s: unknown dtype", what);
  if (!(temperature > 0.f) || !(1.0f / temperature > 0.f) || !(1.0f / temperature < INFINITY))
    return fail(FRWKV_ERR_ARGUMENT, "%s: temperature and its reciprocal must be positive and finite", what);
  return FRWKV_OK;
}

}  // namespace
}  // namespace frwkv

extern "C" int frwkv_sm100_token_logprobs(
    const void* logits, long long outer, long long inner, long long stride_outer, long long stride_inner,
    const void* ids, int ids_are_int64, long long ignore_index, int vocab, int io_dtype, float temperature, int top_k, float* logprobs, float* entropy, float* stats,
    int64_t* top_ids, float* top_logprobs, void* stream) {
  using namespace frwkv;
  const int bad = check_rows("token_logprobs", logits, outer, inner, ids, vocab, io_dtype, temperature);
  if (bad != FRWKV_OK) return bad;
  if (!logprobs || !entropy || !stats)
    return fail(FRWKV_ERR_ARGUMENT, "token_logprobs: logprobs, entropy and stats must be non-null");
  if (top_k < 0 || top_k > FRWKV_TOP_K_MAX || top_k > vocab || (top_k > 0 && (!top_ids || !top_logprobs)))
    return fail(FRWKV_ERR_ARGUMENT, "token_logprobs: top_k must be in 0..%d, at most vocab, with arrays to write to",
                FRWKV_TOP_K_MAX);
  const Rows p{logits, outer * inner, inner, stride_outer, stride_inner, ids, ids_are_int64, ignore_index, vocab,
               1.0f / temperature};
  const unsigned grid = static_cast<unsigned>(p.rows);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (io_dtype == FRWKV_IO_BF16)
    token_logprobs_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(p, top_k, logprobs, entropy, stats, top_ids, top_logprobs);
  else if (io_dtype == FRWKV_IO_FP16)
    token_logprobs_kernel<__half><<<grid, kThreads, 0, s>>>(p, top_k, logprobs, entropy, stats, top_ids, top_logprobs);
  else
    token_logprobs_kernel<float><<<grid, kThreads, 0, s>>>(p, top_k, logprobs, entropy, stats, top_ids, top_logprobs);
  return check_launch("token_logprobs_kernel");
}

extern "C" int frwkv_sm100_token_logprobs_backward(
    const void* logits, long long outer, long long inner, long long stride_outer, long long stride_inner,
    const void* ids, int ids_are_int64, long long ignore_index, int vocab, int io_dtype, float temperature, const float* stats, const float* entropy, const float* dlogprobs,
    const float* dentropy, void* dlogits, void* stream) {
  using namespace frwkv;
  const int bad = check_rows("token_logprobs backward", logits, outer, inner, ids, vocab, io_dtype, temperature);
  if (bad != FRWKV_OK) return bad;
  if (!stats || !entropy || !dlogits)
    return fail(FRWKV_ERR_ARGUMENT, "token_logprobs backward: stats, entropy and dlogits must be non-null");
  const Rows p{logits, outer * inner, inner, stride_outer, stride_inner, ids, ids_are_int64, ignore_index, vocab,
               1.0f / temperature};
  const unsigned grid = static_cast<unsigned>(p.rows);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (io_dtype == FRWKV_IO_BF16)
    token_logprobs_backward_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(p, stats, entropy, dlogprobs, dentropy,
                                                                            static_cast<__nv_bfloat16*>(dlogits));
  else if (io_dtype == FRWKV_IO_FP16)
    token_logprobs_backward_kernel<__half><<<grid, kThreads, 0, s>>>(p, stats, entropy, dlogprobs, dentropy,
                                                                     static_cast<__half*>(dlogits));
  else
    token_logprobs_backward_kernel<float><<<grid, kThreads, 0, s>>>(p, stats, entropy, dlogprobs, dentropy,
                                                                    static_cast<float*>(dlogits));
  return check_launch("token_logprobs_backward_kernel");
}
