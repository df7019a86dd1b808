// Gated scan: in-place serving operator and training forward pass.
//
// Three elements of traffic a cell (x, decay, y), plus the state and, in training, a saved state every 16 rows: bound by HBM
// as long as the gates' instructions (about 21 for a logit, its sigmoid and exponential among them) are hidden.  Measured on
// bf16 logits: 64 x 2048 x 2560 335 us = 0.92 of the HBM copy rate (400 us when it runs for seconds and the power limit
// takes the clock down: then the instructions bound it; given retentions 324 and 357 us), 8 x 4096 x 2048 83 us = 0.74 (512 units
// of work on 148 SMs: some have four, some three), 1 x 65536 x 2048 206 us = 0.59 (clusters of eight: a step waits for the
// cluster's barrier).
#include "gated_scan_walk.cuh"

namespace frwkv {
namespace {

template <typename io_t, int ALIGN, bool LOGITS, bool COMPLEMENT, bool CLUSTER>
__global__ void __launch_bounds__(kThreads, forward_ctas(ALIGN, LOGITS, COMPLEMENT, sizeof(io_t))) gated_scan_forward_kernel(const GatedScanParams p, const Grid grid) {
  constexpr int V = 8 / sizeof(io_t);
  using L = Lanes<V>;
  using D = Decay<LOGITS, COMPLEMENT, V>;
  using R = Rows<io_t, ALIGN, S>;
  extern __shared__ uint2 staged[];  // x of two tiles, then the decays of one: [warp][R::kWords]
  __shared__ int lengths[kRanked];
  __shared__ Pieces<V, CLUSTER> pieces[2][kWarps];
  __shared__ Pieces<V, true> slots[2][CLUSTER ? kMaxCluster : 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (p.status != nullptr && p.status[0] != 0) {
    fill_rows_nan<io_t>(p, static_cast<io_t*>(p.y), nullptr, p.boundary != nullptr ? p.final_state : nullptr, p.n_seq);
    return;
  }
  if constexpr (CLUSTER) cg::this_cluster().sync();  // everyone's shared memory is there before it is written to
  const int n_seq = p.status != nullptr ? p.status[2] : p.n_seq;
  const int ranks = CLUSTER ? grid.cluster : 1, rank = CLUSTER ? static_cast<int>(blockIdx.x) % ranks : 0;
  Unit unit = unit_of<V>(p, grid, static_cast<int>(blockIdx.x) / ranks, n_seq, lengths);
  const int channel = unit.channel, count = min(V, p.channels - channel);
  const int block_channel = channel - lane % kLanes * V, block_count = min(kLanes * V, p.channels - block_channel);
  const long long least_stride = min(p.x_stride, p.decay_stride);
  const auto first_tile = [&](int seq) {
    if (seq < 0) return Tile{-1, 0, 0, 0};
    const int begin = row_begin(p, seq);
    return Tile{seq, begin, rank * kTile, row_begin(p, seq + 1) - begin};
  };
  const auto tile_after = [&](const Tile& t) {
    const int at = t.at + ranks * kTile;
    return at - rank * kTile < t.len ? Tile{t.seq, t.begin, at, t.len} : first_tile(unit.next());
  };
  const auto is_full = [&](const Tile& t) {
    return t.at + kTile <= t.len && block_count == kLanes * V && (ALIGN != 0 || (t.begin + t.at) * least_stride >= 16);
  };
  const int warp_row = warp * kGroups * S, own = warp_row + lane / kLanes * S;  // first rows in a tile
  uint2* const decays = staged + (2 * kWarps + warp) * R::kWords;
  const auto inputs = [&](int buffer) { return staged + (buffer * kWarps + warp) * R::kWords; };
  const auto fetch = [&](const Tile& t, int buffer) {
    if (t.seq < 0) return;
    const int row = t.begin + t.at + warp_row, left = t.len - t.at - warp_row;
    const io_t *x = static_cast<const io_t*>(p.x), *d = static_cast<const io_t*>(p.decay);
    const io_t *x_rows = x + row * p.x_stride + block_channel, *d_rows = d + row * p.decay_stride + block_channel;
    if (is_full(t)) {
      R::template fetch<true>(inputs(buffer), x_rows, p.x_stride, left, block_count, x);
      R::template fetch<true>(decays, d_rows, p.decay_stride, left, block_count, d);
    } else {
      R::template fetch<false>(inputs(buffer), x_rows, p.x_stride, left, block_count, x);
      R::template fetch<false>(decays, d_rows, p.decay_stride, left, block_count, d);
    }
    copies_begun();
  };
  const auto state_row = [&](int seq) {
    return static_cast<long long>(p.slots != nullptr ? p.slots[seq] : seq) * p.channels + channel;
  };
  const auto initial_state = [&](const Tile& t) {
    return t.seq >= 0 && p.initial != nullptr ? load_states<V>(p.initial + state_row(t.seq), count) : L::all(0.0f);
  };
  L bias = L::all(0.0f);
  if (LOGITS && p.bias != nullptr) {
    const io_t* from = static_cast<const io_t*>(p.bias) + channel;
    float b[V];
#pragma unroll
    for (int i = 0; i < V; ++i) b[i] = i < count ? to_f32(from[i]) * -kLog2e : 0.0f;
#pragma unroll
    for (int i = 0; i < V / 2; ++i) bias.v[i] = make_float2(b[2 * i], b[2 * i + 1]);
  }
  Tile tile = first_tile(unit.next());
  fetch(tile, 0);
  L carry = initial_state(tile);
  for (int round = 0; tile.seq >= 0; ++round) {
    const int buffer = round & 1;
    const Tile next = tile_after(tile);
    copies_done();
    __syncwarp();  // what the warp's other lanes copied

    // first sweep: the gates into registers, and the map of this lane's rows
    const long long own_row = tile.begin + tile.at + own;
    const typename R::Mine x = R::mine(inputs(buffer), lane / kLanes, static_cast<const io_t*>(p.x) + own_row * p.x_stride + block_channel, p.x_stride);
    const typename R::Mine d = R::mine(decays, lane / kLanes, static_cast<const io_t*>(p.decay) + own_row * p.decay_stride + block_channel, p.decay_stride);
    L kept[S];
    uint2 given[S];
    const auto keep = [&](int i) { return LOGITS ? kept[i] : unpack<io_t>(given[i]); };
    L behind = L::all(0.0f);
    Fade<LOGITS, V> fade = Fade<LOGITS, V>::none();
#pragma unroll
    for (int i = 0; i < S; ++i) {
      given[i] = d.words(i);
      L gate = unpack<io_t>(given[i]);
      if constexpr (LOGITS) gate = D::sigmoid(gate, bias);
      kept[i] = LOGITS ? D::keep_gate(gate) : gate;
      behind = D::step(kept[i], behind, x[i]);
      fade.take(gate, kept[i]);
    }
    if constexpr (!LOGITS) {
      // until the second sweep the decays stay as they came, which is half the registers for 16-bit tokens
#pragma unroll
      for (int i = 0; i < S; ++i) asm volatile("" : "+r"(given[i].x), "+r"(given[i].y));
    }
    __syncwarp();  // the decays have been read: their place is free
    fetch(next, buffer ^ 1);  // in flight while this tile is joined and written
    Map<V> map = Map<V>::of(fade, behind);
    join_groups(map);
    if (lane >= 32 - kLanes) pieces[buffer][warp].put(map);
    __syncthreads();

    // the state before this warp's rows, and behind the tile
    L h = carry;
    if constexpr (CLUSTER) {
      Map<V> cta = pieces[buffer][0].get();
#pragma unroll
      for (int w = 1; w < kWarps; ++w) cta.then(pieces[buffer][w].get());
      h = join_cluster(cta, slots[buffer], carry);
      for (int w = 0; w < warp; ++w) h = pieces[buffer][w].get().apply(h);
    } else {
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (w == warp) h = carry;
        carry = pieces[buffer][w].get().apply(carry);
      }
    }
    h = state_before_group(map, h);
    const int left = tile.len - tile.at - own;
    if (p.boundary != nullptr && left > 0) {
      float* to = p.boundary + saved_row(tile.seq, tile.begin, tile.at + own) * p.channels + channel;
      if (ALIGN == 16 && count == V) store_states_whole<V>(to, h);
      else store_states<V>(to, h, count);
    }
    if (next.seq != tile.seq) carry = initial_state(next);

    // second sweep
    io_t* y = static_cast<io_t*>(p.y) + own_row * p.channels + channel;
    if (is_full(tile)) {
#pragma unroll
      for (int i = 0; i < S; ++i) {
        h = D::step(keep(i), h, x[i]);
        R::template store<true>(y, h, count);
        y += p.channels;
      }
      if (left == S) store_states<V>(p.final_state + state_row(tile.seq), h, count);
    } else {
#pragma unroll
      for (int i = 0; i < S; ++i) {
        h = D::step(keep(i), h, x[i]);
        if (i < left) R::template store<false>(y, h, count);
        if (i + 1 == left) store_states<V>(p.final_state + state_row(tile.seq), h, count);
        y += p.channels;
      }
    }
    __syncwarp();  // the inputs have been read
    tile = next;
  }
}

// Decode steps and other short sequences: a thread walks V channels of one sequence, 16 bytes of a row.  The state pool is
// most of what a step reads and writes.  2048 x 4096 fp16: 18.1 us alone = 0.99 of the HBM copy rate, 20.1 us a step in a
// row of steps; 256 x 2048 bf16: 5.7 us, which is the host's time for a call.
template <typename io_t, int V, bool LOGITS, bool COMPLEMENT>
__global__ void __launch_bounds__(256) gated_scan_step_kernel(const GatedScanParams p) {
  // The next step's launch may begin while this one runs, and this one may have begun while the launch before it ran
  // (programmatic dependent launch); nothing is read before that one is done.
  asm volatile("griddepcontrol.launch_dependents;" : : : "memory");
  asm volatile("griddepcontrol.wait;" : : : "memory");
  if (p.status != nullptr && p.status[0] != 0) {
    fill_rows_nan<io_t>(p, static_cast<io_t*>(p.y), nullptr, nullptr, 0);
    return;
  }
  const int n_seq = p.status != nullptr ? p.status[2] : p.n_seq;
  const unsigned per_row = static_cast<unsigned>(p.channels / V), at = blockIdx.x * 256u + threadIdx.x;
  const int seq = static_cast<int>(at / per_row), channel = static_cast<int>(at % per_row) * V;
  if (seq >= n_seq) return;
  const int first = p.cu[seq], last = p.cu[seq + 1];
  if (last - first > p.longer_than) return;  // the other kernel's
  float* state = p.final_state + static_cast<long long>(p.slots[seq]) * p.channels + channel;
  constexpr int kPairs = (V + 1) / 2;  // V = 1 works on half a pair
  using D = Decay<LOGITS, COMPLEMENT, 2>;
  alignas(16) io_t x[V], d[V], b[V], y[V];
  alignas(16) float h[2 * kPairs];
  if constexpr (V == 1) {
    h[0] = *state;
    h[1] = 0.0f;
    if (p.bias != nullptr) b[0] = static_cast<const io_t*>(p.bias)[channel];
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 4) *reinterpret_cast<float4*>(h + i) = __ldcs(reinterpret_cast<const float4*>(state + i));
    if (p.bias != nullptr) *reinterpret_cast<uint4*>(b) = __ldg(reinterpret_cast<const uint4*>(static_cast<const io_t*>(p.bias) + channel));
  }
  for (long long row = first; row < last; ++row) {
    const io_t* xs = static_cast<const io_t*>(p.x) + row * p.x_stride + channel;
    const io_t* ds = static_cast<const io_t*>(p.decay) + row * p.decay_stride + channel;
    if constexpr (V == 1) {
      x[0] = *xs;
      d[0] = *ds;
    } else {
      *reinterpret_cast<uint4*>(x) = __ldcs(reinterpret_cast<const uint4*>(xs));
      *reinterpret_cast<uint4*>(d) = __ldcs(reinterpret_cast<const uint4*>(ds));
    }
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const auto pair = [&](const io_t* from) {
        Lanes<2> r;
        r.v[0] = make_float2(to_f32(from[2 * i]), V == 1 ? 0.0f : to_f32(from[V == 1 ? 0 : 2 * i + 1]));
        return r;
      };
      Lanes<2> bias = Lanes<2>::all(0.0f), state_pair;
      if (LOGITS && p.bias != nullptr) bias = mul(pair(b), Lanes<2>::all(-kLog2e));
      state_pair.v[0] = make_float2(h[2 * i], h[2 * i + 1]);
      state_pair = D::step(D::keep(pair(d), bias), state_pair, pair(x));
      h[2 * i] = state_pair.v[0].x;
      h[2 * i + 1] = state_pair.v[0].y;
      y[2 * i] = from_f32<io_t>(h[2 * i]);
      if constexpr (V > 1) y[2 * i + 1] = from_f32<io_t>(h[2 * i + 1]);
    }
    io_t* ys = static_cast<io_t*>(p.y) + row * p.channels + channel;
    if constexpr (V == 1) *ys = y[0];
    else __stcs(reinterpret_cast<uint4*>(ys), *reinterpret_cast<const uint4*>(y));
  }
  if constexpr (V == 1) {
    *state = h[0];
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 4) __stcs(reinterpret_cast<float4*>(state + i), *reinterpret_cast<const float4*>(h + i));
  }
}

int run_forward(const GatedScanParams& p, int io_dtype, int decay_mode, int input_mode, int max_seqlen, void* stream) {
  int rc = FRWKV_OK;
  with_type(io_dtype, alignment_of(p, io_dtype, {p.x, p.decay, p.y, p.boundary}), [&](auto io, auto align) {
    with_modes(decay_mode, input_mode, [&](auto logits, auto complement) {
      using io_t = decltype(io);
      const Grid g = cut(p, max_seqlen, kLanes * 8 / static_cast<int>(sizeof(io_t)), forward_ctas(align(), logits(), complement(), sizeof(io_t)) * sm_count());
      constexpr int kWords = 3 * Rows<io_t, align(), S>::kWords;
      constexpr const char* kName = "gated_scan_forward_kernel";
      rc = g.cluster > 1 ? launch(gated_scan_forward_kernel<io_t, align(), logits(), complement(), true>, g, p, kWords, stream, kName)
                         : launch(gated_scan_forward_kernel<io_t, align(), logits(), complement(), false>, g, p, kWords, stream, kName);
    });
  });
  return rc;
}

int run_steps(const GatedScanParams& p, int io_dtype, int decay_mode, int input_mode, void* stream) {
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int wide = io_dtype == FRWKV_IO_FP32 ? 4 : 8;
  const bool vectors = p.channels % wide == 0 && p.x_stride % wide == 0 && p.decay_stride % wide == 0 &&
                       multiple_of(16, {p.x, p.decay, p.bias, p.y, p.final_state});
  const unsigned grid = static_cast<unsigned>((static_cast<long long>(p.n_seq) * (p.channels / (vectors ? wide : 1)) + 255) / 256);
  with_modes(decay_mode, input_mode, [&](auto logits, auto complement) {
    const auto launch = [&](auto io, auto v) {
      cudaLaunchAttribute dependent;
      dependent.id = cudaLaunchAttributeProgrammaticStreamSerialization;
      dependent.val.programmaticStreamSerializationAllowed = 1;
      cudaLaunchConfig_t config = {};
      config.gridDim = dim3(grid);
      config.blockDim = dim3(256);
      config.stream = s;
      config.attrs = &dependent;
      config.numAttrs = 1;
      cudaLaunchKernelEx(&config, gated_scan_step_kernel<decltype(io), v(), logits(), complement()>, p);
    };
    using one = std::integral_constant<int, 1>;
    if (io_dtype == FRWKV_IO_FP32) vectors ? launch(float{}, std::integral_constant<int, 4>{}) : launch(float{}, one{});
    else if (io_dtype == FRWKV_IO_BF16) vectors ? launch(__nv_bfloat16{}, std::integral_constant<int, 8>{}) : launch(__nv_bfloat16{}, one{});
    else vectors ? launch(__half{}, std::integral_constant<int, 8>{}) : launch(__half{}, one{});
  });
  return check_launch("gated_scan_step_kernel");
}

}  // namespace
}  // namespace frwkv

extern "C" int frwkv_sm100_gated_scan(
    const int32_t* cu_seqlens, const int32_t* slots, const int32_t* status, float* state_pool, const void* x,
    long long x_row_stride, const void* decay, long long decay_row_stride, const void* decay_bias, void* y, int n_seq,
    int total_tokens, int channels, int io_dtype, int decay_mode, int input_mode, int max_seqlen, void* stream) {
  using namespace frwkv;
  if (!cu_seqlens || !slots || !state_pool || !x || !decay || !y)
    return fail(FRWKV_ERR_ARGUMENT, "gated_scan: cu_seqlens, slots, state_pool, x, decay and y must be non-null");
  if (decay_bias != nullptr && decay_mode != FRWKV_DECAY_LOGITS)
    return fail(FRWKV_ERR_ARGUMENT, "gated_scan: decay_bias only applies to decay logits");
  // where the status word has live counts n_seq is a capacity, which may exceed that of tokens
  const int bad = check_sizes("gated_scan", n_seq, total_tokens, status != nullptr ? 1 : n_seq, channels, io_dtype, decay_mode, input_mode);
  if (bad != FRWKV_OK) return bad;
  // short sequences go through the step kernel, the others through the tiled one; where it is known that there are none of
  // one kind, its kernel is not launched.  (The step kernel counts its threads in 32 bits.)
  const bool step_fits = static_cast<long long>(n_seq) * channels < 0x7fffffffll;
  const bool all_short = step_fits && max_seqlen > 0 && max_seqlen <= kShortRows;
  const bool none_short = !step_fits || n_seq == 1 || (max_seqlen > 0 && static_cast<long long>(max_seqlen) * n_seq == total_tokens);
  const GatedScanParams p{cu_seqlens, slots, status, x, decay, decay_bias, x_row_stride, decay_row_stride, state_pool,
                          state_pool, nullptr, y, n_seq, total_tokens, channels, 0,
                          all_short ? 0x7fffffff : none_short ? 0 : kShortRows};
  int rc = FRWKV_OK;
  if (all_short || !none_short) rc = run_steps(p, io_dtype, decay_mode, input_mode, stream);
  if (rc == FRWKV_OK && !all_short) rc = run_forward(p, io_dtype, decay_mode, input_mode, max_seqlen, stream);
  return rc;
}

extern "C" int frwkv_sm100_gated_scan_train_forward(
    const int32_t* cu_seqlens, const int32_t* status, const void* x, long long x_row_stride, const void* decay,
    long long decay_row_stride, const float* initial, void* y, float* final_state, float* boundary, int n_seq,
    int total_tokens, int channels, int io_dtype, int decay_mode, int input_mode, int max_seqlen, void* stream) {
  using namespace frwkv;
  if (!x || !decay || !y || !final_state || !boundary)
    return fail(FRWKV_ERR_ARGUMENT, "gated_scan training: x, decay, y, final_state and boundary must be non-null");
  const int bad = check_sizes("gated_scan training", n_seq, total_tokens, n_seq, channels, io_dtype, decay_mode, input_mode);
  if (bad != FRWKV_OK) return bad;
  if (cu_seqlens == nullptr && total_tokens % n_seq != 0)
    return fail(FRWKV_ERR_ARGUMENT, "gated_scan training: dense rows must be a multiple of the sequence count");
  const GatedScanParams p{cu_seqlens, nullptr, status, x, decay, nullptr, x_row_stride, decay_row_stride, initial,
                          final_state, boundary, y, n_seq, total_tokens, channels, total_tokens / n_seq, 0};
  return run_forward(p, io_dtype, decay_mode, input_mode, max_seqlen, stream);
}
