// Gated scan: training backward pass.
//
// Five elements of traffic a cell (x, decay, dy in, dx, ddecay out) and the saved states.  Gates, states and slopes are computed
// in one sweep with time, the gradient is carried against it; both stay in registers (250 of them, so eight warps an SM, whose
// sixteen independent rows a lane hide the latencies).  Measured on bf16 logits: 64 x 1024 x 2048 277 us = 0.74 of the HBM
// copy rate, 8 x 4096 x 2048 153 us = 0.67 (512 units of work on 296 places: two rounds for 1.7).
#include "gated_scan_walk.cuh"

namespace frwkv {
namespace {

// With c_t = rho_t g_t the same recurrence runs against time: g_t = dy_t + c_{t+1}, and c behind the last token is the final
// state's gradient.  Steps go from the end of a sequence to its start and rank 0 of a cluster takes the last of a step's
// tiles; inside a tile warps, lane groups and rows are counted from its end, so that all joins are those of the forward
// pass.  The states come from those that the forward pass saved before every lane's rows.

template <typename io_t, int ALIGN, bool LOGITS, bool COMPLEMENT, bool CLUSTER>
__global__ void __launch_bounds__(kThreads, kBackwardCtas)
gated_scan_backward_kernel(const GatedScanParams p, const GatedScanGrads g, const Grid grid) {
  constexpr int V = 8 / sizeof(io_t), kWarpRows = kGroups * S;
  using L = Lanes<V>;
  using D = Decay<LOGITS, COMPLEMENT, V>;
  using R = Rows<io_t, ALIGN, S>;
  extern __shared__ uint2 staged[];  // x and the decays of one tile, then dy of two: [warp][R::kWords]
  __shared__ int lengths[kRanked];
  __shared__ Pieces<V, CLUSTER> pieces[2][kWarps];
  __shared__ Pieces<V, true> slots[2][CLUSTER ? kMaxCluster : 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (p.status != nullptr && p.status[0] != 0) {
    fill_rows_nan<io_t>(p, static_cast<io_t*>(g.dx), static_cast<io_t*>(g.ddecay), g.dinitial, p.n_seq);
    return;
  }
  if constexpr (CLUSTER) cg::this_cluster().sync();
  const int ranks = CLUSTER ? grid.cluster : 1, rank = CLUSTER ? static_cast<int>(blockIdx.x) % ranks : 0;
  Unit unit = unit_of<V>(p, grid, static_cast<int>(blockIdx.x) / ranks, p.n_seq, lengths);
  const int channel = unit.channel, count = min(V, p.channels - channel);
  const int block_channel = channel - lane % kLanes * V, block_count = min(kLanes * V, p.channels - block_channel);
  const long long least_stride = min(p.x_stride, p.decay_stride);
  const int step_rows = ranks * kTile;
  const auto first_tile = [&](int seq) {
    if (seq < 0) return Tile{-1, 0, 0, 0};
    const int begin = row_begin(p, seq), len = row_begin(p, seq + 1) - begin;
    return Tile{seq, begin, (len - 1) / step_rows * step_rows + (ranks - 1 - rank) * kTile, len};
  };
  const auto tile_after = [&](const Tile& t) {
    return t.at >= step_rows ? Tile{t.seq, t.begin, t.at - step_rows, t.len} : first_tile(unit.next());
  };
  const auto is_full = [&](const Tile& t) {
    return t.at + kTile <= t.len && block_count == kLanes * V && (ALIGN != 0 || (t.begin + t.at) * least_stride >= 16);
  };
  // In memory the lane groups of a warp lie as in the forward pass, first in time first; along the chain a lane works on
  // group kGroups - 1 - lane / kLanes.
  const int warp_row = (kWarps - 1 - warp) * kWarpRows, group = kGroups - 1 - lane / kLanes, own = warp_row + group * S;
  const auto space = [&](int i) { return staged + (i * kWarps + warp) * R::kWords; };
  const auto fetch = [&](const Tile& t, int buffer) {
    if (t.seq < 0) return;
    const int row = t.begin + t.at + warp_row, left = t.len - t.at - warp_row;
    const io_t *x = static_cast<const io_t*>(p.x), *d = static_cast<const io_t*>(p.decay), *dy = static_cast<const io_t*>(g.dy);
    const io_t *x_rows = x + row * p.x_stride + block_channel, *d_rows = d + row * p.decay_stride + block_channel;
    const io_t* dy_rows = dy + static_cast<long long>(row) * p.channels + block_channel;
    if (is_full(t)) {
      R::template fetch<true>(space(0), x_rows, p.x_stride, left, block_count, x);
      R::template fetch<true>(space(1), d_rows, p.decay_stride, left, block_count, d);
      R::template fetch<true>(space(2 + buffer), dy_rows, p.channels, left, block_count, dy);
    } else {
      R::template fetch<false>(space(0), x_rows, p.x_stride, left, block_count, x);
      R::template fetch<false>(space(1), d_rows, p.decay_stride, left, block_count, d);
      R::template fetch<false>(space(2 + buffer), dy_rows, p.channels, left, block_count, dy);
    }
    copies_begun();
  };
  const auto final_grad = [&](const Tile& t) {
    return t.seq >= 0 && g.dfinal != nullptr ? load_states<V>(g.dfinal + static_cast<long long>(t.seq) * p.channels + channel, count)
                                             : L::all(0.0f);
  };
  Tile tile = first_tile(unit.next());
  fetch(tile, 0);
  L carry = final_grad(tile);
  for (int round = 0; tile.seq >= 0; ++round) {
    const int buffer = round & 1, left = tile.len - tile.at - own;
    const Tile next = tile_after(tile);
    // the state before this lane's rows, where it has any
    L h = L::all(0.0f);
    if (left > 0) {
      const float* from = p.boundary + saved_row(tile.seq, tile.begin, tile.at + own) * p.channels + channel;
      h = ALIGN == 16 && count == V ? load_states_whole<V>(from) : load_states<V>(from, count);
    }
    copies_done();
    __syncwarp();  // what the warp's other lanes copied
    const long long own_row = tile.begin + tile.at + own;
    const typename R::Mine x = R::mine(space(0), group, static_cast<const io_t*>(p.x) + own_row * p.x_stride + block_channel, p.x_stride);
    const typename R::Mine d = R::mine(space(1), group, static_cast<const io_t*>(p.decay) + own_row * p.decay_stride + block_channel, p.decay_stride);
    const typename R::Mine dy = R::mine(space(2 + buffer), group, static_cast<const io_t*>(g.dy) + own_row * p.channels + block_channel, p.channels);

    // with time: the gates, and what a row's gradient is multiplied by for ddecay: the state before it, less its input
    // (complement), by the gate's slope
    L kept[S], states[S];
    Fade<LOGITS, V> fade = Fade<LOGITS, V>::none();
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const L value = x[i];
      L sigmoid = d[i], e;
      if constexpr (LOGITS) {
        e = D::exponential(sigmoid, L::all(0.0f));
        sigmoid = D::sigmoid_of(e);
      }
      kept[i] = LOGITS ? D::keep_gate(sigmoid) : sigmoid;
      if (i < left) fade.take(sigmoid, kept[i]);
      states[i] = COMPLEMENT ? minus(h, value) : h;
      if constexpr (LOGITS) states[i] = mul(states[i], D::slope(e, sigmoid, kept[i]));
      h = D::step(kept[i], h, value);
    }
    // against it: the map of c.  Rows behind the sequence's end leave c as it is.
    L back_b = L::all(0.0f);
#pragma unroll
    for (int i = S - 1; i >= 0; --i) {
      if (i < left) back_b = D::fade(kept[i], add(dy[i], back_b));
    }
    Map<V> back = Map<V>::of(fade, back_b);
    join_groups(back);
    if (lane >= 32 - kLanes) pieces[buffer][warp].put(back);
    __syncwarp();  // the inputs and the decays have been read: their place is free
    fetch(next, buffer ^ 1);
    __syncthreads();

    L c = carry;
    if constexpr (CLUSTER) {
      Map<V> cta = pieces[buffer][0].get();
#pragma unroll
      for (int w = 1; w < kWarps; ++w) cta.then(pieces[buffer][w].get());
      c = join_cluster(cta, slots[buffer], carry);
      for (int w = 0; w < warp; ++w) c = pieces[buffer][w].get().apply(c);
    } else {
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (w == warp) c = carry;
        carry = pieces[buffer][w].get().apply(carry);
      }
    }
    c = state_before_group(back, c);
    if (next.seq != tile.seq) carry = final_grad(next);

    // second sweep
    io_t* dx = static_cast<io_t*>(g.dx) + (own_row + S - 1) * p.channels + channel;
    io_t* dd = static_cast<io_t*>(g.ddecay) + (own_row + S - 1) * p.channels + channel;
    const auto sweep = [&](auto full) {
#pragma unroll
      for (int i = S - 1; i >= 0; --i) {
        if (full() || i < left) {
          const L grad = add(dy[i], c);
          c = D::fade(kept[i], grad);
          R::template store<full()>(dx, D::input_grad(kept[i], grad), count);
          R::template store<full()>(dd, mul(grad, states[i]), count);
        }
        dx -= p.channels;
        dd -= p.channels;
      }
    };
    if (is_full(tile)) sweep(std::true_type{});
    else sweep(std::false_type{});
    __syncwarp();  // dy has been read
    if (tile.at + own == 0 && g.dinitial != nullptr)
      store_states<V>(g.dinitial + static_cast<long long>(tile.seq) * p.channels + channel, c, count);
    tile = next;
  }
}

}  // namespace
}  // namespace frwkv

extern "C" int frwkv_sm100_gated_scan_train_backward(
    const int32_t* cu_seqlens, const int32_t* status, const void* x, long long x_row_stride, const void* decay,
    long long decay_row_stride, const float* initial, const float* boundary, const void* dy, const float* dfinal,
    void* dx, void* ddecay, float* dinitial, int n_seq, int total_tokens, int channels, int io_dtype, int decay_mode,
    int input_mode, int max_seqlen, void* stream) {
  using namespace frwkv;
  if (!x || !decay || !boundary || !dy || !dx || !ddecay)
    return fail(FRWKV_ERR_ARGUMENT, "gated_scan backward: x, decay, boundary, dy, dx and ddecay must be non-null");
  const int bad = check_sizes("gated_scan backward", n_seq, total_tokens, n_seq, channels, io_dtype, decay_mode, input_mode);
  if (bad != FRWKV_OK) return bad;
  if (cu_seqlens == nullptr && total_tokens % n_seq != 0)
    return fail(FRWKV_ERR_ARGUMENT, "gated_scan backward: dense rows must be a multiple of the sequence count");
  const GatedScanParams p{cu_seqlens, nullptr, status, x, decay, nullptr, x_row_stride, decay_row_stride, initial,
                          nullptr, const_cast<float*>(boundary), nullptr, n_seq, total_tokens, channels,
                          total_tokens / n_seq, 0};
  const GatedScanGrads g{dy, dfinal, dx, ddecay, dinitial};
  int rc = FRWKV_OK;
  with_type(io_dtype, alignment_of(p, io_dtype, {x, decay, dy, dx, ddecay, boundary}) == 16 ? 16 : 0, [&](auto io, auto alignment) {
    with_modes(decay_mode, input_mode, [&](auto logits, auto complement) {
      using io_t = decltype(io);
      constexpr int kAlign = alignment() == 16 ? 16 : 0;  // by pieces rather than by 4 bytes
      const Grid grid = cut(p, max_seqlen, kLanes * 8 / static_cast<int>(sizeof(io_t)), kBackwardCtas * sm_count());
      constexpr int kWords = 4 * Rows<io_t, kAlign, S>::kWords;
      constexpr const char* kName = "gated_scan_backward_kernel";
      rc = grid.cluster > 1 ? launch(gated_scan_backward_kernel<io_t, kAlign, logits(), complement(), true>, grid, p, kWords, stream, kName, g)
                            : launch(gated_scan_backward_kernel<io_t, kAlign, logits(), complement(), false>, grid, p, kWords, stream, kName, g);
    });
  });
  return rc;
}
