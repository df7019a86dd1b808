// Gated scan: in-place serving operator and training forward / backward (see gated_scan.cuh for the arithmetic).
//
// A cluster of CTAs (one, where there is enough to do) walks one sequence over 64 bytes of channels, the state carried from
// step to step.  In a step each CTA takes a tile of 256 tokens: a warp 32 of them, a lane 8 tokens of 8 bytes of channels.
// The tokens come through shared memory (cp.async, the next tile's while this one is worked on).  A first sweep computes the
// gates into registers and gives each lane an affine map of the state, h -> a h + b, over its 8 tokens; the maps are joined
// over the warp's four lane groups (shuffles), its warps (shared memory) and the cluster's CTAs (distributed shared
// memory), always in the same order; a second sweep over the registers writes the rows.  So the tokens are read once and
// the outputs written once, and nothing waits for anything outside its cluster.
#include "gated_scan.cuh"

#include <cooperative_groups.h>

#include <algorithm>

namespace frwkv {
namespace {

namespace cg = cooperative_groups;

constexpr int kTile = 256;           // tokens of a CTA's tile
constexpr int S = 16;                // tokens of a lane in a tile
constexpr int kWarps = kTile / (kGroups * S), kThreads = kWarps * 32;
// CTAs per SM, by registers and by the staging of their rows.  Copies of 4 bytes go through L1, which the staging of a fourth
// CTA would leave too small (16 x 1024 rows of 1003 fp32 channels: 86 us with four, 56 us with three).
constexpr int forward_ctas(int align) { return align == 16 ? 4 : 3; }
constexpr int kBackwardCtas = 2;
constexpr int kMaxCluster = 8;
constexpr int kShortRows = 16;       // sequences of at most this many tokens are served by the step kernel
constexpr int kRanked = 128;         // up to this many sequences are taken longest first
static_assert(S == kSavedRows, "the backward pass loads a state for every lane's rows");

// NaN in every row that the call would write (fail-closed), by the whole grid.
template <typename io_t>
__device__ void fill_rows_nan(const GatedScanParams& p, io_t* rows, io_t* more_rows, float* states, int n_states) {
  const long long self = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  const long long threads = static_cast<long long>(gridDim.x) * blockDim.x;
  fill_output_nan(rows, nullptr, static_cast<long long>(p.total) * p.channels, self, threads);
  if (more_rows != nullptr) fill_output_nan(more_rows, nullptr, static_cast<long long>(p.total) * p.channels, self, threads);
  if (states != nullptr)
    fill_output_nan<float>(states, nullptr, static_cast<long long>(n_states) * p.channels, self, threads);
}

__device__ __forceinline__ void copies_begun() { asm volatile("cp.async.commit_group;" : : : "memory"); }
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_group 0;" : : : "memory"); }

// The work of a cluster: a block of channels of up to 32 consecutive sequences, one after the other.
struct Unit {
  unsigned left;   // bit i: sequence first_seq + i is still to do
  int first_seq;
  int channel;     // of this lane

  // Next sequence, or -1.
  __device__ __forceinline__ int next() {
    if (left == 0) return -1;
    const int i = __ffs(left) - 1;
    left &= left - 1;
    return first_seq + i;
  }
};

struct Grid {
  int blocks;    // channel blocks
  int per_unit;  // sequences of a unit
  int cluster;   // CTAs of a cluster
};

__device__ __forceinline__ int row_begin(const GatedScanParams& p, int seq) { return p.cu != nullptr ? p.cu[seq] : seq * p.seq_len; }

// By all threads of the CTA.  Long sequences that start last would leave the GPU to a few CTAs, so a batch of a few
// sequences of different lengths is taken longest first.  Each warp ranks them for itself and takes its answer from a vote:
// the compiler then knows that the warp agrees, and what follows from it costs one lane, not 32 (64 x 2048 rows of 2560
// channels: 317 us; with the answer read from shared memory 370).
template <int V> __device__ __forceinline__ Unit unit_of(const GatedScanParams& p, const Grid& g, int unit, int n_seq, int* lengths) {
  const int lane = threadIdx.x & 31, chunk = unit / g.blocks;
  Unit u;
  u.first_seq = chunk * g.per_unit;
  u.channel = ((unit - chunk * g.blocks) * kLanes + lane % kLanes) * V;
  if (p.cu != nullptr && g.per_unit == 1 && n_seq > 1 && n_seq <= kRanked) {
    int longest = 0, shortest = 0x7fffffff;
    for (int at = lane; at < n_seq; at += 32) {
      const int len = p.cu[at + 1] - p.cu[at];
      lengths[at] = len;  // every warp writes the same
      longest = max(longest, len);
      shortest = min(shortest, len);
    }
    if (__reduce_max_sync(0xffffffffu, longest) != __reduce_min_sync(0xffffffffu, shortest)) {
      __syncwarp();
      u.first_seq = n_seq;
      for (int base = 0; base < n_seq; base += 32) {
        const int at = base + lane, len = at < n_seq ? lengths[at] : -1;
        int rank = 0;
        for (int i = 0; i < n_seq; ++i) rank += lengths[i] > len || (lengths[i] == len && i < at);
        const unsigned hit = __ballot_sync(0xffffffffu, at < n_seq && rank == chunk);
        if (hit != 0) u.first_seq = base + __ffs(hit) - 1;
      }
    }
  }
  const int seq = u.first_seq + lane;
  const bool mine = lane < g.per_unit && seq < n_seq && row_begin(p, seq + 1) - row_begin(p, seq) > p.longer_than;
  u.left = __ballot_sync(0xffffffffu, mine);
  return u;
}

// A CTA's tile: rows [at, at + kTile) of a sequence, as far as it goes.
struct Tile {
  int seq;    // < 0: there is none
  int begin;  // first row of the sequence
  int at;     // of the tile, in the sequence
  int len;    // of the sequence
};

template <int V> struct Scan {
  using L = Lanes<V>;

  // Inclusive join of the maps of a warp's lane groups, in their order; returns the map before this lane's rows.
  static __device__ __forceinline__ Map<V> join_groups(Map<V>& m) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int d = kLanes; d < 32; d *= 2) {
      Map<V> before{shuffle_up(m.a, d), shuffle_up(m.b, d)};
      if (lane >= d) {
        before.then(m);
        m = before;
      }
    }
    Map<V> before{shuffle_up(m.a, kLanes), shuffle_up(m.b, kLanes)};
    return lane >= kLanes ? before : Map<V>::identity();
  }
};

// The maps of one warp's or CTA's rows in shared memory, by lane along the channels.
template <int V> struct Pieces {
  Lanes<V> a[kLanes], b[kLanes];

  __device__ __forceinline__ void put(const Map<V>& m) {
    a[threadIdx.x % kLanes] = m.a;
    b[threadIdx.x % kLanes] = m.b;
  }
  __device__ __forceinline__ Map<V> get() const { return Map<V>{a[threadIdx.x % kLanes], b[threadIdx.x % kLanes]}; }
};

// Joins the CTAs of a cluster: each writes its map into everyone's shared memory (slots[rank]), a cluster barrier, and each
// applies the maps of the ranks before it.  Returns the state before this CTA's tile and moves `carry` behind the cluster's.
template <int V>
__device__ __forceinline__ Lanes<V> join_cluster(const Map<V>& cta, Pieces<V>* slots, Lanes<V>& carry) {
  const cg::cluster_group cluster = cg::this_cluster();
  const int ranks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int r = warp; r < ranks; r += static_cast<int>(blockDim.x) / 32)
    if (lane < kLanes) cluster.map_shared_rank(&slots[rank], r)->put(cta);
  cluster.sync();
  Lanes<V> mine = carry;
  for (int r = 0; r < ranks; ++r) {
    if (r == rank) mine = carry;
    carry = slots[r].get().apply(carry);
  }
  return mine;
}

// ---- forward

template <typename io_t, int ALIGN, bool LOGITS, bool COMPLEMENT, bool CLUSTER>
__global__ void __launch_bounds__(kThreads, forward_ctas(ALIGN)) gated_scan_forward_kernel(const GatedScanParams p, const Grid grid) {
  constexpr int V = 8 / sizeof(io_t);
  using L = Lanes<V>;
  using D = Decay<LOGITS, COMPLEMENT, V>;
  using R = Rows<io_t, ALIGN, S>;
  extern __shared__ uint2 staged[];  // x of two tiles, then the decays of one: [warp][R::kWords]
  __shared__ int lengths[kRanked];
  __shared__ Pieces<V> pieces[2][kWarps], slots[2][CLUSTER ? kMaxCluster : 1];
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
    Map<V> map = Map<V>::identity();
#pragma unroll
    for (int i = 0; i < S; ++i) {
      kept[i] = D::keep(d[i], bias);
      map.b = D::step(kept[i], map.b, x[i]);
      map.a = D::fade(kept[i], map.a);
    }
    __syncwarp();  // the decays have been read: their place is free
    fetch(next, buffer ^ 1);  // in flight while this tile is joined and written
    const Map<V> before = Scan<V>::join_groups(map);
    if (lane >= 32 - kLanes) pieces[buffer][warp].put(map);
    __syncthreads();

    // the state before this warp's rows, and behind the tile
    L h = carry;
    if constexpr (CLUSTER) {
      Map<V> cta = pieces[buffer][0].get();
#pragma unroll
      for (int w = 1; w < kWarps; ++w) cta.then(pieces[buffer][w].get());
      h = join_cluster<V>(cta, slots[buffer], carry);
      for (int w = 0; w < warp; ++w) h = pieces[buffer][w].get().apply(h);
    } else {
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (w == warp) h = carry;
        carry = pieces[buffer][w].get().apply(carry);
      }
    }
    h = before.apply(h);
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
        h = D::step(kept[i], h, x[i]);
        R::template store<true>(y, h, count);
        y += p.channels;
      }
      if (left == S) store_states<V>(p.final_state + state_row(tile.seq), h, count);
    } else {
#pragma unroll
      for (int i = 0; i < S; ++i) {
        h = D::step(kept[i], h, x[i]);
        if (i < left) R::template store<false>(y, h, count);
        if (i + 1 == left) store_states<V>(p.final_state + state_row(tile.seq), h, count);
        y += p.channels;
      }
    }
    __syncwarp();  // the inputs have been read
    tile = next;
  }
}

// Decode steps (and rows of a few tokens): a thread walks V channels of one sequence, 16 bytes of a row; no chain.  The
// state pool is most of what a step reads and writes.
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

// ---- backward
//
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
  __shared__ Pieces<V> pieces[2][kWarps], slots[2][CLUSTER ? kMaxCluster : 1];
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
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const L value = x[i];
      L sigmoid;
      if constexpr (LOGITS) {
        sigmoid = D::sigmoid(d[i], L::all(0.0f));
        kept[i] = D::keep_gate(sigmoid);
      } else {
        kept[i] = d[i];
      }
      states[i] = COMPLEMENT ? minus(h, value) : h;
      if constexpr (LOGITS) states[i] = mul(states[i], D::slope(sigmoid, kept[i]));
      h = D::step(kept[i], h, value);
    }
    // against it: the map of c.  Rows behind the sequence's end leave c as it is.
    Map<V> back = Map<V>::identity();
#pragma unroll
    for (int i = S - 1; i >= 0; --i) {
      if (i < left) {
        back.b = D::fade(kept[i], add(dy[i], back.b));
        back.a = D::fade(kept[i], back.a);
      }
    }
    const Map<V> behind = Scan<V>::join_groups(back);
    if (lane >= 32 - kLanes) pieces[buffer][warp].put(back);
    __syncwarp();  // the inputs and the decays have been read: their place is free
    fetch(next, buffer ^ 1);
    __syncthreads();

    L c = carry;
    if constexpr (CLUSTER) {
      Map<V> cta = pieces[buffer][0].get();
#pragma unroll
      for (int w = 1; w < kWarps; ++w) cta.then(pieces[buffer][w].get());
      c = join_cluster<V>(cta, slots[buffer], carry);
      for (int w = 0; w < warp; ++w) c = pieces[buffer][w].get().apply(c);
    } else {
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (w == warp) c = carry;
        carry = pieces[buffer][w].get().apply(carry);
      }
    }
    c = behind.apply(c);
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

// ---- launches

int sm_count() {
  static const int count = [] {
    int device = 0, n = 0;
    if (cudaGetDevice(&device) != cudaSuccess ||
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || n <= 0)
      n = 148;
    return n;
  }();
  return count;
}

bool multiple_of(int bytes, std::initializer_list<const void*> pointers) {
  for (const void* p : pointers)
    if ((reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0) return false;
  return true;
}

int check_sizes(const char* what, int n_seq, int total, int channels, int io_dtype, int decay_mode, int input_mode) {
  if (n_seq <= 0 || n_seq > 65535) return fail(FRWKV_ERR_ARGUMENT, "%s: sequence count must be in 1..65535, got %d", what, n_seq);
  if (total < n_seq || channels <= 0)
    return fail(FRWKV_ERR_ARGUMENT, "%s: every sequence needs a token and there must be a channel", what);
  if (channels > 0x7fffff00 || total > 0x7ffff000)
    return fail(FRWKV_ERR_UNSUPPORTED, "%s: token and channel counts must leave room for a tile below 2^31", what);
  if (io_dtype < FRWKV_IO_BF16 || io_dtype > FRWKV_IO_FP32) return fail(FRWKV_ERR_UNSUPPORTED, "%s: unknown token dtype", what);
  if ((decay_mode != FRWKV_DECAY_LOGITS && decay_mode != FRWKV_DECAY_RETENTION) ||
      (input_mode != FRWKV_INPUT_UNIT && input_mode != FRWKV_INPUT_COMPLEMENT))
    return fail(FRWKV_ERR_ARGUMENT, "%s: unknown decay or input mode", what);
  return FRWKV_OK;
}

// Calls f with the modes as compile-time constants.
template <typename F> void with_modes(int decay_mode, int input_mode, F f) {
  using yes = std::true_type;
  using no = std::false_type;
  if (decay_mode == FRWKV_DECAY_LOGITS) {
    if (input_mode == FRWKV_INPUT_UNIT) f(yes{}, no{});
    else f(yes{}, yes{});
  } else {
    if (input_mode == FRWKV_INPUT_UNIT) f(no{}, no{});
    else f(no{}, yes{});
  }
}

// Calls f with the token type and the rows' alignment as compile-time constants.
template <typename F> void with_type(int io_dtype, int align, F f) {
  using none = std::integral_constant<int, 0>;
  using four = std::integral_constant<int, 4>;
  using all = std::integral_constant<int, 16>;
  const auto with_align = [&](auto io) {
    if (align == 16) f(io, all{});
    else if (align == 4) f(io, four{});
    else f(io, none{});
  };
  if (io_dtype == FRWKV_IO_FP32) with_align(float{});
  else if (io_dtype == FRWKV_IO_BF16) with_align(__nv_bfloat16{});
  else with_align(__half{});
}

// 16 or 4 where the channels, the strides and all starts are multiples of that many bytes, else 0.
int alignment_of(const GatedScanParams& p, int io_dtype, std::initializer_list<const void*> rows) {
  for (int align : {16, 4}) {
    const int n = align / (io_dtype == FRWKV_IO_FP32 ? 4 : 2);
    if (p.channels % n == 0 && p.x_stride % n == 0 && p.decay_stride % n == 0 && multiple_of(align, rows)) return align;
  }
  return 0;
}

// How the work is cut.  Few sequences with few channels leave the GPU empty, so a cluster shares a sequence: the size that
// needs the least time in rounds of CTAs (`slots` are resident at once) times steps, a cluster's step counting half as much
// again.  (65536 rows of 2048 channels: 462 us for single CTAs, 259 for four, 207 for eight; 8 x 4096 rows, where 512 single
// CTAs fill the GPU: 80 us, and 92, 100, 116 us for clusters of 2, 4, 8.)  Very many sequences are taken several to a
// unit, so that the CTAs outlive their start.
Grid cut(const GatedScanParams& p, int max_seqlen, int lanes, int slots) {
  Grid g{(p.channels + lanes - 1) / lanes, 1, 1};
  const long long items = static_cast<long long>(p.n_seq) * g.blocks;
  g.per_unit = static_cast<int>(std::min<long long>(32, std::max<long long>(1, items / 16384)));
  const long long units = static_cast<long long>((p.n_seq + g.per_unit - 1) / g.per_unit) * g.blocks;
  const int longest = max_seqlen > 0 ? max_seqlen : (p.total + p.n_seq - 1) / p.n_seq;
  const int tiles = (longest + kTile - 1) / kTile;
  double best = 0.0;
  for (int size = 1; size <= kMaxCluster && size <= tiles; ++size) {
    const double time = static_cast<double>((units * size + slots - 1) / slots) * ((tiles + size - 1) / size) * (size > 1 ? 1.5 : 1.0);
    if (size == 1 || time < 0.95 * best) {
      best = time;
      g.cluster = size;
    }
  }
  return g;
}

template <typename K, typename... Args>
int launch(K kernel, const Grid& g, const GatedScanParams& p, int words, void* stream, const char* what, Args... args) {
  const long long units = static_cast<long long>((p.n_seq + g.per_unit - 1) / g.per_unit) * g.blocks;
  if (units * g.cluster > 0x7fffffffll) return fail(FRWKV_ERR_UNSUPPORTED, "%s: too many sequences by channels", what);
  const int shared = kWarps * words * 8;
  const cudaError_t error = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, shared);
  if (error != cudaSuccess) return fail(FRWKV_ERR_CUDA, "%s: preparing the launch: %s", what, cudaGetErrorString(error));
  cudaLaunchAttribute cluster;
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = static_cast<unsigned>(g.cluster);
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(units * g.cluster));
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = static_cast<size_t>(shared);
  config.stream = static_cast<cudaStream_t>(stream);
  config.attrs = &cluster;
  config.numAttrs = g.cluster > 1 ? 1 : 0;
  cudaLaunchKernelEx(&config, kernel, p, args..., g);
  return check_launch(what);
}

int run_forward(const GatedScanParams& p, int io_dtype, int decay_mode, int input_mode, int max_seqlen, void* stream) {
  int rc = FRWKV_OK;
  with_type(io_dtype, alignment_of(p, io_dtype, {p.x, p.decay, p.y, p.boundary}), [&](auto io, auto align) {
    with_modes(decay_mode, input_mode, [&](auto logits, auto complement) {
      using io_t = decltype(io);
      const Grid g = cut(p, max_seqlen, kLanes * 8 / static_cast<int>(sizeof(io_t)), forward_ctas(align()) * sm_count());
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
  const int bad = check_sizes("gated_scan", n_seq, total_tokens, channels, io_dtype, decay_mode, input_mode);
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
  const int bad = check_sizes("gated_scan training", n_seq, total_tokens, channels, io_dtype, decay_mode, input_mode);
  if (bad != FRWKV_OK) return bad;
  if (cu_seqlens == nullptr && total_tokens % n_seq != 0)
    return fail(FRWKV_ERR_ARGUMENT, "gated_scan training: dense rows must be a multiple of the sequence count");
  const GatedScanParams p{cu_seqlens, nullptr, status, x, decay, nullptr, x_row_stride, decay_row_stride, initial,
                          final_state, boundary, y, n_seq, total_tokens, channels, total_tokens / n_seq, 0};
  return run_forward(p, io_dtype, decay_mode, input_mode, max_seqlen, stream);
}

extern "C" int frwkv_sm100_gated_scan_train_backward(
    const int32_t* cu_seqlens, const int32_t* status, const void* x, long long x_row_stride, const void* decay,
    long long decay_row_stride, const float* initial, const float* boundary, const void* dy, const float* dfinal,
    void* dx, void* ddecay, float* dinitial, int n_seq, int total_tokens, int channels, int io_dtype, int decay_mode,
    int input_mode, int max_seqlen, void* stream) {
  using namespace frwkv;
  if (!x || !decay || !boundary || !dy || !dx || !ddecay)
    return fail(FRWKV_ERR_ARGUMENT, "gated_scan backward: x, decay, boundary, dy, dx and ddecay must be non-null");
  const int bad = check_sizes("gated_scan backward", n_seq, total_tokens, channels, io_dtype, decay_mode, input_mode);
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
