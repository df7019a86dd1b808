// Gated scan: in-place serving operator and training forward / backward (see gated_scan.cuh for the arithmetic).
//
// Rows are cut into tiles of 64 consecutive tokens by 256 bytes of channels, without regard to sequences: a start inside a
// tile cuts the recurrence there.  A warp owns 8 tokens, a lane 8 bytes of channels.  The tokens come through shared
// memory (cp.async, the next tile's while this one is worked on); a first sweep computes the gates into registers and
// gives the warp's affine map, the CTA joins the maps of its warps, the chain (gated_scan.cuh) gives the state before the
// tile, a second sweep writes the rows.  So the tokens are read once and the outputs written once, time is split over the
// whole GPU even for one sequence, and a batch of ragged sequences is as regular as a dense one.
#include "gated_scan.cuh"

namespace frwkv {
namespace {

constexpr int kTile = FRWKV_GATED_SCAN_TILE;
constexpr int S = 8, kWarps = 8, kThreads = kWarps * 32;
constexpr int kForwardCtas = 2, kBackwardCtas = 2;  // per SM: 96 KB of staging each
static_assert(S * kWarps == kTile, "the forward pass saves one state for each tile of the backward pass");

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

// Persistent CTAs take tiles in order and learn their next one a tile ahead; with one tile of rows there is no chain
// and no counter.
__device__ __forceinline__ int take_ticket(const ChainSpace& chain) { return atomicAdd(chain.ticket, 1) + 1; }

// A CTA's tiles: time tile, channel block.  Persistent CTAs take tiles in order and learn their next one a tile ahead.
struct Tile {
  int time, block;  // time < 0: none left
};

// Which tile a ticket stands for; `tiles` of them are in use.
__device__ __forceinline__ Tile tile_of(int ticket, int tiles, int blocks) {
  if (ticket >= tiles) return Tile{-1, 0};
  const int time = ticket / blocks;
  return Tile{time, ticket - time * blocks};
}

__device__ __forceinline__ void copies_begun() { asm volatile("cp.async.commit_group;" : : : "memory"); }
template <int LEFT> __device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_group %0;" : : "n"(LEFT) : "memory"); }

// Barrier of a CTA whose warps have taken different ways.
__device__ __forceinline__ void tile_barrier() { asm volatile("bar.sync 1, %0;" : : "n"(kThreads + 32) : "memory"); }

// ---- forward

// Eight warps sweep, a ninth keeps the chain.  While the eight do the first sweep of tile n + 1, the ninth publishes
// tile n's map and finds the state before it, so a tile's second sweep comes one tile after its first and nobody waits for
// another CTA; the gates of two tiles are in registers.  One barrier a tile.
template <typename io_t, int GRANULE, bool LOGITS, bool COMPLEMENT>
__global__ void __launch_bounds__(kThreads + 32, kForwardCtas) gated_scan_forward_kernel(const GatedScanParams p, const ChainSpace chain) {
  constexpr int V = 8 / sizeof(io_t);
  using L = Lanes<V>;
  using D = Decay<LOGITS, COMPLEMENT, V>;
  using A = Access<io_t, GRANULE>;
  // [3 tiles][warp][x or decay][S][lane]; a warp's decays make room for its map and for the state before its rows
  extern __shared__ uint2 staged[];
  constexpr int kTensor = S * 32, kWarpSpace = 2 * kTensor, kTileSpace = kWarps * kWarpSpace;
  __shared__ unsigned cuts[2][kWarps];
  __shared__ Tile ring[4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (p.status != nullptr && p.status[0] != 0) {
    fill_rows_nan<io_t>(p, static_cast<io_t*>(p.y), nullptr, p.boundary != nullptr ? p.final_state : nullptr, p.n_seq);
    return;
  }
  const int active = p.status != nullptr ? p.status[1] : p.total;
  const int n_seq = p.status != nullptr ? p.status[2] : p.n_seq;
  const int tiles = (active + kTile - 1) / kTile * chain.blocks;  // of the rows in use
  const bool chained = chain.tiles > 1;
  const bool more = chained && tiles > static_cast<int>(gridDim.x);  // than one tile for each CTA
  if (threadIdx.x == 0) {  // one after the other: a CTA's tickets ascend
    for (int i = 0; i < 3; ++i) {
      int ticket = i == 0 ? blockIdx.x : tiles;
      if (i == 0 ? chained : more) ticket = atomicAdd(chain.ticket, 1) + 1;
      ring[i] = tile_of(ticket, tiles, chain.blocks);
    }
  }
  __syncthreads();
  const auto map_space = [&](int buffer, int w) { return reinterpret_cast<Map<V>*>(staged + buffer * kTileSpace + w * kWarpSpace + kTensor) + lane; };
  const auto state_space = [&](int buffer, int w) {
    return reinterpret_cast<L*>(staged + buffer * kTileSpace + w * kWarpSpace + kTensor + kTensor / 2) + lane;
  };

  if (warp == kWarps) {
    tile_barrier();
    for (int n = 0, buffer = 0;; ++n, buffer = buffer == 2 ? 0 : buffer + 1) {
      const Tile tile = ring[n & 3];
      if (tile.time < 0) break;
      int ticket = tiles;
      if (more && lane == 0) ticket = atomicAdd(chain.ticket, 1) + 1;
      const unsigned* cut = cuts[n & 1];
      const int group = tile.time / kGroup, behind = tile.time % kGroup;
      const bool publish = tile.time + 1 < chain.tiles;
      Map<V> all = Map<V>::identity();
      bool cut_inside = false;
      if (publish) {
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const Map<V> m = *map_space(buffer, w);
          if (cut[w] != 0) {
            all = m;
            cut_inside = true;
          } else {
            all.then(m);
          }
        }
        Chain<V>::publish(chain, tile.block, tile.time, all, cut_inside);
      }
      L h = L::all(0.0f);
      if ((cut[0] & 1) == 0) h = Chain<V>::state_before(chain, tile.block, group, behind);  // the tile continues a sequence
      if (publish && behind == kGroup - 1)
        Chain<V>::put(Chain<V>::state_at(chain, tile.block, group), cut_inside ? all.b : all.apply(h));
      const int channel = (tile.block * 32 + lane) * V;
      if (p.boundary != nullptr)
        store_states<V>(p.boundary + static_cast<long long>(tile.time) * p.channels + channel, h, min(V, p.channels - channel));
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        *state_space(buffer, w) = h;
        const Map<V> m = *map_space(buffer, w);
        h = cut[w] != 0 ? m.b : m.apply(h);
      }
      if (lane == 0) ring[(n + 3) & 3] = tile_of(ticket, tiles, chain.blocks);
      tile_barrier();
    }
    return;
  }

  const auto fetch = [&](const Tile& t, int buffer) {
    if (t.time >= 0) {
      const int row = t.time * kTile + warp * S, channel = (t.block * 32 + lane) * V;
      const int count = min(V, p.channels - channel), rows = min(S, active - row);
      const io_t* x = static_cast<const io_t*>(p.x) + row * p.x_stride + channel;
      const io_t* d = static_cast<const io_t*>(p.decay) + row * p.decay_stride + channel;
      uint2* to = staged + buffer * kTileSpace + warp * kWarpSpace + lane;
#pragma unroll
      for (int i = 0; i < S; ++i) {
        const int n = i < rows ? count : 0;
        A::stage(to + i * 32, n > 0 ? x + i * p.x_stride : static_cast<const io_t*>(p.x), n);
        A::stage(to + kTensor + i * 32, n > 0 ? d + i * p.decay_stride : static_cast<const io_t*>(p.decay), n);
      }
    }
    copies_begun();
  };
  const auto state_row = [&](const RowMap& rows, int i, int channel) {  // of row i's sequence
    const int seq = rows.seq_of(i);
    return static_cast<long long>(p.slots != nullptr ? p.slots[seq] : seq) * p.channels + channel;
  };
  // First sweep: the gates into registers, and the warp's map.  A start keeps the state behind it in place of its gate.
  const auto first_sweep = [&](const Tile& tile, int n, int buffer, L (&kept)[S]) {
    const int row = tile.time * kTile + warp * S, channel = (tile.block * 32 + lane) * V;
    const int count = min(V, p.channels - channel);
    const RowMap rows = map_rows<S>(p, row, active, n_seq);
    L bias = L::all(0.0f);
    if (LOGITS && p.bias != nullptr) {
      const io_t* from = static_cast<const io_t*>(p.bias) + channel;
      float b[V];
#pragma unroll
      for (int i = 0; i < V; ++i) b[i] = i < count ? to_f32(from[i]) * -kLog2e : 0.0f;
#pragma unroll
      for (int i = 0; i < V / 2; ++i) bias.v[i] = make_float2(b[2 * i], b[2 * i + 1]);
    }
    const uint2* x = staged + buffer * kTileSpace + warp * kWarpSpace + lane;
    Map<V> map = Map<V>::identity();
#pragma unroll
    for (int i = 0; i < S; ++i) {
      kept[i] = D::keep(unpack<io_t>(x[kTensor + i * 32]), bias);
      const L value = unpack<io_t>(x[i * 32]);
      if (rows.starts >> i & 1) {
        const L h = p.initial != nullptr ? load_states<V>(p.initial + state_row(rows, i, channel), count) : L::all(0.0f);
        kept[i] = map.b = D::step(kept[i], h, value);
      } else {
        map.b = D::step(kept[i], map.b, value);
        map.a = D::fade(kept[i], map.a);
      }
    }
    __syncwarp();  // every lane has read its decays
    *map_space(buffer, warp) = map;
    if (lane == 0) cuts[n & 1][warp] = rows.starts;
    return rows;
  };
  const auto second_sweep = [&](const Tile& tile, const RowMap& rows, int buffer, const L (&kept)[S]) {
    const int row = tile.time * kTile + warp * S, channel = (tile.block * 32 + lane) * V;
    const int count = min(V, p.channels - channel);
    const uint2* x = staged + buffer * kTileSpace + warp * kWarpSpace + lane;
    L h = *state_space(buffer, warp);
    io_t* y = static_cast<io_t*>(p.y) + static_cast<long long>(row) * p.channels + channel;
#pragma unroll
    for (int i = 0; i < S; ++i) {
      h = (rows.starts >> i & 1) ? kept[i] : D::step(kept[i], h, unpack<io_t>(x[i * 32]));
      if (row + i < active) A::store(y + static_cast<long long>(i) * p.channels, h, count);
      if (rows.ends >> i & 1) store_states<V>(p.final_state + state_row(rows, i, channel), h, count);
    }
    __syncwarp();  // every lane has read its state: the space may be filled again
  };
  L kept_even[S], kept_odd[S];
  RowMap rows_even, rows_odd;
  Tile tile = ring[0];
  fetch(tile, 0);
  fetch(ring[1], 1);
  fetch(ring[2], 2);
  if (tile.time >= 0) {
    copies_done<2>();
    rows_even = first_sweep(tile, 0, 0, kept_even);
  }
  tile_barrier();
  // one tile: the first sweep of the next, the barrier, the second sweep of this one, its space to the tile after next
  int n = 0, buffer = 0;
  const auto advance = [&](const RowMap& rows, const L (&kept)[S], RowMap& next_rows, L (&next_kept)[S]) {
    const Tile next = ring[(n + 1) & 3];
    const int next_buffer = buffer == 2 ? 0 : buffer + 1;
    if (next.time >= 0) {
      copies_done<1>();
      next_rows = first_sweep(next, n + 1, next_buffer, next_kept);
    }
    tile_barrier();
    second_sweep(tile, rows, buffer, kept);
    fetch(ring[(n + 3) & 3], buffer);
    tile = next;
    buffer = next_buffer;
    ++n;
  };
  while (tile.time >= 0) {
    advance(rows_even, kept_even, rows_odd, kept_odd);
    if (tile.time < 0) break;
    advance(rows_odd, kept_odd, rows_even, kept_even);
  }
  copies_done<0>();
}

// Decode steps (and rows of a few tokens): a thread walks V channels of one sequence, 16 bytes of a row; no chain.  The
// state pool is most of what a step reads and writes.
template <typename io_t, int V, bool LOGITS, bool COMPLEMENT>
__global__ void __launch_bounds__(256) gated_scan_step_kernel(const GatedScanParams p) {
  if (p.status != nullptr && p.status[0] != 0) {
    fill_rows_nan<io_t>(p, static_cast<io_t*>(p.y), nullptr, nullptr, 0);
    return;
  }
  const int n_seq = p.status != nullptr ? p.status[2] : p.n_seq;
  const unsigned per_row = static_cast<unsigned>(p.channels / V), at = blockIdx.x * 256u + threadIdx.x;
  const int seq = static_cast<int>(at / per_row), channel = static_cast<int>(at % per_row) * V;
  if (seq >= n_seq) return;
  const int first = p.cu[seq], last = p.cu[seq + 1];
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
// With c_t = rho_t g_t the same recurrence runs against time: g_t = dy_t + c_{t+1}, cut behind a sequence's last token,
// where c is the final state's gradient.  A tile first scans h forward from the state saved before it, keeps the
// states in registers, and then does with g what the forward pass does with h.

template <typename io_t, int GRANULE, bool LOGITS, bool COMPLEMENT>
__global__ void __launch_bounds__(kThreads, kBackwardCtas)
gated_scan_backward_kernel(const GatedScanParams p, const GatedScanGrads g, const ChainSpace chain) {
  constexpr int V = 8 / sizeof(io_t);
  using L = Lanes<V>;
  using D = Decay<LOGITS, COMPLEMENT, V>;
  using A = Access<io_t, GRANULE>;
  extern __shared__ uint2 staged[];  // [2 tiles][warp][x, decay or dy][S][lane]
  __shared__ Map<V> pieces[kWarps][32];  // of h
  __shared__ L carry[32];
  __shared__ L back[kWarps][32];         // B of c's map; its A is that of h's where neither is cut
  __shared__ unsigned cut[kWarps], cut_back[kWarps];
  __shared__ Tile coming[2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (p.status != nullptr && p.status[0] != 0) {
    fill_rows_nan<io_t>(p, static_cast<io_t*>(g.dx), static_cast<io_t*>(g.ddecay), g.dinitial, p.n_seq);
    return;
  }
  const int active = p.total, tiles = chain.tiles * chain.blocks;
  const bool chained = chain.tiles > 1;
  if (threadIdx.x == 0) coming[0] = tile_of(chained ? atomicAdd(chain.ticket, 1) + 1 : blockIdx.x, tiles, chain.blocks);
  __syncthreads();
  Tile tile = coming[0];  // counts against time
  const auto fetch = [&](const Tile& t, int buffer) {
    if (t.time >= 0) {
      const int row = (chain.tiles - 1 - t.time) * kTile + warp * S, channel = (t.block * 32 + lane) * V;
      const int count = min(V, p.channels - channel), rows = min(S, active - row);
      const io_t* x = static_cast<const io_t*>(p.x) + row * p.x_stride + channel;
      const io_t* d = static_cast<const io_t*>(p.decay) + row * p.decay_stride + channel;
      const io_t* dy = static_cast<const io_t*>(g.dy) + static_cast<long long>(row) * p.channels + channel;
      uint2* to = staged + (buffer * kWarps + warp) * 3 * S * 32 + lane;
#pragma unroll
      for (int i = 0; i < S; ++i) {
        const int n = i < rows ? count : 0;
        A::stage(to + i * 32, n > 0 ? x + i * p.x_stride : static_cast<const io_t*>(p.x), n);
        A::stage(to + (S + i) * 32, n > 0 ? d + i * p.decay_stride : static_cast<const io_t*>(p.decay), n);
        A::stage(to + (2 * S + i) * 32, n > 0 ? dy + static_cast<long long>(i) * p.channels : static_cast<const io_t*>(g.dy), n);
      }
    }
    copies_begun();
  };
  fetch(tile, 0);
  for (int round = 0; tile.time >= 0; ++round) {
    const int index = tile.time, time = chain.tiles - 1 - index;
    const int row = time * kTile + warp * S, channel = (tile.block * 32 + lane) * V;
    const int count = min(V, p.channels - channel);
    if (threadIdx.x == 0)
      coming[(round + 1) & 1] = tile_of(chained ? atomicAdd(chain.ticket, 1) + 1 : tiles, tiles, chain.blocks);
    const RowMap rows = map_rows<S>(p, row, active, p.n_seq);
    L h = load_states<V>(p.boundary + static_cast<long long>(time) * p.channels + channel, count);
    const auto state_of = [&](const float* states, int i) {  // of row i's sequence
      return states != nullptr ? load_states<V>(states + static_cast<long long>(rows.seq_of(i)) * p.channels + channel, count)
                               : L::all(0.0f);
    };
    copies_done<0>();
    const uint2* x = staged + ((round & 1) * kWarps + warp) * 3 * S * 32 + lane;
    const uint2* d = x + S * 32;
    const uint2* dy = d + S * 32;

    // the warp's map of h, and its map of c: the same decays, the gradients against time
    L kept[S];
    Map<V> map = Map<V>::identity();
    L back_b = L::all(0.0f);
#pragma unroll
    for (int i = 0; i < S; ++i) {
      kept[i] = D::keep(unpack<io_t>(d[i * 32]), L::all(0.0f));
      const L value = unpack<io_t>(x[i * 32]);
      if (rows.starts >> i & 1) {
        map.b = D::step(kept[i], state_of(p.initial, i), value);
      } else {
        map.b = D::step(kept[i], map.b, value);
      }
      map.a = D::fade(kept[i], map.a);  // of all rows: it counts only where no bound lies between them
    }
#pragma unroll
    for (int i = S - 1; i >= 0; --i)
      back_b = D::fade(kept[i], add(unpack<io_t>(dy[i * 32]), (rows.ends >> i & 1) ? state_of(g.dfinal, i) : back_b));
    pieces[warp][lane] = map;
    back[warp][lane] = back_b;
    if (lane == 0) {
      cut[warp] = rows.starts;
      cut_back[warp] = rows.ends;
    }
    __syncthreads();
    const Tile next = coming[(round + 1) & 1];
    fetch(next, (round + 1) & 1);

    // the map of the warps behind this one; the last warp joins all of them and publishes the tile's
    const bool open = index > 0 && (cut_back[kWarps - 1] >> (S - 1) & 1) == 0;  // the last row's sequence goes on
    const int group = index / kGroup, before = index % kGroup;
    bool cut_behind = false;
    Map<V> behind = Map<V>::identity();
    const int stop = warp == kWarps - 1 ? 0 : warp + 1;
    for (int w = kWarps - 1; w >= stop; --w) {
      const Map<V> m{pieces[w][lane].a, back[w][lane]};
      if (cut_back[w] != 0) {
        behind = m;
        cut_behind = true;
      } else {
        behind.then(m);
      }
    }
    const bool publish = index + 1 < chain.tiles;
    if (warp == kWarps - 1 && publish) Chain<V>::publish(chain, tile.block, index, behind, cut_behind);
    L c = L::all(0.0f);
    // what ddecay needs of the states: the state before every row, less its input (complement)
    for (int w = 0; w < warp; ++w) {
      const Map<V> m = pieces[w][lane];
      h = cut[w] != 0 ? m.b : m.apply(h);
    }
    L states[S];
#pragma unroll
    for (int i = 0; i < S; ++i) {
      if (rows.starts >> i & 1) h = state_of(p.initial, i);
      const L value = unpack<io_t>(x[i * 32]);
      states[i] = COMPLEMENT ? minus(h, value) : h;
      h = D::step(kept[i], h, value);
    }
    if (warp == kWarps - 1) {
      if (open) c = Chain<V>::state_before(chain, tile.block, group, before);
      carry[lane] = c;
    }
    __syncthreads();
    c = carry[lane];
    if (warp == kWarps - 1) {
      if (publish && before == kGroup - 1)
        Chain<V>::put(Chain<V>::state_at(chain, tile.block, group), cut_behind ? behind.b : behind.apply(c));
    } else {
      c = cut_behind ? behind.b : behind.apply(c);
    }

    io_t* dx = static_cast<io_t*>(g.dx) + static_cast<long long>(row) * p.channels + channel;
    io_t* dd = static_cast<io_t*>(g.ddecay) + static_cast<long long>(row) * p.channels + channel;
#pragma unroll
    for (int i = S - 1; i >= 0; --i) {
      const L grad = add(unpack<io_t>(dy[i * 32]), (rows.ends >> i & 1) ? state_of(g.dfinal, i) : c);
      c = D::fade(kept[i], grad);
      if (row + i < active) {
        A::store(dx + static_cast<long long>(i) * p.channels, D::input_grad(kept[i], grad), count);
        L drho = mul(grad, states[i]);
        if constexpr (LOGITS) drho = mul(drho, D::slope(D::sigmoid(unpack<io_t>(d[i * 32]), L::all(0.0f)), kept[i]));
        A::store(dd + static_cast<long long>(i) * p.channels, drho, count);
      }
      if ((rows.starts >> i & 1) && g.dinitial != nullptr)
        store_states<V>(g.dinitial + static_cast<long long>(rows.seq_of(i)) * p.channels + channel, c, count);
    }
    tile = next;
  }
  copies_done<0>();
}

// ---- launches

// Where the chain lives in the workspace.  All of it is filled with kEmpty by every call that uses it.
ChainSpace chain_space(void* workspace, int total, int channels, int lanes, long long* bytes) {
  ChainSpace c{};
  c.tiles = (total + kTile - 1) / kTile;
  c.groups = (c.tiles + kGroup - 1) / kGroup;
  c.blocks = (channels + lanes - 1) / lanes;
  char* base = static_cast<char*>(workspace);
  const long long maps = 8ll * c.tiles * c.blocks * lanes, states = 4ll * c.groups * c.blocks * lanes;
  c.ticket = reinterpret_cast<int*>(base);
  c.maps = reinterpret_cast<float*>(base + 256);
  c.states = reinterpret_cast<float*>(base + 256 + maps);
  *bytes = c.tiles > 1 ? 256 + maps + states : 0;
  return c;
}

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

int check_sizes(const char* what, int n_seq, int total, int channels, int io_dtype, int decay_mode, int input_mode,
                const void* workspace, size_t workspace_bytes) {
  if (n_seq <= 0 || n_seq > 65535) return fail(FRWKV_ERR_ARGUMENT, "%s: sequence count must be in 1..65535, got %d", what, n_seq);
  if (total < n_seq || channels <= 0)
    return fail(FRWKV_ERR_ARGUMENT, "%s: every sequence needs a token and there must be a channel", what);
  if (static_cast<long long>((total + kTile - 1) / kTile) * ((channels + 31) / 32) > 0x7f000000ll)
    return fail(FRWKV_ERR_UNSUPPORTED, "%s: more than 2^31 tiles of %d tokens by 32 channels", what, kTile);
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

// Calls f with the token type and the largest access that fits everything as compile-time constants.
template <typename F> void with_type(int io_dtype, int granule, F f) {
  using two = std::integral_constant<int, 2>;
  using four = std::integral_constant<int, 4>;
  using eight = std::integral_constant<int, 8>;
  if (io_dtype == FRWKV_IO_FP32) granule == 8 ? f(float{}, eight{}) : f(float{}, four{});
  else if (io_dtype == FRWKV_IO_BF16) granule == 8 ? f(__nv_bfloat16{}, eight{}) : granule == 4 ? f(__nv_bfloat16{}, four{}) : f(__nv_bfloat16{}, two{});
  else granule == 8 ? f(__half{}, eight{}) : granule == 4 ? f(__half{}, four{}) : f(__half{}, two{});
}

// The bytes of a token row that one access may move: 8 where the channels, the strides and all starts allow it.
int granule_of(const GatedScanParams& p, int io_dtype, std::initializer_list<const void*> rows) {
  const int element = io_dtype == FRWKV_IO_FP32 ? 4 : 2;
  for (int granule = 8; granule > element; granule /= 2) {
    const int n = granule / element;
    if (p.channels % n == 0 && p.x_stride % n == 0 && p.decay_stride % n == 0 && multiple_of(granule, rows)) return granule;
  }
  return element;
}

// Launches a chained kernel: fills the chain's space, as many CTAs as are resident at most.
template <typename K, typename... Args>
int launch_chained(K kernel, int lanes, int threads, int tensors, int ctas, const GatedScanParams& p, void* workspace, cudaStream_t s,
                   const char* what, Args... args) {
  long long bytes;
  const ChainSpace chain = chain_space(workspace, p.total, p.channels, lanes, &bytes);
  const int shared = tensors * kTile * 256;  // 256-byte rows
  cudaError_t error = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, shared);
  if (error == cudaSuccess && chain.tiles > 1) error = cudaMemsetAsync(workspace, 0xff, bytes, s);
  if (error != cudaSuccess) return fail(FRWKV_ERR_CUDA, "%s: preparing the launch: %s", what, cudaGetErrorString(error));
  const long long tiles = static_cast<long long>(chain.tiles) * chain.blocks, resident = static_cast<long long>(ctas) * sm_count();
  const unsigned grid = static_cast<unsigned>(chain.tiles > 1 && tiles > resident ? resident : tiles);
  kernel<<<grid, threads, shared, s>>>(p, args..., chain);
  return check_launch(what);
}

int run_forward(const GatedScanParams& p, int io_dtype, int decay_mode, int input_mode, void* workspace, void* stream) {
  int rc = FRWKV_OK;
  with_type(io_dtype, granule_of(p, io_dtype, {p.x, p.decay, p.y}), [&](auto io, auto granule) {
    with_modes(decay_mode, input_mode, [&](auto logits, auto complement) {
      rc = launch_chained(gated_scan_forward_kernel<decltype(io), granule(), logits(), complement()>, 256 / static_cast<int>(sizeof(io)), kThreads + 32, 3 * 2,
                          kForwardCtas, p, workspace, static_cast<cudaStream_t>(stream), "gated_scan_forward_kernel");
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
      gated_scan_step_kernel<decltype(io), v(), logits(), complement()><<<grid, 256, 0, s>>>(p);
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

extern "C" size_t frwkv_sm100_gated_scan_workspace_bytes(int total_tokens, int channels) {
  if (total_tokens <= 0 || channels <= 0) return 0;
  long long wide, narrow;  // channel blocks of fp32 and of 16-bit tokens
  frwkv::chain_space(nullptr, total_tokens, channels, 64, &wide);
  frwkv::chain_space(nullptr, total_tokens, channels, 128, &narrow);
  return static_cast<size_t>(wide > narrow ? wide : narrow);
}

extern "C" int frwkv_sm100_gated_scan(
    const int32_t* cu_seqlens, const int32_t* slots, const int32_t* status, float* state_pool, const void* x,
    long long x_row_stride, const void* decay, long long decay_row_stride, const void* decay_bias, void* y, int n_seq,
    int total_tokens, int channels, int io_dtype, int decay_mode, int input_mode, int max_seqlen, void* workspace,
    size_t workspace_bytes, void* stream) {
  using namespace frwkv;
  if (!cu_seqlens || !slots || !state_pool || !x || !decay || !y)
    return fail(FRWKV_ERR_ARGUMENT, "gated_scan: cu_seqlens, slots, state_pool, x, decay and y must be non-null");
  if (decay_bias != nullptr && decay_mode != FRWKV_DECAY_LOGITS)
    return fail(FRWKV_ERR_ARGUMENT, "gated_scan: decay_bias only applies to decay logits");
  const int bad = check_sizes("gated_scan", n_seq, total_tokens, channels, io_dtype, decay_mode, input_mode, workspace,
                              workspace_bytes);
  if (bad != FRWKV_OK) return bad;
  const GatedScanParams p{cu_seqlens, slots, status, x, decay, decay_bias, x_row_stride, decay_row_stride, state_pool,
                          state_pool, nullptr, y, n_seq, total_tokens, channels, 0};
  if (max_seqlen == 1 && static_cast<long long>(n_seq) * channels < 0x7fffffffll)
    return run_steps(p, io_dtype, decay_mode, input_mode, stream);
  return run_forward(p, io_dtype, decay_mode, input_mode, workspace, stream);
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
  return run_forward(p, io_dtype, decay_mode, input_mode, workspace, stream);
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
  int rc = FRWKV_OK;
  with_type(io_dtype, granule_of(p, io_dtype, {x, decay, dy, dx, ddecay}), [&](auto io, auto granule) {
    with_modes(decay_mode, input_mode, [&](auto logits, auto complement) {
      rc = launch_chained(gated_scan_backward_kernel<decltype(io), granule(), logits(), complement()>, 256 / static_cast<int>(sizeof(io)), kThreads, 2 * 3,
                          kBackwardCtas, p, workspace, static_cast<cudaStream_t>(stream), "gated_scan_backward_kernel", g);
    });
  });
  return rc;
}
