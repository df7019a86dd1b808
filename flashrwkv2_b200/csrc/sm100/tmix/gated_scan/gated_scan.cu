// Gated scan: in-place serving operator and training forward / backward (see gated_scan.cuh for the arithmetic).
//
// Rows are cut into tiles of kWarps * S consecutive tokens by 32 * V channels, without regard to sequences: a start inside
// a tile cuts the recurrence there.  A lane owns V channels, a warp S tokens, whose gates and inputs stay in registers
// from the only time they are read: one sweep gives the warp's affine map, the CTA joins the maps of its warps, the chain
// (gated_scan.cuh) gives the state before the tile, a second sweep over the registers writes the rows.  So the tokens are
// read once and the outputs written once, time is split over the whole GPU even for one sequence, and a batch of ragged
// sequences is as regular as a dense one.
#include "gated_scan.cuh"

namespace frwkv {
namespace {

constexpr int kTile = FRWKV_GATED_SCAN_TILE;

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

// ---- forward

template <typename io_t, int V, int S, int kWarps, bool LOGITS, bool COMPLEMENT>
__global__ void __launch_bounds__(kWarps * 32, 1024 / (kWarps * 32))
gated_scan_forward_kernel(const GatedScanParams p, const ChainSpace chain) {
  using L = Lanes<V>;
  using F = typename L::type;
  using D = Decay<LOGITS, V>;
  using W = Word<io_t, V>;
  struct Piece {  // a warp's affine map
    F a, b;
  };
  constexpr int kRows = kWarps * S;
  __shared__ Piece pieces[kWarps][32];
  __shared__ unsigned cut[kWarps];
  __shared__ F carry[32];
  __shared__ int next_ticket[2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (p.status != nullptr && p.status[0] != 0) {
    fill_rows_nan<io_t>(p, static_cast<io_t*>(p.y), nullptr, p.boundary != nullptr ? p.final_state : nullptr, p.n_seq);
    return;
  }
  const int active = p.status != nullptr ? p.status[1] : p.total;
  const int n_seq = p.status != nullptr ? p.status[2] : p.n_seq;
  const int tiles = (active + kRows - 1) / kRows * chain.blocks;  // of the rows in use
  int round = 0, ticket = blockIdx.x;
  if (chain.tiles > 1) {
    if (threadIdx.x == 0) next_ticket[0] = atomicAdd(chain.ticket, 1);
    __syncthreads();
    ticket = next_ticket[0];
  }
  typename W::type raw_x[S], raw_d[S];
  const auto fetch = [&](int t) {
    if (t >= tiles) return;
    const int row = t / chain.blocks * kRows + warp * S, channel = (t % chain.blocks * 32 + lane) * V;
    const io_t* x = static_cast<const io_t*>(p.x) + row * p.x_stride + channel;
    const io_t* d = static_cast<const io_t*>(p.decay) + row * p.decay_stride + channel;
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const bool in = row + i < active && channel < p.channels;
      raw_x[i] = in ? W::load(x + i * p.x_stride) : W::zero();
      raw_d[i] = in ? W::load(d + i * p.decay_stride) : W::zero();
    }
  };
  fetch(ticket);
  for (; ticket < tiles; ++round) {
    const int time = ticket / chain.blocks, block = ticket % chain.blocks;
    const int row = time * kRows + warp * S, channel = (block * 32 + lane) * V;
    const bool mine = channel < p.channels;
    int coming = 0;
    if (chain.tiles > 1 && threadIdx.x == 0) coming = atomicAdd(chain.ticket, 1);
    const RowMap rows = map_rows<S>(p, row, active, n_seq);
    const F bias = p.bias != nullptr && mine ? W::unpack(W::load(static_cast<const io_t*>(p.bias) + channel)) : L::all(0.0f);

    // first sweep: gates and inputs into registers, and the warp's map.  A start takes its initial state into u.
    F kept[S], u[S];
    Piece map{L::all(1.0f), L::all(0.0f)};
#pragma unroll
    for (int i = 0; i < S; ++i) {
      kept[i] = D::keep(LOGITS ? L::add(W::unpack(raw_d[i]), bias) : W::unpack(raw_d[i]));
      const F x = W::unpack(raw_x[i]);
      u[i] = COMPLEMENT ? L::mul(D::complement(kept[i]), x) : x;
      if (rows.starts >> i & 1) {
        F h = L::all(0.0f);
        if (p.initial != nullptr && mine) {
          const int seq = rows.seq_of(i);
          // a plain load: the pool is written by this kernel as well
          h = Word<float, V>::unpack(Word<float, V>::load_plain(
              p.initial + static_cast<long long>(p.slots != nullptr ? p.slots[seq] : seq) * p.channels + channel));
        }
        u[i] = D::step(kept[i], h, u[i]);
        map.b = u[i];
      } else {
        map.b = D::step(kept[i], map.b, u[i]);
        map.a = D::fade(kept[i], map.a);
      }
    }
    pieces[warp][lane] = map;
    if (lane == 0) cut[warp] = rows.starts;
    if (chain.tiles > 1 && threadIdx.x == 0) next_ticket[(round + 1) & 1] = coming;
    __syncthreads();
    const int next = chain.tiles > 1 ? next_ticket[(round + 1) & 1] : tiles;
    fetch(next);  // in flight while this tile waits and writes

    // the map of the warps before this one; warp 0 joins all of them for the tile
    bool cut_before = false;
    Piece before{L::all(1.0f), L::all(0.0f)};
    const int count = warp == 0 ? kWarps : warp;
    for (int w = 0; w < count; ++w) {
      const Piece m = pieces[w][lane];
      if (cut[w] != 0) {
        before = m;
        cut_before = true;
      } else {
        before.b = L::fma(m.a, before.b, m.b);
        before.a = L::mul(m.a, before.a);
      }
    }
    const bool open = (cut[0] & 1) == 0;  // the tile continues a sequence
    if (warp == 0) {
      const bool publish = time + 1 < chain.tiles;
      if (publish) Chain<V>::publish(chain, block, time, {before.a, before.b}, cut_before);
      F h = L::all(0.0f);
      if (open) h = Chain<V>::state_before(chain, block, time);
      carry[lane] = h;
      if (publish && time % kGroup == kGroup - 1)
        Chain<V>::publish_state(chain, block, time / kGroup, cut_before ? before.b : L::fma(before.a, h, before.b));
    }
    __syncthreads();
    F h = carry[lane];
    if (warp != 0) h = cut_before ? before.b : L::fma(before.a, h, before.b);

    // second sweep
    if (p.boundary != nullptr && row % kTile == 0 && row < active && mine)
      Word<float, V>::store(p.boundary + static_cast<long long>(row / kTile) * p.channels + channel, h);
    io_t* y = static_cast<io_t*>(p.y) + static_cast<long long>(row) * p.channels + channel;
#pragma unroll
    for (int i = 0; i < S; ++i) {
      h = (rows.starts >> i & 1) ? u[i] : D::step(kept[i], h, u[i]);
      if (mine && row + i < active) W::store(y + static_cast<long long>(i) * p.channels, h);
      if ((rows.ends >> i & 1) && mine) {
        const int seq = rows.seq_of(i);
        Word<float, V>::store(p.final_state + static_cast<long long>(p.slots != nullptr ? p.slots[seq] : seq) * p.channels + channel, h);
      }
    }
    ticket = next;
  }
}

// Decode steps (and rows of a few tokens): a thread walks V channels of one sequence, 16 bytes of a row; no chain.  The
// state pool is most of what a step reads and writes.
template <typename io_t, int V, bool LOGITS, bool COMPLEMENT>
__global__ void __launch_bounds__(256) gated_scan_step_kernel(const GatedScanParams p) {
  using D = Decay<LOGITS, 1>;
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
  alignas(16) io_t x[V], d[V], b[V], y[V];
  alignas(16) float h[V];
  if constexpr (V == 1) {
    h[0] = *state;
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
    for (int i = 0; i < V; ++i) {
      const float kept = D::keep(to_f32(d[i]) + (LOGITS && p.bias != nullptr ? to_f32(b[i]) : 0.f));
      const float value = to_f32(x[i]);
      h[i] = D::step(kept, h[i], COMPLEMENT ? D::complement(kept) * value : value);
      y[i] = from_f32<io_t>(h[i]);
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

template <typename io_t, int V, bool LOGITS, bool COMPLEMENT>
__global__ void __launch_bounds__(256, 2)
gated_scan_backward_kernel(const GatedScanParams p, const GatedScanGrads g, const ChainSpace chain) {
  using L = Lanes<V>;
  using F = typename L::type;
  using D = Decay<LOGITS, V>;
  using W = Word<io_t, V>;
  struct Piece {
    F a, b;
  };
  constexpr int S = 8, kWarps = 8, kRows = kWarps * S;
  static_assert(kRows == kTile, "the forward pass saves one state for each tile of the backward pass");
  __shared__ Piece pieces[kWarps][32], back[kWarps][32];
  __shared__ unsigned cut[kWarps], cut_back[kWarps];
  __shared__ F carry[32];
  __shared__ int next_ticket[2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (p.status != nullptr && p.status[0] != 0) {
    fill_rows_nan<io_t>(p, static_cast<io_t*>(g.dx), static_cast<io_t*>(g.ddecay), g.dinitial, p.n_seq);
    return;
  }
  const int active = p.total, n_seq = p.n_seq;
  const int tiles = chain.tiles * chain.blocks;
  int round = 0, ticket = blockIdx.x;
  if (chain.tiles > 1) {
    if (threadIdx.x == 0) next_ticket[0] = atomicAdd(chain.ticket, 1);
    __syncthreads();
    ticket = next_ticket[0];
  }
  typename W::type raw_x[S], raw_d[S], raw_g[S];
  const auto fetch = [&](int t) {
    if (t >= tiles) return;
    const int row = (chain.tiles - 1 - t / chain.blocks) * kRows + warp * S, channel = (t % chain.blocks * 32 + lane) * V;
    const io_t* x = static_cast<const io_t*>(p.x) + row * p.x_stride + channel;
    const io_t* d = static_cast<const io_t*>(p.decay) + row * p.decay_stride + channel;
    const io_t* dy = static_cast<const io_t*>(g.dy) + static_cast<long long>(row) * p.channels + channel;
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const bool in = row + i < active && channel < p.channels;
      raw_x[i] = in ? W::load(x + i * p.x_stride) : W::zero();
      raw_d[i] = in ? W::load(d + i * p.decay_stride) : W::zero();
      raw_g[i] = in ? W::load(dy + static_cast<long long>(i) * p.channels) : W::zero();
    }
  };
  fetch(ticket);
  for (; ticket < tiles; ++round) {
    const int index = ticket / chain.blocks, block = ticket % chain.blocks;  // index counts against time
    const int time = chain.tiles - 1 - index;
    const int row = time * kRows + warp * S, channel = (block * 32 + lane) * V;
    const bool mine = channel < p.channels;
    int coming = 0;
    if (chain.tiles > 1 && threadIdx.x == 0) coming = atomicAdd(chain.ticket, 1);
    const RowMap rows = map_rows<S>(p, row, active, n_seq);

    // the warp's map of h, and its map of c: the same decays, the gradients against time
    F kept[S], x[S], dy[S], slope[S], start[S];
    Piece map{L::all(1.0f), L::all(0.0f)};
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const F raw = W::unpack(raw_d[i]);
      kept[i] = D::keep(raw);
      slope[i] = D::slope(raw, kept[i]);
      x[i] = W::unpack(raw_x[i]);
      dy[i] = W::unpack(raw_g[i]);
      const F u = COMPLEMENT ? L::mul(D::complement(kept[i]), x[i]) : x[i];
      start[i] = L::all(0.0f);
      if (rows.starts >> i & 1) {
        if (p.initial != nullptr && mine)
          start[i] = Word<float, V>::unpack(Word<float, V>::load(p.initial + static_cast<long long>(rows.seq_of(i)) * p.channels + channel));
        map.b = D::step(kept[i], start[i], u);
      } else {
        map.b = D::step(kept[i], map.b, u);
        map.a = D::fade(kept[i], map.a);
      }
    }
    Piece map_back{L::all(1.0f), L::all(0.0f)};
#pragma unroll
    for (int i = S - 1; i >= 0; --i) {
      if (rows.ends >> i & 1) {
        const F last = g.dfinal != nullptr && mine
                           ? Word<float, V>::unpack(Word<float, V>::load(g.dfinal + static_cast<long long>(rows.seq_of(i)) * p.channels + channel))
                           : L::all(0.0f);
        dy[i] = L::add(dy[i], last);
        map_back.b = D::fade(kept[i], dy[i]);
      } else {
        map_back.b = D::fade(kept[i], L::add(dy[i], map_back.b));
        map_back.a = D::fade(kept[i], map_back.a);
      }
    }
    F h = L::all(0.0f);
    if (mine)
      h = Word<float, V>::unpack(Word<float, V>::load(p.boundary + static_cast<long long>(time) * p.channels + channel));
    pieces[warp][lane] = map;
    back[warp][lane] = map_back;
    if (lane == 0) {
      cut[warp] = rows.starts;
      cut_back[warp] = rows.ends;
    }
    if (chain.tiles > 1 && threadIdx.x == 0) next_ticket[(round + 1) & 1] = coming;
    __syncthreads();
    const int next = chain.tiles > 1 ? next_ticket[(round + 1) & 1] : tiles;
    fetch(next);

    for (int w = 0; w < warp; ++w) {
      const Piece m = pieces[w][lane];
      h = cut[w] != 0 ? m.b : L::fma(m.a, h, m.b);
    }
    bool cut_behind = false;
    Piece behind{L::all(1.0f), L::all(0.0f)};  // of the warps behind this one; the last warp joins all of them
    const int stop = warp == kWarps - 1 ? 0 : warp + 1;
    for (int w = kWarps - 1; w >= stop; --w) {
      const Piece m = back[w][lane];
      if (cut_back[w] != 0) {
        behind = m;
        cut_behind = true;
      } else {
        behind.b = L::fma(m.a, behind.b, m.b);
        behind.a = L::mul(m.a, behind.a);
      }
    }
    if (warp == kWarps - 1) {
      const bool publish = index + 1 < chain.tiles;
      if (publish) Chain<V>::publish(chain, block, index, {behind.a, behind.b}, cut_behind);
      F c = L::all(0.0f);
      // the tile's last row in use continues into the next tile
      if (index > 0 && (rows.ends >> (S - 1) & 1) == 0) c = Chain<V>::state_before(chain, block, index);
      carry[lane] = c;
      if (publish && index % kGroup == kGroup - 1)
        Chain<V>::publish_state(chain, block, index / kGroup, cut_behind ? behind.b : L::fma(behind.a, c, behind.b));
    }
    __syncthreads();
    F c = carry[lane];
    if (warp != kWarps - 1) c = cut_behind ? behind.b : L::fma(behind.a, c, behind.b);

    // states before every row
    F states[S];
#pragma unroll
    for (int i = 0; i < S; ++i) {
      if (rows.starts >> i & 1) h = start[i];
      states[i] = h;
      h = D::step(kept[i], h, COMPLEMENT ? L::mul(D::complement(kept[i]), x[i]) : x[i]);
    }
    io_t* dx = static_cast<io_t*>(g.dx) + static_cast<long long>(row) * p.channels + channel;
    io_t* dd = static_cast<io_t*>(g.ddecay) + static_cast<long long>(row) * p.channels + channel;
#pragma unroll
    for (int i = S - 1; i >= 0; --i) {
      const F grad = (rows.ends >> i & 1) ? dy[i] : L::add(dy[i], c);
      c = D::fade(kept[i], grad);
      if (mine && row + i < active) {
        W::store(dx + static_cast<long long>(i) * p.channels, COMPLEMENT ? L::mul(D::complement(kept[i]), grad) : grad);
        // d / d(1 - rho): the input (complement) less the state before
        const F source = L::fma(states[i], L::all(-1.0f), COMPLEMENT ? x[i] : L::all(0.0f));
        W::store(dd + static_cast<long long>(i) * p.channels, L::mul(L::mul(grad, source), slope[i]));
      }
      if ((rows.starts >> i & 1) && mine && g.dinitial != nullptr)
        Word<float, V>::store(g.dinitial + static_cast<long long>(rows.seq_of(i)) * p.channels + channel, c);
    }
    ticket = next;
  }
}

// ---- launches

constexpr int kForwardWarps = 16, kForwardRows = 8;  // a warp's rows

long long round_up(long long n, long long to) { return (n + to - 1) / to * to; }

// Where the chain lives in the workspace; the flags and the counter come first and are cleared by every call.
ChainSpace chain_space(void* workspace, int total, int channels, int rows, int lanes, long long* clear_bytes, long long* bytes) {
  ChainSpace c{};
  c.tiles = (total + rows - 1) / rows;
  c.groups = (c.tiles + kGroup - 1) / kGroup;
  c.blocks = (channels + lanes - 1) / lanes;
  char* base = static_cast<char*>(workspace);
  const long long tile_flags = 4ll * c.tiles * c.blocks, group_flags = 4ll * c.groups * c.blocks;
  c.ticket = reinterpret_cast<int*>(base);
  c.tile_flags = reinterpret_cast<int*>(base + 16);
  c.group_flags = reinterpret_cast<int*>(base + 16 + tile_flags);
  *clear_bytes = 16 + tile_flags + group_flags;
  const long long maps = round_up(*clear_bytes, 256), states = maps + 8ll * c.tiles * c.blocks * lanes;
  c.maps = reinterpret_cast<float*>(base + maps);
  c.states = reinterpret_cast<float*>(base + states);
  *bytes = c.tiles > 1 ? states + 4ll * c.groups * c.blocks * lanes : 0;
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

// Calls f with the token type and the channels of a lane as compile-time constants: pairs of 16-bit channels (one
// 128-byte row piece for a warp) where `pairs` allows them, else single channels (fp32: 128 bytes as well).
template <typename F> void with_type(int io_dtype, bool pairs, F f) {
  using one = std::integral_constant<int, 1>;
  using two = std::integral_constant<int, 2>;
  if (io_dtype == FRWKV_IO_FP32) f(float{}, one{});
  else if (io_dtype == FRWKV_IO_BF16 && pairs) f(__nv_bfloat16{}, two{});
  else if (io_dtype == FRWKV_IO_BF16) f(__nv_bfloat16{}, one{});
  else if (pairs) f(__half{}, two{});
  else f(__half{}, one{});
}

bool pairs_fit(const GatedScanParams& p) {
  return p.channels % 2 == 0 && p.x_stride % 2 == 0 && p.decay_stride % 2 == 0 && multiple_of(4, {p.x, p.decay, p.bias, p.y}) &&
         multiple_of(8, {p.initial, p.final_state, p.boundary});
}

int run_forward(const GatedScanParams& p, int io_dtype, int decay_mode, int input_mode, void* workspace, void* stream) {
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t cleared = cudaSuccess;
  with_type(io_dtype, pairs_fit(p), [&](auto io, auto v) {
    with_modes(decay_mode, input_mode, [&](auto logits, auto complement) {
      long long clear_bytes, bytes;
      const ChainSpace chain =
          chain_space(workspace, p.total, p.channels, kForwardWarps * kForwardRows, 32 * v(), &clear_bytes, &bytes);
      if (chain.tiles > 1) cleared = cudaMemsetAsync(workspace, 0, clear_bytes, s);
      const long long tiles = static_cast<long long>(chain.tiles) * chain.blocks, resident = 2ll * sm_count();
      const unsigned grid = static_cast<unsigned>(chain.tiles > 1 && tiles > resident ? resident : tiles);
      gated_scan_forward_kernel<decltype(io), v(), kForwardRows, kForwardWarps, logits(), complement()>
          <<<grid, kForwardWarps * 32, 0, s>>>(p, chain);
    });
  });
  if (cleared != cudaSuccess) return fail(FRWKV_ERR_CUDA, "gated_scan: clearing the workspace: %s", cudaGetErrorString(cleared));
  return check_launch("gated_scan_forward_kernel");
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
  // the backward pass has the smaller tiles; the wider of single channels and pairs
  long long clear_bytes, single, pairs;
  frwkv::chain_space(nullptr, total_tokens, channels, FRWKV_GATED_SCAN_TILE, 32, &clear_bytes, &single);
  frwkv::chain_space(nullptr, total_tokens, channels, FRWKV_GATED_SCAN_TILE, 64, &clear_bytes, &pairs);
  return static_cast<size_t>(single > pairs ? single : pairs);
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
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t cleared = cudaSuccess;
  const bool pairs = pairs_fit(p) && multiple_of(4, {dy, dx, ddecay}) && multiple_of(8, {dfinal, dinitial});
  with_type(io_dtype, pairs, [&](auto io, auto v) {
    with_modes(decay_mode, input_mode, [&](auto logits, auto complement) {
      long long clear_bytes, bytes;
      const ChainSpace chain = chain_space(workspace, total_tokens, channels, kTile, 32 * v(), &clear_bytes, &bytes);
      if (chain.tiles > 1) cleared = cudaMemsetAsync(workspace, 0, clear_bytes, s);
      const long long tiles = static_cast<long long>(chain.tiles) * chain.blocks, resident = 2ll * sm_count();
      const unsigned grid = static_cast<unsigned>(chain.tiles > 1 && tiles > resident ? resident : tiles);
      gated_scan_backward_kernel<decltype(io), v(), logits(), complement()><<<grid, 256, 0, s>>>(p, g, chain);
    });
  });
  if (cleared != cudaSuccess) return fail(FRWKV_ERR_CUDA, "gated_scan: clearing the workspace: %s", cudaGetErrorString(cleared));
  return check_launch("gated_scan_backward_kernel");
}
