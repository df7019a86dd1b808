// How the gated scan's kernels walk sequences, and how they are launched (see gated_scan.cuh for the arithmetic).
//
// A cluster of CTAs (one, where there is enough to do) walks one sequence over 64 bytes of channels, the state carried from
// step to step.  In a step each CTA takes a tile of 256 tokens: a warp 64 of them, a lane 16 tokens of 8 bytes of channels.
// The tokens come through shared memory (cp.async, the next tile's while this one is worked on).  A first sweep computes the
// gates into registers and gives each lane an affine map of the state, h -> a h + b, over its 16 tokens; the maps are joined
// over the warp's four lane groups (shuffles), its warps (shared memory) and the cluster's CTAs (distributed shared
// memory), always in the same order; a second sweep over the registers writes the rows.  So the tokens are read once and
// the outputs written once, and nothing waits for anything outside its cluster.
//
// Why this split.  A tile walked by itself and chained to its neighbours through global memory (time split over the whole GPU
// whatever the batch) was built first: a tile then waits for tiles that are in work beside it, 10 us of waiting for each 3 us
// of work (130927 ragged rows of 2560 bf16 channels: 1.2 ms, here 0.42).  16 tokens a lane rather than 8 halves what the joins
// cost (64 x 2048 rows of 2560 channels, when it was chosen: 335 and 400 us), and 64 bytes of channels are two whole sectors of a row and give 64
// units of work for each sequence of 2048 channels.
#pragma once

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
// The moving average by given retentions of 16 bits does not fit into the registers of four (64 x 2048 x 2560: it spills, 391 us;
// with three 347 us).
constexpr int forward_ctas(int align, bool logits, bool complement, int element) {
  return align == 16 && (logits || !complement || element == 4) ? 4 : 3;
}
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
// channels, when it was chosen: 317 us; with the answer read from shared memory 370).
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

// Inclusive join of the maps of a warp's lane groups, in their order.
template <int V> __device__ __forceinline__ void join_groups(Map<V>& m) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int d = kLanes; d < 32; d *= 2) {
    Map<V> before{shuffle_up(m.a, d), shuffle_up(m.low, d), shuffle_up(m.b, d)};
    if (lane >= d) {
      before.then(m);
      m = before;
    }
  }
}

// The state before a lane group's rows, from that before its warp's and the joined maps.
template <int V> __device__ __forceinline__ Lanes<V> state_before_group(const Map<V>& joined, const Lanes<V>& warp_state) {
  const Lanes<V> behind_previous = shuffle_up(joined.apply(warp_state), kLanes);
  return (threadIdx.x & 31) >= kLanes ? behind_previous : warp_state;
}

// The maps of one warp's or CTA's rows in shared memory, by lane along the channels.  SHORT keeps eight bits of `low`, which is
// 2^-23 of a at most: all of it would cost a cluster's CTAs the room of the fourth on an SM.
template <int V, bool SHORT> struct Pieces {
  Lanes<V> a[kLanes], b[kLanes];
  std::conditional_t<SHORT, unsigned[kLanes][V / 2], Lanes<V>[kLanes]> low;

  __device__ __forceinline__ void put(const Map<V>& m) {
    const int at = static_cast<int>(threadIdx.x) % kLanes;
    a[at] = m.a;
    b[at] = m.b;
    if constexpr (SHORT) {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) low[at][i] = pack_pair<__nv_bfloat16>(m.low.v[i]);
    } else {
      low[at] = m.low;
    }
  }
  __device__ __forceinline__ Map<V> get() const {
    const int at = static_cast<int>(threadIdx.x) % kLanes;
    if constexpr (SHORT) {
      Map<V> m{a[at], Lanes<V>::all(0.0f), b[at]};
#pragma unroll
      for (int i = 0; i < V / 2; ++i) m.low.v[i] = make_float2(__uint_as_float(low[at][i] << 16), __uint_as_float(low[at][i] & 0xffff0000u));
      return m;
    } else {
      return Map<V>{a[at], low[at], b[at]};
    }
  }
};

// Joins the CTAs of a cluster: each writes its map into everyone's shared memory (slots[rank]), a cluster barrier, and each
// applies the maps of the ranks before it.  Returns the state before this CTA's tile and moves `carry` behind the cluster's.
template <int V>
__device__ __forceinline__ Lanes<V> join_cluster(const Map<V>& cta, Pieces<V, true>* slots, Lanes<V>& carry) {
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

// `least`: the fewest tokens that there can be.
int check_sizes(const char* what, int n_seq, int total, int least, int channels, int io_dtype, int decay_mode, int input_mode) {
  if (n_seq <= 0 || n_seq > 65535) return fail(FRWKV_ERR_ARGUMENT, "%s: sequence count must be in 1..65535, got %d", what, n_seq);
  if (total < least || channels <= 0)
    return fail(FRWKV_ERR_ARGUMENT, "%s: there must be at least %d token(s) and a channel", what, least);
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
// again.  (65536 rows of 2048 channels: 464 us for single CTAs, 370, 245, 207 for 2, 4, 8; 8 x 4096 rows, where 512 single
// CTAs fill the GPU: 83 us, and 90, 98, 113 us for clusters of 2, 4, 8.)  Very many sequences are taken several to a
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

}  // namespace
}  // namespace frwkv
