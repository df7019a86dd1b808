// Log probabilities of given tokens, entropy and top alternatives of rows of vocabulary logits; gradient.
//
// With m the largest logit of a row, z_j = (x_j - m) / T and e_j = exp(z_j):  S = sum e_j,  W = sum e_j z_j,
//   logprob = z_id - log S,   entropy = log S - W / S,
//   dx_j = (a ([j = id] - p_j) - b p_j (log p_j + entropy)) / T,   p_j = e_j / S.
// Differences to m are formed before anything is scaled, so a common offset of a row costs no precision; exponents are
// base 2 inside (z times log2 e).  Everything is fp32 but the logits and their gradient.
//
// The row is read once (backward: read once, written once), so HBM is the floor; an element also costs one exponential on the
// SFU, 16 a clock and SM, which is 0.7 of that floor for 16-bit logits.  Measured on bf16: 4096 x 65536 91 us = 0.90 of the
// HBM copy rate (106 us when it runs for seconds and the power limit takes the clock down), with the top 20 119 us;
// 777 x 50277 fp32 28 us = 0.85 (777 CTAs are one round on 888 places); gradient of 2048 x 65536 84 us = 0.97.
// 32 x 65536 with the top 20: 12.3 us, all latency (launch, load, selection, two cluster barriers).
#include "../common.cuh"

#include <cooperative_groups.h>

#include <type_traits>

namespace frwkv {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kBatch = 4;      // 16-byte loads that a thread has in flight
constexpr int kAbove = 512;    // room for logits above the bar that bounds the top_k (see select_top)
constexpr int kEqual = 128;    // room for logits equal to it
constexpr int kMaxCluster = 4;         // 32 rows of 65536, top 20: 17.8 us for single CTAs, 15.3, 13.4, 14.4 us for 2, 4, 8 a row
// No more CTAs than this by splitting rows.  So a row's sums are added up in another order, and differ in their last bits, where the
// number of rows (or the row's alignment) changes.  Sections that follow from the vocabulary alone, summed by themselves whoever
// takes them, would agree at any number of rows, but cost what they do many rows most: 4096 x 65536 bf16 101 -> 105 us,
// 777 x 50277 fp32 with the top 8 33.1 -> 35.7 us.
constexpr int kClusterCtas = 512;
constexpr int kClusterBytes = 16384;   // and no part of a row smaller than this (one batch of a CTA)
// exp2 of anything below is 0 in fp32; keeps 0 * -inf out of W and of the gradient
constexpr float kLowest = -160.0f;
constexpr float kSlack = 4.0f;  // how far, in powers of two, a logit may lie above the reference of a thread's sums

struct Rows {
  const void* logits;
  long long rows, inner, stride_outer, stride_inner;
  const void* ids;
  int ids_are_int64;
  long long ignore_index;
  int vocab;
  float inv_temperature;
};

// A row's first logit; rows and p.inner fit in 31 bits.
template <typename io_t> __device__ __forceinline__ const io_t* row_start(const Rows& p, long long row) {
  const unsigned at = static_cast<unsigned>(row), inner = static_cast<unsigned>(p.inner);
  const unsigned outer = at < inner ? 0 : at / inner;
  return static_cast<const io_t*>(p.logits) + static_cast<long long>(outer) * p.stride_outer +
         static_cast<long long>(at - outer * inner) * p.stride_inner;
}

__device__ __forceinline__ long long row_id(const Rows& p, long long row) {
  return p.ids_are_int64 ? static_cast<const long long*>(p.ids)[row] : static_cast<const int*>(p.ids)[row];
}

__device__ __forceinline__ float exp2_fast(float x) {  // relative error about 2^-22, that of exp2f
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float max_keep_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// Total order of logits, larger first: monotone in the value, -0 equal to +0, NaN above everything (but below the
// largest number, which means "no bound yet").  Never 0.
__device__ __forceinline__ unsigned order_of(float x) {
  if (x != x) return 0xfffffffeu;
  const unsigned bits = __float_as_uint(x + 0.0f);
  return (bits & 0x80000000u) ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned order) {
  if (order == 0xfffffffeu) return __int_as_float(0x7fffffff);
  return __uint_as_float((order & 0x80000000u) ? order & 0x7fffffffu : ~order);
}
// Larger logits first, then lower ids.
__device__ __forceinline__ unsigned long long rank_key(float x, int id) {
  return static_cast<unsigned long long>(order_of(x)) << 32 | (0xffffffffu - static_cast<unsigned>(id));
}
__device__ __forceinline__ int key_id(unsigned long long key) {
  return static_cast<int>(0xffffffffu - static_cast<unsigned>(key));
}

// 16 bytes of logits as pairs of floats.
template <typename io_t> struct Pack {
  static constexpr int kCount = 16 / sizeof(io_t);
  uint4 raw;

  __device__ __forceinline__ void load(const io_t* p) {
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(raw.x), "=r"(raw.y), "=r"(raw.z), "=r"(raw.w) : "l"(p));
  }
  __device__ __forceinline__ void fill_lowest() {  // -inf in every place
    unsigned word;
    if constexpr (sizeof(io_t) == 4) word = 0xff800000u;
    else if constexpr (std::is_same_v<io_t, __nv_bfloat16>) word = 0xff80ff80u;
    else word = 0xfc00fc00u;
    raw = make_uint4(word, word, word, word);
  }
  __device__ __forceinline__ unsigned word(int i) const { return i == 0 ? raw.x : i == 1 ? raw.y : i == 2 ? raw.z : raw.w; }
  __device__ __forceinline__ float2 pair(int i) const {
    if constexpr (sizeof(io_t) == 4) {
      return make_float2(__uint_as_float(word(2 * i)), __uint_as_float(word(2 * i + 1)));
    } else if constexpr (std::is_same_v<io_t, __nv_bfloat16>) {
      const unsigned w = word(i);
      return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    } else {
      const unsigned w = word(i);
      return __half22float2(*reinterpret_cast<const __half2*>(&w));
    }
  }
};

// The largest value of kBatch packs; NaN where there is one.
template <typename io_t> __device__ __forceinline__ float largest(const Pack<io_t> (&v)[kBatch]) {
  if constexpr (sizeof(io_t) == 4) {
    float top = -INFINITY;
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) top = max_keep_nan(top, __uint_as_float(v[b].word(i)));
    return top;
  } else {
    using pair_t = std::conditional_t<std::is_same_v<io_t, __nv_bfloat16>, __nv_bfloat162, __half2>;
    unsigned first = v[0].word(0);
    pair_t top = *reinterpret_cast<pair_t*>(&first);
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
#pragma unroll
      for (int i = b == 0 ? 1 : 0; i < 4; ++i) {
        const unsigned w = v[b].word(i);
        top = __hmax2_nan(top, *reinterpret_cast<const pair_t*>(&w));
      }
    return max_keep_nan(to_f32(top.x), to_f32(top.y));
  }
}

// A thread's largest logit, and its sums relative to a reference logit m that is not far below it (two lanes each, for
// packed fp32 arithmetic).  The reference moves only when a batch exceeds it by more than 2^kSlack in the exponential: with
// the maximum itself as reference some lane of a warp would move it in almost every batch.  An exponent of kSlack costs
// no more precision than one of -kSlack.
struct Sums {
  float top, m;
  float2 s, w;
  float next;  // the largest logit outside the batch that holds `top`
  int top_batch;

  __device__ __forceinline__ void clear() {
    top = next = m = -INFINITY;
    top_batch = 0;
    s = w = make_float2(0.f, 0.f);
  }
  // moves the sums to a larger reference: e_j becomes e_j f and z_j becomes z_j + c, f = 2^c
  __device__ __forceinline__ void rise(float to, float k) {
    if (m != -INFINITY) {
      const float c = fmaxf((m - to) * k, kLowest), f = exp2_fast(c);
      w = make_float2(f * fmaf(c, s.x, w.x), f * fmaf(c, s.y, w.y));
      s = make_float2(f * s.x, f * s.y);
    }
    m = to;
  }
  template <typename io_t, bool TOP> __device__ __forceinline__ void add(const Pack<io_t> (&v)[kBatch], int batch, float k) {
    const float most = largest(v);
    if (most == -INFINITY) return;
    if ((most - m) * k > kSlack) rise(most, k);
    if constexpr (TOP) {
      next = fmaxf(next, fminf(top, most));
      top_batch = most > top ? batch : top_batch;
    }
    top = fmaxf(top, most);
    const float2 minus_m = make_float2(-m, -m), k2 = make_float2(k, k);
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
#pragma unroll
      for (int i = 0; i < Pack<io_t>::kCount / 2; ++i) {
        float2 z = __fmul2_rn(__fadd2_rn(v[b].pair(i), minus_m), k2);
        z = make_float2(max_keep_nan(z.x, kLowest), max_keep_nan(z.y, kLowest));
        const float2 e = make_float2(exp2_fast(z.x), exp2_fast(z.y));
        s = __fadd2_rn(s, e);
        w = __ffma2_rn(e, z, w);
      }
    }
  }
  __device__ __forceinline__ void add(float x, float k) {
    if (x == -INFINITY) return;
    if ((x - m) * k > kSlack) rise(x, k);
    top = fmaxf(top, x);
    const float z = max_keep_nan((x - m) * k, kLowest), e = exp2_fast(z);
    s.x += e;
    w.x = fmaf(e, z, w.x);
  }
};

// Largest logit, and sums relative to it (relative to m before they are joined).
struct Total {
  float m, s, w;
};

// Joins the totals of a warp's lanes; every lane gets the result.  All sums are moved to the common maximum of `top` and
// added in a fixed tree.  A part without a reference holds nothing, or NaN.
__device__ __forceinline__ Total join_lanes(float top, Total part, float k) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  const float c = part.m == -INFINITY ? 0.f : fmaxf((part.m - top) * k, kLowest), f = exp2_fast(c);
  float s = f * part.s, w = f * fmaf(c, part.s, part.w);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, d);
    w += __shfl_xor_sync(0xffffffffu, w, d);
  }
  return Total{top, s, w};
}

// A CTA's part of a row: packs [first, last) behind `lead` single logits; the CTA that owns the singles takes those
// before the first aligned pack and behind the last.
template <typename io_t> struct Part {
  const io_t* row;
  int lead, packs, vocab;  // of the whole row
  int first, last;         // packs of this CTA
  bool singles;

  __device__ __forceinline__ int tail() const { return lead + packs * Pack<io_t>::kCount; }
  __device__ __forceinline__ int single_count() const { return singles ? lead + (vocab - tail()) : 0; }
  __device__ __forceinline__ int single(int i) const { return i < lead ? i : tail() + i - lead; }
  __device__ __forceinline__ int pack_id(int pack) const { return lead + pack * Pack<io_t>::kCount; }
};

struct TopScratch {
  // keys above the bar, and from kAbove on those equal to it; the joined lists of a cluster
  unsigned long long found[kAbove + kEqual];
  unsigned long long list[FRWKV_TOP_K_MAX];  // the answer: descending keys, 0 where there are fewer
  unsigned long long warp_best[kWarps];
  unsigned bars[kWarps];
  int hot[kThreads], wide[kThreads], warp_count[kWarps];
  int hot_count, wide_count, above_count, equal_count;
};

// Writes the CTA's top_k keys into t.list.
//
// While the sums were taken every thread kept its largest logit, the batch of loads that held it and the largest one
// outside that batch.  Each warp offers its ceil(top_k / 8)-th largest of these 32 maxima; the smallest offer is a bar that
// at least top_k logits reach, and few more do (about 35 of 65536 for top_k 20) where the row's finite logits lie in all warps.
// Only the batches of the threads that reach the bar are read again (a tenth of the row, from L2), all of a thread's batches
// where its second one may reach it too; what reaches it is collected and ranked by counting.  Logits equal to the bar count
// only as far as those above do not suffice; where they are too many to collect (masked rows: -inf), the lowest ids among them
// are found in order.  Rows with NaN, and with more logits above the bar than there is room for, take top_k passes.
//
// Where some warp has too few finite maxima its offer, and so the bar, is the mask (-inf): all of the row is read again, each of
// its masked logits counted by an atomic, and all finite ones are candidates.  That is right but slow.  256 rows of 65536 bf16,
// top 20: 17.5 us as they come, 52 us with 1 to 20 tokens allowed, 33 with 200, 18 with 2000 anywhere; 78 us with 400 neighbouring
// ids allowed, and 350 us with 1000 or 4000 of them, more than there is room for (32 rows: 10, 22, 33, 87 us).  All logits equal:
// 54 us.  Small vocabularies leave warps without packs: 256 rows of 500 and of 1000 32 and 23 us, of 4000 8 us.
template <typename io_t>
__device__ void select_top(const Part<io_t>& part, const Sums& sums, bool has_nan, int top_k, TopScratch& t) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid < FRWKV_TOP_K_MAX) t.list[tid] = 0;
  if (tid == 0) t.hot_count = t.wide_count = t.above_count = t.equal_count = 0;
  unsigned mine = order_of(sums.top), offer = 0;
  for (int r = 0; r < (top_k + kWarps - 1) / kWarps; ++r) {
    offer = __reduce_max_sync(0xffffffffu, mine);
    const unsigned who = __ballot_sync(0xffffffffu, mine == offer);
    if (lane == __ffs(who) - 1) mine = 0;
  }
  if (lane == 0) t.bars[warp] = offer;
  const bool any_nan = __syncthreads_or(has_nan);
  unsigned bar_order = t.bars[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) bar_order = min(bar_order, t.bars[w]);
  const float bar = value_of(bar_order);
  const auto consider_logit = [&](float x, int id) {
    if (x > bar) {
      const int at = atomicAdd(&t.above_count, 1);
      if (at < kAbove) t.found[at] = rank_key(x, id);
    } else if (x == bar) {
      const int at = atomicAdd(&t.equal_count, 1);
      if (at < kEqual) t.found[kAbove + at] = rank_key(x, id);
    }
  };
  if (!any_nan && sums.top >= bar) {
    t.hot[atomicAdd(&t.hot_count, 1)] = tid | sums.top_batch << 8;
    if (sums.next >= bar) t.wide[atomicAdd(&t.wide_count, 1)] = tid | sums.top_batch << 8;
  }
  __syncthreads();
  if (!any_nan) {
    for (int i = tid; i < part.single_count(); i += kThreads) consider_logit(to_f32(part.row[part.single(i)]), part.single(i));
    const int batches = (part.last - part.first + kBatch * kThreads - 1) / (kBatch * kThreads);
    const int narrow = t.hot_count * kBatch, all = narrow + t.wide_count * batches * kBatch;
    for (int i = tid; i < all; i += kThreads) {
      int entry, batch;
      if (i < narrow) {
        entry = t.hot[i / kBatch];
        batch = entry >> 8;
      } else {
        const int j = (i - narrow) / kBatch;
        entry = t.wide[j / batches];
        batch = j % batches;
        if (batch == entry >> 8) continue;  // among the narrow ones
      }
      const int pack = part.first + (batch * kBatch + i % kBatch) * kThreads + (entry & 0xff);
      if (pack >= part.last) continue;
      Pack<io_t> v;
      v.load(part.row + part.pack_id(pack));
#pragma unroll
      for (int j = 0; j < Pack<io_t>::kCount / 2; ++j) {
        const float2 x = v.pair(j);
        if (fmaxf(x.x, x.y) >= bar) {
          consider_logit(x.x, part.pack_id(pack) + 2 * j);
          consider_logit(x.y, part.pack_id(pack) + 2 * j + 1);
        }
      }
    }
  }
  __syncthreads();
  const int above = t.above_count, equal = t.equal_count;
  if (any_nan || above > kAbove) {
    // one pass for each of the top_k, below the one before
    unsigned long long below = ~0ull;
    for (int r = 0; r < top_k; ++r) {
      unsigned long long best = 0;
      const auto consider = [&](float x, int id) {
        const unsigned long long key = rank_key(x, id);
        if (key < below && key > best) best = key;
      };
      for (int i = tid; i < part.single_count(); i += kThreads) consider(to_f32(part.row[part.single(i)]), part.single(i));
      for (int pack = part.first + tid; pack < part.last; pack += kThreads) {
        Pack<io_t> v;
        v.load(part.row + part.pack_id(pack));
#pragma unroll
        for (int j = 0; j < Pack<io_t>::kCount / 2; ++j) {
          const float2 x = v.pair(j);
          consider(x.x, part.pack_id(pack) + 2 * j);
          consider(x.y, part.pack_id(pack) + 2 * j + 1);
        }
      }
#pragma unroll
      for (int m = 16; m > 0; m >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, m));
      if (lane == 0) t.warp_best[warp] = best;
      __syncthreads();
      best = t.warp_best[0];
      for (int w = 1; w < kWarps; ++w) best = max(best, t.warp_best[w]);
      if (tid == 0) t.list[r] = best;
      if (best == 0) break;  // the part holds fewer than top_k
      below = best;
      __syncthreads();
    }
    __syncthreads();
    return;
  }
  const bool collected = equal <= kEqual;
  const int total = above + (collected ? equal : 0);
  const auto found = [&](int i) { return t.found[i < above ? i : kAbove + i - above]; };
  for (int i = tid; i < total; i += kThreads) {
    const unsigned long long key = found(i);
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < total; ++j) rank += found(j) > key;
    if (rank < top_k) t.list[rank] = key;
  }
  if (!collected) {
    // the lowest ids among the logits equal to the bar: 256 packs after 256 packs until there are enough.  The singles
    // before the first pack come first, those behind the last pack last.
    int have = above;
    const auto take = [&](const float (&x)[Pack<io_t>::kCount], int id, int n) {
      int mine_count = 0;
#pragma unroll
      for (int j = 0; j < Pack<io_t>::kCount; ++j) mine_count += j < n && x[j] == bar;
      int before = mine_count;
#pragma unroll
      for (int m = 1; m < 32; m <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, before, m);
        if (lane >= m) before += other;
      }
      if (lane == 31) t.warp_count[warp] = before;
      __syncthreads();
      int at = have + before - mine_count;
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) at += t.warp_count[w];
        have += t.warp_count[w];
      }
#pragma unroll
      for (int j = 0; j < Pack<io_t>::kCount; ++j)
        if (j < n && x[j] == bar) {
          if (at < top_k) t.list[at] = rank_key(bar, id + j);
          ++at;
        }
      __syncthreads();
    };
    float x[Pack<io_t>::kCount];
    const int lead = part.singles ? part.lead : 0;
    if (lead > 0) {
      x[0] = tid < lead ? to_f32(part.row[tid]) : 0.f;
      take(x, tid, tid < lead ? 1 : 0);
    }
    for (int base = part.first; base < part.last && have < top_k; base += kThreads) {
      Pack<io_t> v;
      v.fill_lowest();
      const int pack = base + tid;
      if (pack < part.last) v.load(part.row + part.pack_id(pack));
#pragma unroll
      for (int j = 0; j < Pack<io_t>::kCount / 2; ++j) {
        x[2 * j] = v.pair(j).x;
        x[2 * j + 1] = v.pair(j).y;
      }
      take(x, part.pack_id(pack), pack < part.last ? Pack<io_t>::kCount : 0);
    }
    const int rest = part.singles ? part.vocab - part.tail() : 0;
    if (rest > 0 && have < top_k) {
      x[0] = tid < rest ? to_f32(part.row[part.tail() + tid]) : 0.f;
      take(x, part.tail() + tid, tid < rest ? 1 : 0);
    }
  }
  __syncthreads();
}

// One row per CTA, or per cluster of CTAs that take equal parts of it (few rows: a row alone cannot fill the GPU).
// Per thread: kBatch 16-byte loads in flight; the sums are rescaled only when a batch raises the running maximum.
template <typename io_t, bool TOP>
__global__ void __launch_bounds__(kThreads, 6)
token_logprobs_kernel(const Rows p, int top_k, float* __restrict__ logprobs, float* __restrict__ entropy,
                      float* __restrict__ stats, int64_t* __restrict__ top_ids, float* __restrict__ top_logprobs) {
  __shared__ Total warp_total[kWarps];
  __shared__ Total cta_total;
  __shared__ std::conditional_t<TOP, TopScratch, char> top_scratch[1];
  const cg::cluster_group cluster = cg::this_cluster();
  const int parts = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const long long row = blockIdx.x / static_cast<unsigned>(parts);
  const int tid = threadIdx.x;
  const long long id = row_id(p, row);
  if (id == p.ignore_index) {  // the whole cluster leaves
    if (rank != 0) return;
    if (tid == 0) {
      logprobs[row] = entropy[row] = 0.f;
      stats[2 * row] = stats[2 * row + 1] = 0.f;
    }
    if (TOP && tid < top_k) {
      top_ids[row * top_k + tid] = -1;
      top_logprobs[row * top_k + tid] = -INFINITY;
    }
    return;
  }
  Part<io_t> part;
  part.row = row_start<io_t>(p, row);
  part.vocab = p.vocab;
  const int misaligned = static_cast<int>(reinterpret_cast<uintptr_t>(part.row) & 15) / static_cast<int>(sizeof(io_t));
  part.lead = misaligned == 0 ? 0 : min(p.vocab, Pack<io_t>::kCount - misaligned);
  part.packs = (p.vocab - part.lead) / Pack<io_t>::kCount;
  const int share = (part.packs + parts - 1) / parts;
  part.first = min(part.packs, rank * share);
  part.last = min(part.packs, part.first + share);
  part.singles = rank == 0;
  const bool known = id >= 0 && id < p.vocab;
  const float given = rank == 0 && tid == 0 && known ? to_f32(part.row[id]) : 0.f;

  const float k = p.inv_temperature * kLog2e;
  Sums sums;
  sums.clear();
  int batch = 0;
  for (int pack = part.first + tid; pack < part.last; pack += kBatch * kThreads) {
    Pack<io_t> v[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      if (pack + b * kThreads < part.last) v[b].load(part.row + part.pack_id(pack + b * kThreads));
      else v[b].fill_lowest();
    }
    sums.template add<io_t, TOP>(v, batch++, k);
  }
  for (int i = tid; i < part.single_count(); i += kThreads) sums.add(to_f32(part.row[part.single(i)]), k);

  // thread, warp, CTA, cluster: always in the same order
  const Total mine{sums.m, sums.s.x + sums.s.y, sums.w.x + sums.w.y};
  const Total warp_sum = join_lanes(sums.top, mine, k);
  if ((tid & 31) == 0) warp_total[tid >> 5] = warp_sum;
  if constexpr (TOP) select_top(part, sums, mine.s != mine.s, top_k, top_scratch[0]);
  else __syncthreads();
  if (parts == 1 && tid >= 32) return;
  const Total nothing{-INFINITY, 0.f, 0.f};
  Total all = nothing;
  if (tid < 32) {
    all = tid < kWarps ? warp_total[tid] : nothing;
    all = join_lanes(all.m, all, k);
  }
  if (parts > 1) {
    if (tid == 0) cta_total = all;
    cluster.sync();
    if (rank == 0) {
      if (tid < 32) {
        all = tid < parts ? *cluster.map_shared_rank(&cta_total, tid) : nothing;
        all = join_lanes(all.m, all, k);
      }
      if constexpr (TOP) {
        // the parts' lists, joined by counting
        const int n = parts * top_k;
        for (int i = tid; i < n; i += kThreads)
          top_scratch[0].found[i] = cluster.map_shared_rank(top_scratch[0].list, i / top_k)[i % top_k];
        __syncthreads();
        for (int i = tid; i < n; i += kThreads) {
          const unsigned long long key = top_scratch[0].found[i];
          int place = 0;
#pragma unroll 8
          for (int j = 0; j < n; ++j) place += top_scratch[0].found[j] > key;
          if (key != 0 && place < top_k) top_scratch[0].list[place] = key;
        }
        __syncthreads();
      }
    }
    cluster.sync();  // rank 0 has read the others' shared memory
    if (rank != 0 || tid >= 32) return;
  }
  // a row of -inf alone has no maximum and no sum; NaN shows in the sum
  const bool empty = all.m == -INFINITY && all.s == 0.f;
  const float log_s = empty ? 0.f : logf(all.s);
  const auto logprob_of = [&](float x) {
    float z = (x - all.m) * p.inv_temperature;
    // the type's lowest value far below the largest logit: a difference that only a temperature brings back into fp32's range
    if (z == -INFINITY && x != -INFINITY) z = (0.5f * x - 0.5f * all.m) * p.inv_temperature * 2.0f;
    return empty ? -INFINITY : z - log_s;
  };
  if (tid == 0) {
    logprobs[row] = known ? logprob_of(given) : __int_as_float(0x7fffffff);
    entropy[row] = empty ? 0.f : log_s - all.w / all.s * 0.6931471805599453f;
    stats[2 * row] = all.m;
    stats[2 * row + 1] = all.s;
  }
  if constexpr (TOP) {
    if (tid < top_k) {
      const unsigned long long key = top_scratch[0].list[tid];
      top_ids[row * top_k + tid] = key_id(key);
      top_logprobs[row * top_k + tid] = logprob_of(value_of(static_cast<unsigned>(key >> 32)));
    }
  }
}

template <typename io_t> __device__ __forceinline__ unsigned pack_two(float x, float y) {
  if constexpr (std::is_same_v<io_t, __nv_bfloat16>) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const unsigned*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(x, y);
    return *reinterpret_cast<const unsigned*>(&v);
  }
}

// dx_j = e_j (c1 z_j + c0) off the given token, with c1 = -b / (S T), c0 = -(a + b (entropy - log S)) / (S T).
// A CTA takes kBatch * kThreads packs of a row; where the row and its gradient differ in alignment it goes element by
// element (rows of an odd vocabulary cut out of a larger tensor).
template <typename io_t>
__global__ void __launch_bounds__(kThreads)
token_logprobs_backward_kernel(const Rows p, int segments, const float* __restrict__ stats, const float* __restrict__ entropy,
                               const float* __restrict__ dlogprobs, const float* __restrict__ dentropy,
                               io_t* __restrict__ dlogits) {
  constexpr int kCount = Pack<io_t>::kCount;
  const unsigned row_index = blockIdx.x / static_cast<unsigned>(segments);
  const long long row = row_index;
  const int segment = static_cast<int>(blockIdx.x - row_index * segments), tid = threadIdx.x;
  const long long id = row_id(p, row);
  const io_t* x = row_start<io_t>(p, row);
  io_t* out = dlogits + row * p.vocab;
  const float m = stats[2 * row], s = stats[2 * row + 1];
  const bool live = id != p.ignore_index, known = id >= 0 && id < p.vocab;
  const bool zero = !live || (known && m == -INFINITY && s == 0.f);
  const float a = zero ? 0.f : !known ? __int_as_float(0x7fffffff) : dlogprobs != nullptr ? dlogprobs[row] : 0.f;
  const float b = zero || dentropy == nullptr ? 0.f : dentropy[row];
  const float k = p.inv_temperature * kLog2e;
  const float scale = -p.inv_temperature / s;
  const float c1 = b * 0.6931471805599453f * scale, c0 = (a + b * (entropy[row] - logf(s))) * scale;
  const float at_id = a * p.inv_temperature;
  const auto one = [&](float v, long long j) {
    const float z = max_keep_nan((v - m) * k, kLowest);
    const float g = exp2_fast(z) * fmaf(c1, z, c0);
    return j == id ? g + at_id : g;
  };
  const unsigned phase = static_cast<unsigned>(reinterpret_cast<uintptr_t>(x) & 15);
  if (phase != static_cast<unsigned>(reinterpret_cast<uintptr_t>(out) & 15)) {
    const long long span = kBatch * kThreads * kCount, last = min(static_cast<long long>(p.vocab), (segment + 1) * span);
    for (long long j = segment * span + tid; j < last; j += kThreads) out[j] = from_f32<io_t>(zero ? 0.f : one(to_f32(x[j]), j));
    return;
  }
  const int misaligned = static_cast<int>(phase) / static_cast<int>(sizeof(io_t));
  const int lead = misaligned == 0 ? 0 : min(p.vocab, kCount - misaligned);
  const int packs = (p.vocab - lead) / kCount;
  if (segment == 0) {
    const int tail = lead + packs * kCount;
    for (int i = tid; i < lead + (p.vocab - tail); i += kThreads) {
      const int j = i < lead ? i : tail + i - lead;
      out[j] = from_f32<io_t>(zero ? 0.f : one(to_f32(x[j]), j));
    }
  }
  const int first = segment * kBatch * kThreads + tid;
  x += lead + static_cast<long long>(first) * kCount;
  out += lead + static_cast<long long>(first) * kCount;
  // the given token's place, counted from this thread's first logit (far away where it is not among the row's packs)
  const long long from_first = id - lead - static_cast<long long>(first) * kCount;
  const int hit = from_first >= 0 && from_first < kBatch * kThreads * kCount ? static_cast<int>(from_first) : -1;
  const int left = packs - first;
  Pack<io_t> v[kBatch];
#pragma unroll
  for (int i = 0; i < kBatch; ++i) {
    if (!zero && i * kThreads < left) v[i].load(x + i * kThreads * kCount);
    else v[i].raw = make_uint4(0, 0, 0, 0);
  }
  const float2 minus_m = make_float2(-m, -m), k2 = make_float2(k, k), c1_2 = make_float2(c1, c1), c0_2 = make_float2(c0, c0);
#pragma unroll
  for (int i = 0; i < kBatch; ++i) {
    if (i * kThreads >= left) break;
    unsigned words[4] = {0, 0, 0, 0};
    if (!zero) {
      float g[kCount];
#pragma unroll
      for (int j = 0; j < kCount / 2; ++j) {
        float2 z = __fmul2_rn(__fadd2_rn(v[i].pair(j), minus_m), k2);
        z = make_float2(max_keep_nan(z.x, kLowest), max_keep_nan(z.y, kLowest));
        const float2 y = __fmul2_rn(make_float2(exp2_fast(z.x), exp2_fast(z.y)), __ffma2_rn(c1_2, z, c0_2));
        g[2 * j] = y.x;
        g[2 * j + 1] = y.y;
      }
      const unsigned place = static_cast<unsigned>(hit - i * kThreads * kCount);
      if (place < kCount) {
#pragma unroll
        for (int j = 0; j < kCount; ++j) g[j] = j == static_cast<int>(place) ? g[j] + at_id : g[j];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(io_t) == 4) words[j] = __float_as_uint(g[j]);
        else words[j] = pack_two<io_t>(g[2 * j], g[2 * j + 1]);
      }
    }
    __stcs(reinterpret_cast<uint4*>(out + i * kThreads * kCount), make_uint4(words[0], words[1], words[2], words[3]));
  }
}

int check_rows(const char* what, const void* logits, long long outer, long long inner, const void* ids, int vocab,
               int io_dtype, float temperature) {
  if (!logits || !ids) return fail(FRWKV_ERR_ARGUMENT, "%s: logits and ids must be non-null", what);
  if (outer <= 0 || inner <= 0 || outer > 0x7fffffffLL / inner)
    return fail(FRWKV_ERR_ARGUMENT, "%s: the row count must be positive and fit in int32", what);
  if (vocab <= 0) return fail(FRWKV_ERR_ARGUMENT, "%s: vocab must be positive", what);
  if (io_dtype < FRWKV_IO_BF16 || io_dtype > FRWKV_IO_FP32) return fail(FRWKV_ERR_UNSUPPORTED, "%s: unknown dtype", what);
  // so that its reciprocal, times log2 e and times gradients, neither overflows (0 * inf) nor is subnormal
  if (!(temperature >= FRWKV_TEMPERATURE_MIN && temperature <= FRWKV_TEMPERATURE_MAX))
    return fail(FRWKV_ERR_ARGUMENT, "%s: temperature must be in 1e-30..1e30", what);
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
  const auto launch = [&](auto kernel, int element) {
    // The largest power of two of CTAs a row that leaves each of them a full batch of loads and does not start more CTAs
    // than about three per SM.
    int parts = 1;
    while (parts < kMaxCluster && p.rows * parts * 2 <= kClusterCtas &&
           static_cast<long long>(vocab) * element >= static_cast<long long>(parts) * 2 * kClusterBytes)
      parts *= 2;
    cudaLaunchAttribute cluster;
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = static_cast<unsigned>(parts);
    cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<unsigned>(p.rows * parts));
    config.blockDim = dim3(kThreads);
    config.stream = static_cast<cudaStream_t>(stream);
    config.attrs = &cluster;
    config.numAttrs = parts > 1 ? 1 : 0;
    cudaLaunchKernelEx(&config, kernel, p, top_k, logprobs, entropy, stats, top_ids, top_logprobs);
  };
  if (io_dtype == FRWKV_IO_BF16) {
    if (top_k > 0) launch(token_logprobs_kernel<__nv_bfloat16, true>, 2);
    else launch(token_logprobs_kernel<__nv_bfloat16, false>, 2);
  } else if (io_dtype == FRWKV_IO_FP16) {
    if (top_k > 0) launch(token_logprobs_kernel<__half, true>, 2);
    else launch(token_logprobs_kernel<__half, false>, 2);
  } else {
    if (top_k > 0) launch(token_logprobs_kernel<float, true>, 4);
    else launch(token_logprobs_kernel<float, false>, 4);
  }
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
  const int element = io_dtype == FRWKV_IO_FP32 ? 4 : 2;
  const long long per_cta = static_cast<long long>(kBatch) * kThreads * (16 / element);
  const int segments = static_cast<int>((vocab + per_cta - 1) / per_cta);
  if (p.rows * segments > 0x7fffffffLL) return fail(FRWKV_ERR_ARGUMENT, "token_logprobs backward: too many rows");
  const unsigned grid = static_cast<unsigned>(p.rows * segments);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (io_dtype == FRWKV_IO_BF16)
    token_logprobs_backward_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(
        p, segments, stats, entropy, dlogprobs, dentropy, static_cast<__nv_bfloat16*>(dlogits));
  else if (io_dtype == FRWKV_IO_FP16)
    token_logprobs_backward_kernel<__half><<<grid, kThreads, 0, s>>>(p, segments, stats, entropy, dlogprobs, dentropy,
                                                                     static_cast<__half*>(dlogits));
  else
    token_logprobs_backward_kernel<float><<<grid, kThreads, 0, s>>>(p, segments, stats, entropy, dlogprobs, dentropy,
                                                                    static_cast<float*>(dlogits));
  return check_launch("token_logprobs_backward_kernel");
}
