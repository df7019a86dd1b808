// Arithmetic, row metadata and the chain between tiles that the gated scan's kernels share.
//
//   h_t = rho_t * h_{t-1} + i_t * x_t,   rho = exp(-s), s = exp(-1/2) * sigmoid(logit + bias)   or rho itself.
// From logits the kernels work with delta = 1 - rho and write rho * h as h - delta * h: a slow channel has delta of
// 1e-4 and less, and rho rounded to fp32 would then be off by 2^-25 / delta of the decay it stands for, at every token
// with the same sign.  A retention that the caller gives is used as it is (1 - rho loses a small rho instead).
#pragma once

#include "../../common.cuh"

#include <type_traits>

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

struct GatedScanGrads {
  const void* dy;
  const float* dfinal;
  void *dx, *ddecay;
  float* dinitial;
};

// ---- V channels of a lane: one float, or two in packed fp32 arithmetic

template <int V> struct Lanes;
template <> struct Lanes<1> {
  using type = float;
  static __device__ __forceinline__ float all(float x) { return x; }
  static __device__ __forceinline__ float fma(float a, float b, float c) { return fmaf(a, b, c); }
  static __device__ __forceinline__ float mul(float a, float b) { return a * b; }
  static __device__ __forceinline__ float add(float a, float b) { return a + b; }
  template <typename F> static __device__ __forceinline__ float map(F f, float a) { return f(a); }
};
template <> struct Lanes<2> {
  using type = float2;
  static __device__ __forceinline__ float2 all(float x) { return make_float2(x, x); }
  static __device__ __forceinline__ float2 fma(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
  static __device__ __forceinline__ float2 mul(float2 a, float2 b) { return __fmul2_rn(a, b); }
  static __device__ __forceinline__ float2 add(float2 a, float2 b) { return __fadd2_rn(a, b); }
  template <typename F> static __device__ __forceinline__ float2 map(F f, float2 a) { return make_float2(f(a.x), f(a.y)); }
};

// ---- V elements of a token tensor: one load, one store

template <typename io_t, int V> struct Word {
  using type = std::conditional_t<sizeof(io_t) * V == 2, unsigned short, std::conditional_t<sizeof(io_t) * V == 4, unsigned, uint2>>;
  static __device__ __forceinline__ type load(const io_t* p) {  // read once: not kept in L1
    type w;
    if constexpr (sizeof(type) == 2) asm volatile("ld.global.nc.L1::no_allocate.u16 %0, [%1];" : "=h"(w) : "l"(p));
    else if constexpr (sizeof(type) == 4) asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(w) : "l"(p));
    else asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(w.x), "=r"(w.y) : "l"(p));
    return w;
  }
  static __device__ __forceinline__ type load_plain(const io_t* p) { return *reinterpret_cast<const type*>(p); }
  static __device__ __forceinline__ type zero() {
    if constexpr (sizeof(type) == 8) return make_uint2(0, 0);
    else return 0;
  }
  static __device__ __forceinline__ typename Lanes<V>::type unpack(type w) {
    if constexpr (V == 1) {
      if constexpr (sizeof(io_t) == 4) return __uint_as_float(w);
      else if constexpr (std::is_same_v<io_t, __nv_bfloat16>) return __uint_as_float(static_cast<unsigned>(w) << 16);
      else return __half2float(__ushort_as_half(w));
    } else {
      if constexpr (sizeof(io_t) == 4) return make_float2(__uint_as_float(w.x), __uint_as_float(w.y));
      else if constexpr (std::is_same_v<io_t, __nv_bfloat16>)
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
      else return __half22float2(*reinterpret_cast<const __half2*>(&w));
    }
  }
  static __device__ __forceinline__ void store(io_t* p, typename Lanes<V>::type v) {
    if constexpr (V == 1) {
      *p = from_f32<io_t>(v);
    } else if constexpr (sizeof(io_t) == 4) {
      __stcs(reinterpret_cast<float2*>(p), v);
    } else if constexpr (std::is_same_v<io_t, __nv_bfloat16>) {
      const __nv_bfloat162 r = __floats2bfloat162_rn(v.x, v.y);
      __stcs(reinterpret_cast<unsigned*>(p), *reinterpret_cast<const unsigned*>(&r));
    } else {
      const __half2 r = __floats2half2_rn(v.x, v.y);
      __stcs(reinterpret_cast<unsigned*>(p), *reinterpret_cast<const unsigned*>(&r));
    }
  }
};

// ---- gate

// What a token does to the state.  LOGITS keeps delta = 1 - rho, otherwise rho is kept (see the top of the file).
template <bool LOGITS, int V> struct Decay {
  using L = Lanes<V>;
  using F = typename L::type;

  // The kept form of a raw decay (+ bias).  With SFU approximations of exp2 and the reciprocal (2^-22 each) and the
  // series of 1 - exp(-s), which is a sum of few terms for s <= 0.61: the ninth is below 2^-24 of the result.
  static __device__ __forceinline__ F keep(F raw) {
    if constexpr (!LOGITS) return raw;
    const F s = L::mul(sigmoid(raw), L::all(kRate));
    F d = L::fma(s, L::all(-1.0f / 40320), L::all(1.0f / 5040));
    d = L::fma(s, d, L::all(-1.0f / 720));
    d = L::fma(s, d, L::all(1.0f / 120));
    d = L::fma(s, d, L::all(-1.0f / 24));
    d = L::fma(s, d, L::all(1.0f / 6));
    d = L::fma(s, d, L::all(-0.5f));
    d = L::fma(s, d, L::all(1.0f));
    return L::mul(s, d);
  }
  static __device__ __forceinline__ F sigmoid(F raw) {
    const F e = L::map([](float v) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; },
                       L::mul(raw, L::all(-kLog2e)));
    return L::map([](float v) { float r; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; },
                  L::add(e, L::all(1.0f)));
  }
  static __device__ __forceinline__ F complement(F kept) { return LOGITS ? kept : L::fma(kept, L::all(-1.0f), L::all(1.0f)); }
  static __device__ __forceinline__ F minus_kept(F kept) { return L::mul(kept, L::all(-1.0f)); }
  // rho * h + u
  static __device__ __forceinline__ F step(F kept, F h, F u) {
    if constexpr (LOGITS) return L::add(h, L::fma(L::mul(kept, L::all(-1.0f)), h, u));
    else return L::fma(kept, h, u);
  }
  // rho * h
  static __device__ __forceinline__ F fade(F kept, F h) {
    if constexpr (LOGITS) return L::fma(L::mul(kept, L::all(-1.0f)), h, h);
    else return L::mul(kept, h);
  }
  // d(1 - rho) / d raw
  static __device__ __forceinline__ F slope(F raw, F kept) {
    if constexpr (!LOGITS) return L::all(-1.0f);
    const F g = sigmoid(raw);
    const F rest = L::mul(L::fma(g, L::all(-1.0f), L::all(1.0f)), L::fma(kept, L::all(-1.0f), L::all(1.0f)));
    return L::mul(L::mul(g, L::all(kRate)), rest);
  }
};

// ---- rows and sequences

// The sequences that S consecutive rows of a warp belong to.
struct RowMap {
  int seq;          // of the first row
  unsigned starts;  // bit i: row i is the first of its sequence
  unsigned ends;    // bit i: row i is the last of its sequence

  // sequence of row i
  __device__ __forceinline__ int seq_of(int i) const { return seq + __popc(starts & ((2u << i) - 2u)); }
};

// Rows [row, row + S) of `active`; all lanes of the warp take part.  S < 31.
template <int S> __device__ __forceinline__ RowMap map_rows(const GatedScanParams& p, int row, int active, int n_seq) {
  const int lane = threadIdx.x & 31;
  RowMap m;
  unsigned bounds;  // bit i: a sequence starts at row + i (or the last one ends before it)
  if (p.cu == nullptr) {
    m.seq = row / p.seq_len;
    bounds = __ballot_sync(0xffffffffu, lane <= S && (row + lane) % p.seq_len == 0);
  } else {
    int low = 0, high = n_seq;  // cu[low] <= row < cu[high]
    while (high - low > 1) {
      const int step = (high - low + 31) / 32, at = low + lane * step;
      const int below = __popc(__ballot_sync(0xffffffffu, at < high && p.cu[at] <= row));
      low += (below - 1) * step;
      high = min(low + step, high);
    }
    m.seq = low;
    const int bound = low + lane <= n_seq ? p.cu[low + lane] : -1;
    const bool inside = bound >= row && bound <= row + S;
    bounds = __reduce_or_sync(0xffffffffu, inside ? 1u << (bound - row) : 0u);
  }
  const unsigned live = row + S <= active ? (1u << S) - 1 : row < active ? (1u << (active - row)) - 1 : 0u;
  m.starts = bounds & live;
  m.ends = (bounds >> 1) & live;
  return m;
}

// ---- the chain between tiles
//
// A tile of rows turns the state h before it into A h + B (B alone behind a sequence's start).  Tiles publish (A, B) as
// soon as they have them; the last tile of every kGroup also publishes the state behind it.  A tile joins the published
// maps of the tiles before it in its group and applies them to the state behind the group before: one hop of the serial
// chain covers kGroup tiles.  What is joined, and in which order, depends on the rows alone and never on timing.
// Tiles are handed out in order by a counter, so what a tile waits for is always in work or done.

constexpr int kGroup = 16;
constexpr int kSpinLimit = 1 << 20;  // about a second of polling; then the state becomes NaN and the kernel ends

__device__ __forceinline__ int poll(const int* flag) {
  int v = 0;
  for (int i = 0; i < kSpinLimit; ++i) {
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(flag) : "memory");
    if (v != 0) break;
  }
  return v;
}

__device__ __forceinline__ void raise(int* flag, int value) {
  asm volatile("st.release.gpu.global.u32 [%0], %1;" : : "l"(flag), "r"(value) : "memory");
}

struct ChainSpace {
  int* ticket;
  int* tile_flags;   // [blocks][tiles]: 1 published, 2 published and a sequence starts (backward: ends) inside
  int* group_flags;  // [blocks][groups]
  float* maps;       // [blocks][tiles][lane][A, B]
  float* states;     // [blocks][groups][lane]
  int tiles, groups, blocks;  // time tiles, groups of them, channel blocks
};

template <int V> struct Chain {
  using L = Lanes<V>;
  using F = typename L::type;
  struct alignas(8 * V) Map {
    F a, b;
  };

  // One warp publishes its tile's map; index counts tiles in the chain's direction.
  static __device__ __forceinline__ void publish(const ChainSpace& c, int block, int index, const Map& map, bool cut) {
    const int lane = threadIdx.x & 31;
    const long long at = static_cast<long long>(block) * c.tiles + index;
    reinterpret_cast<Map*>(c.maps)[at * 32 + lane] = map;
    __syncwarp();
    if (lane == 0) raise(c.tile_flags + at, cut ? 2 : 1);
  }
  static __device__ __forceinline__ void publish_state(const ChainSpace& c, int block, int group, F h) {
    const int lane = threadIdx.x & 31;
    const long long at = static_cast<long long>(block) * c.groups + group;
    reinterpret_cast<F*>(c.states)[at * 32 + lane] = h;
    __syncwarp();
    if (lane == 0) raise(c.group_flags + at, 1);
  }
  // The state before tile `index` > 0, by one warp.
  static __device__ __forceinline__ F state_before(const ChainSpace& c, int block, int index) {
    const int lane = threadIdx.x & 31;
    const int first = index / kGroup * kGroup, n = index - first;
    const long long base = static_cast<long long>(block) * c.tiles + first;
    int flag = 1;
    if (lane < n) flag = poll(c.tile_flags + base + lane);
    bool lost = __any_sync(0xffffffffu, flag == 0);
    __syncwarp();
    const unsigned cuts = __ballot_sync(0xffffffffu, lane < n && flag == 2);
    const int from = cuts != 0 ? 31 - __clz(cuts) : 0;
    const Map* maps = reinterpret_cast<const Map*>(c.maps) + base * 32 + lane;
    Map all{L::all(1.0f), L::all(0.0f)};
    for (int i = from; i < n; ++i) {
      Map m;
      if constexpr (V == 2) {
        const float4 raw = __ldcg(reinterpret_cast<const float4*>(maps + i * 32));
        m.a = make_float2(raw.x, raw.y);
        m.b = make_float2(raw.z, raw.w);
      } else {
        const float2 raw = __ldcg(reinterpret_cast<const float2*>(maps + i * 32));
        m.a = raw.x;
        m.b = raw.y;
      }
      if (i == from) {
        all = m;
      } else {
        all.b = L::fma(m.a, all.b, m.b);
        all.a = L::mul(m.a, all.a);
      }
    }
    F h = all.b;
    if (cuts == 0 && first == 0) return L::all(__int_as_float(0x7fffffff));  // no sequence starts at row 0: not valid
    if (cuts == 0) {  // the group before carries on
      const long long at = static_cast<long long>(block) * c.groups + first / kGroup - 1;
      int there = 1;
      if (lane == 0) there = poll(c.group_flags + at);
      lost = __any_sync(0xffffffffu, there == 0) || lost;
      __syncwarp();
      h = L::fma(all.a, __ldcg(reinterpret_cast<const F*>(c.states) + at * 32 + lane), all.b);
    }
    return lost ? L::all(__int_as_float(0x7fffffff)) : h;
  }
};

}  // namespace frwkv
