// Arithmetic, row metadata and the chain between tiles that the gated scan's kernels share.
//
//   h_t = rho_t * h_{t-1} + i_t * x_t,   rho = exp(-s), s = exp(-1/2) * sigmoid(logit + bias)   or rho itself.
// From logits the kernels work with rho - 1 and write rho * h as h + (rho - 1) * h: a slow channel has 1 - rho of 1e-4
// and less, and rho rounded to fp32 would then be off by 2^-25 / (1 - rho) of the decay it stands for, at every token
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

// ---- the channels of a lane: 8 bytes of a token row, in pairs for packed fp32 arithmetic

template <int V> struct Lanes {
  float2 v[V / 2];

  static __device__ __forceinline__ Lanes all(float x) {
    Lanes r;
#pragma unroll
    for (int i = 0; i < V / 2; ++i) r.v[i] = make_float2(x, x);
    return r;
  }
};
template <int V> __device__ __forceinline__ Lanes<V> fma(const Lanes<V>& a, const Lanes<V>& b, const Lanes<V>& c) {
  Lanes<V> r;
#pragma unroll
  for (int i = 0; i < V / 2; ++i) r.v[i] = __ffma2_rn(a.v[i], b.v[i], c.v[i]);
  return r;
}
template <int V> __device__ __forceinline__ Lanes<V> mul(const Lanes<V>& a, const Lanes<V>& b) {
  Lanes<V> r;
#pragma unroll
  for (int i = 0; i < V / 2; ++i) r.v[i] = __fmul2_rn(a.v[i], b.v[i]);
  return r;
}
template <int V> __device__ __forceinline__ Lanes<V> add(const Lanes<V>& a, const Lanes<V>& b) {
  Lanes<V> r;
#pragma unroll
  for (int i = 0; i < V / 2; ++i) r.v[i] = __fadd2_rn(a.v[i], b.v[i]);
  return r;
}
template <int V> __device__ __forceinline__ Lanes<V> minus(const Lanes<V>& a, const Lanes<V>& b) {  // a - b
  return fma(b, Lanes<V>::all(-1.0f), a);
}
template <int V, typename F> __device__ __forceinline__ Lanes<V> each(F f, const Lanes<V>& a) {
  Lanes<V> r;
#pragma unroll
  for (int i = 0; i < V / 2; ++i) r.v[i] = make_float2(f(a.v[i].x), f(a.v[i].y));
  return r;
}

// 8 bytes of a token row as floats, and back.
template <typename io_t> __device__ __forceinline__ Lanes<8 / sizeof(io_t)> unpack(uint2 w) {
  Lanes<8 / sizeof(io_t)> r;
  if constexpr (sizeof(io_t) == 4) {
    r.v[0] = make_float2(__uint_as_float(w.x), __uint_as_float(w.y));
  } else if constexpr (std::is_same_v<io_t, __nv_bfloat16>) {
    r.v[0] = make_float2(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u));
    r.v[1] = make_float2(__uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
  } else {
    r.v[0] = __half22float2(*reinterpret_cast<const __half2*>(&w.x));
    r.v[1] = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
  }
  return r;
}
template <typename io_t> __device__ __forceinline__ unsigned pack_pair(float2 v) {
  if constexpr (std::is_same_v<io_t, __nv_bfloat16>) {
    const __nv_bfloat162 r = __floats2bfloat162_rn(v.x, v.y);
    return *reinterpret_cast<const unsigned*>(&r);
  } else {
    const __half2 r = __floats2half2_rn(v.x, v.y);
    return *reinterpret_cast<const unsigned*>(&r);
  }
}
template <typename io_t> __device__ __forceinline__ uint2 pack(const Lanes<8 / sizeof(io_t)>& a) {
  if constexpr (sizeof(io_t) == 4) return make_uint2(__float_as_uint(a.v[0].x), __float_as_uint(a.v[0].y));
  else return make_uint2(pack_pair<io_t>(a.v[0]), pack_pair<io_t>(a.v[1]));
}

// How much of a lane's 8 bytes one access may move: 8, 4 or (16-bit types at any alignment) 2 bytes.  `count` is how many
// of the lane's elements exist.
template <typename io_t, int GRANULE> struct Access {
  static constexpr int V = 8 / sizeof(io_t), kElements = GRANULE / sizeof(io_t);

  // One token's 8 bytes into shared memory, asynchronously where the hardware can (4 and 8 bytes), zeros for what does
  // not exist.  A lane reads back only what it copied itself.
  static __device__ __forceinline__ void stage(uint2* to, const io_t* from, int count) {
    if constexpr (GRANULE == 2) {
      alignas(8) io_t w[V];
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] = i < count ? from[i] : from_f32<io_t>(0.0f);
      *to = *reinterpret_cast<const uint2*>(w);
    } else {
      const unsigned at = static_cast<unsigned>(__cvta_generic_to_shared(to));
#pragma unroll
      for (int i = 0; i < 8 / GRANULE; ++i) {
        const bool in = i * kElements < count;
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;"
                     : : "r"(at + i * GRANULE), "l"(in ? from + i * kElements : from), "n"(GRANULE), "r"(in ? GRANULE : 0) : "memory");
      }
    }
  }
  static __device__ __forceinline__ void store(io_t* to, const Lanes<V>& a, int count) {
    const uint2 w = pack<io_t>(a);
    if constexpr (GRANULE == 8) {
      if (count > 0) __stcs(reinterpret_cast<uint2*>(to), w);
    } else if constexpr (GRANULE == 4) {
      if (count > 0) __stcs(reinterpret_cast<unsigned*>(to), w.x);
      if (count > kElements) __stcs(reinterpret_cast<unsigned*>(to) + 1, w.y);
    } else {
      const io_t* e = reinterpret_cast<const io_t*>(&w);
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i < count) to[i] = e[i];
    }
  }
};

// A lane's fp32 states.
template <int V> __device__ __forceinline__ Lanes<V> load_states(const float* from, int count) {
  Lanes<V> r;
#pragma unroll
  for (int i = 0; i < V / 2; ++i) r.v[i] = make_float2(2 * i < count ? from[2 * i] : 0.0f, 2 * i + 1 < count ? from[2 * i + 1] : 0.0f);
  return r;
}
template <int V> __device__ __forceinline__ void store_states(float* to, const Lanes<V>& a, int count) {
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    if (2 * i < count) to[2 * i] = a.v[i].x;
    if (2 * i + 1 < count) to[2 * i + 1] = a.v[i].y;
  }
}

// ---- gate

// What a token does to the state.  LOGITS keeps rho - 1, otherwise rho is kept (see the top of the file).
template <bool LOGITS, bool COMPLEMENT, int V> struct Decay {
  using L = Lanes<V>;

  // sigmoid(raw + bias) from bias * -log2 e, with the SFU's approximations of exp2 and the reciprocal (2^-22 each)
  static __device__ __forceinline__ L sigmoid(const L& raw, const L& bias) {
    const L e = each([](float v) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; },
                     fma(raw, L::all(-kLog2e), bias));
    return each([](float v) { float r; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; },
                add(e, L::all(1.0f)));
  }
  // exp(-c g) - 1, c = exp(-1/2), 0 <= g <= 1, as g times a polynomial of degree 5: the Chebyshev interpolant of
  // (exp(-c g) - 1) / g on [0, 1], whose relative error is 5e-9 (8e-8 with fp32 arithmetic)
  static __device__ __forceinline__ L keep_gate(const L& g) {
    L q = fma(g, L::all(5.351052459445782e-05f), L::all(-6.67280750349164e-04f));
    q = fma(g, q, L::all(5.630488507449627e-03f));
    q = fma(g, q, L::all(-3.7186399102211e-02f));
    q = fma(g, q, L::all(1.8393956124782562e-01f));
    q = fma(g, q, L::all(-6.065306663513184e-01f));
    return mul(g, q);
  }
  static __device__ __forceinline__ L keep(const L& raw, const L& bias) {
    if constexpr (LOGITS) return keep_gate(sigmoid(raw, bias));
    else return raw;
  }
  // rho * h + i * x.  rho h + (1 - rho) x is h + (rho - 1) (h - x), whose difference costs no precision as it is scaled
  // down; x + rho (h - x) would round a slow state to steps of x.
  static __device__ __forceinline__ L step(const L& kept, const L& h, const L& x) {
    if constexpr (COMPLEMENT && LOGITS) return fma(kept, minus(h, x), h);
    else if constexpr (COMPLEMENT) return fma(kept, h, mul(minus(L::all(1.0f), kept), x));
    else if constexpr (LOGITS) return add(h, fma(kept, h, x));
    else return fma(kept, h, x);
  }
  // rho * h
  static __device__ __forceinline__ L fade(const L& kept, const L& h) {
    if constexpr (LOGITS) return fma(kept, h, h);
    else return mul(kept, h);
  }
  // d step / d x * g
  static __device__ __forceinline__ L input_grad(const L& kept, const L& g) {
    if constexpr (!COMPLEMENT) return g;
    else if constexpr (LOGITS) return mul(mul(kept, L::all(-1.0f)), g);
    else return fma(kept, mul(g, L::all(-1.0f)), g);
  }
  // d rho / d raw from g = sigmoid(raw): -c g (1 - g) rho
  static __device__ __forceinline__ L slope(const L& g, const L& kept) {
    const L rest = mul(minus(L::all(1.0f), g), add(kept, L::all(1.0f)));
    return mul(mul(g, L::all(-kRate)), rest);
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
    const int into = row - m.seq * p.seq_len;  // of the first row's sequence
    if (p.seq_len > S) {  // at most one bound, behind the first row
      bounds = (into == 0 ? 1u : 0u) | (p.seq_len - into <= S ? 1u << (p.seq_len - into) : 0u);
    } else {
      bounds = __ballot_sync(0xffffffffu, lane <= S && (into + lane) % p.seq_len == 0);
    }
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
//
// Every published word says by itself whether it is there: the call first fills the space with kEmpty, no value is ever
// stored with those bits (a NaN is stored as another one), and a reader takes a word once it differs.  So one trip to L2
// brings flag and value together, and nothing has to be fenced.

constexpr int kGroup = 16;
constexpr unsigned kEmpty = 0xffffffffu;  // of the filled space
constexpr unsigned kCut = 0x7fc0c0deu;    // A of a tile in which a sequence starts (backward: ends)
constexpr int kSpinLimit = 1 << 20;       // about a second of polling; then the state becomes NaN and the kernel ends

// Any value but kEmpty and kCut: a NaN other than the marks becomes the plain one.
__device__ __forceinline__ float storable(float x) { return x == x ? x : __int_as_float(0x7fffffff); }

struct ChainSpace {
  int* ticket;    // kEmpty at first: the first ticket is 0 after adding 1 to what was there
  float* maps;    // [blocks][tiles][A or B][lane][V]
  float* states;  // [blocks][groups][lane][V]
  int tiles, groups, blocks;  // time tiles, groups of them, channel blocks
};

template <int V> struct alignas(4 * V) Map {
  Lanes<V> a, b;

  static __device__ __forceinline__ Map identity() { return Map{Lanes<V>::all(1.0f), Lanes<V>::all(0.0f)}; }
  __device__ __forceinline__ Lanes<V> apply(const Lanes<V>& h) const { return fma(a, h, b); }
  // this map, then `next`
  __device__ __forceinline__ void then(const Map& next) {
    b = fma(next.a, b, next.b);
    a = mul(next.a, a);
  }
};

template <int V> struct Chain {
  using L = Lanes<V>;

  static __device__ __forceinline__ void put_raw(float* to, const L& x) {
    if constexpr (V == 4)
      asm volatile("st.relaxed.gpu.global.v4.f32 [%0], {%1, %2, %3, %4};"
                   : : "l"(to), "f"(x.v[0].x), "f"(x.v[0].y), "f"(x.v[1].x), "f"(x.v[1].y) : "memory");
    else
      asm volatile("st.relaxed.gpu.global.v2.f32 [%0], {%1, %2};" : : "l"(to), "f"(x.v[0].x), "f"(x.v[0].y) : "memory");
  }
  static __device__ __forceinline__ void put(float* to, const L& x) { put_raw(to, each([](float v) { return storable(v); }, x)); }
  static __device__ __forceinline__ L look(const float* from) {
    L x;
    if constexpr (V == 4)
      asm volatile("ld.relaxed.gpu.global.v4.f32 {%0, %1, %2, %3}, [%4];"
                   : "=f"(x.v[0].x), "=f"(x.v[0].y), "=f"(x.v[1].x), "=f"(x.v[1].y) : "l"(from) : "memory");
    else
      asm volatile("ld.relaxed.gpu.global.v2.f32 {%0, %1}, [%2];" : "=f"(x.v[0].x), "=f"(x.v[0].y) : "l"(from) : "memory");
    return x;
  }
  static __device__ __forceinline__ bool there(const L& x) {
    bool yes = true;
#pragma unroll
    for (int i = 0; i < V / 2; ++i) yes = yes && __float_as_uint(x.v[i].x) != kEmpty && __float_as_uint(x.v[i].y) != kEmpty;
    return yes;
  }
  static __device__ __forceinline__ L wait(const float* from, L x) {  // x: what an earlier look brought
    for (int i = 0; i < kSpinLimit && !there(x); ++i) x = look(from);
    return there(x) ? x : L::all(__int_as_float(0x7fffffff));
  }
  static __device__ __forceinline__ float* map_at(const ChainSpace& c, int block, int index) {
    return c.maps + ((static_cast<long long>(block) * c.tiles + index) * 64 + (threadIdx.x & 31)) * V;
  }
  static __device__ __forceinline__ float* state_at(const ChainSpace& c, int block, int group) {
    return c.states + ((static_cast<long long>(block) * c.groups + group) * 32 + (threadIdx.x & 31)) * V;
  }
  // One warp publishes its tile's map; index counts tiles in the chain's direction.
  static __device__ __forceinline__ void publish(const ChainSpace& c, int block, int index, const Map<V>& m, bool cut) {
    float* to = map_at(c, block, index);
    if (cut) put_raw(to, L::all(__uint_as_float(kCut)));
    else put(to, m.a);
    put(to + 32 * V, m.b);
  }
  static __device__ __forceinline__ bool is_cut(const L& a) { return __float_as_uint(a.v[0].x) == kCut; }  // all lanes agree
  // The state before a tile, by one warp: the maps of the n < kGroup tiles before it in its group behind the state that
  // the group before left.  All maps are asked for in batches before the first is waited for.
  static __device__ __forceinline__ L state_before(const ChainSpace& c, int block, int group, int n) {
    L state = L::all(0.0f);
    if (group > 0) state = look(state_at(c, block, group - 1));
    Map<V> all = Map<V>::identity();
    bool cut = false;
    constexpr int kBatch = 8;
    for (int base = 0; base < n; base += kBatch) {
      const float* from = map_at(c, block, group * kGroup + base);
      Map<V> m[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const float* at = from + (base + i < n ? i : 0) * 64 * V;
        m[i].a = look(at);
        m[i].b = look(at + 32 * V);
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (base + i >= n) break;
        m[i].a = wait(from + i * 64 * V, m[i].a);
        m[i].b = wait(from + i * 64 * V + 32 * V, m[i].b);
        if (is_cut(m[i].a)) {
          all.b = m[i].b;
          cut = true;
        } else {
          all.then(m[i]);
        }
      }
    }
    if (cut) return all.b;
    if (group == 0) return L::all(__int_as_float(0x7fffffff));  // no sequence starts at row 0: not valid
    return all.apply(wait(state_at(c, block, group - 1), state));
  }
};

}  // namespace frwkv
