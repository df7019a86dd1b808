// Arithmetic and memory accesses that the gated scan's kernels share.
//
//   h_t = rho_t * h_{t-1} + i_t * x_t,   rho = exp(-s), s = exp(-1/2) * sigmoid(logit + bias)   or rho itself.
// From logits the kernels work with rho - 1 and write rho * h as h + (rho - 1) * h: a slow channel has 1 - rho of 1e-4
// and less, and rho rounded to fp32 would then be off by 2^-25 / (1 - rho) of the decay it stands for, at every token
// with the same sign.  A retention that the caller gives is used as it is (1 - rho loses a small rho instead).
// (An infinite h becomes NaN in that form, infinity less infinity.  A second way through the rows for it, taken when one shows
// up, made the compiler spill in the first: 64 ragged sequences of 2560 bf16 channels 414 -> 461 us.)
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
  float* boundary;       // training: the state before every kSavedRows-th row of a sequence, see saved_row()
  void* y;
  int n_seq, total, channels, seq_len;
  int longer_than;  // sequences of at most this many tokens are left to the step kernel
};

constexpr int kSavedRows = FRWKV_GATED_SCAN_SAVED_ROWS;

// Where the state before row `at` (a multiple of kSavedRows) of a sequence that begins at row `first` is saved: sequences
// leave room for each other, and total / kSavedRows + n_seq rows hold all of them.
__device__ __forceinline__ long long saved_row(int seq, int first, int at) { return first / kSavedRows + seq + at / kSavedRows; }

struct GatedScanGrads {
  const void* dy;
  const float* dfinal;
  void *dx, *ddecay;
  float* dinitial;
};

// ---- the channels of a lane: 8 bytes of a token row, in pairs for packed fp32 arithmetic

template <int V> struct alignas(4 * V) Lanes {
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

// ---- token rows in shared memory
//
// A warp's rows of one tensor: four lane groups of S rows of 64 bytes each.  ALIGN is what every row's 64 bytes begin at a
// multiple of in global memory: 16, 4, or nothing in particular (0).  With 16 they are copied by 16 bytes, with 4 by 4.
// Otherwise the five 16-byte pieces that a row's 64 bytes touch are copied, as far as they hold bytes of the row or of what
// lies before it in the tensor, and a lane shifts its 8 bytes out of them.  (When it was chosen, 16 x 1024 rows of 1003 fp32
// channels, by 4 bytes and by pieces: forward 57 and 67 us, backward 150 and 106 us; 32 x 1024 rows of 1003 bf16 channels, element
// by element and by pieces: 290 and 88 us, 589 and 146 us.)

constexpr int kLanes = 8, kGroups = 32 / kLanes;  // lanes along the channels (8 bytes each), groups of them along time

template <typename io_t, int ALIGN, int S> struct Rows {
  static constexpr bool ALIGNED = ALIGN >= 4;  // as it lies in shared memory
  static constexpr int V = 8 / sizeof(io_t);
  static constexpr int kPitch = ALIGNED ? 64 : 80;  // bytes of a row
  // of a group, in words of 8 bytes.  Two groups that read their i-th rows at once have to read different banks: groups are an
  // odd multiple of 64 bytes apart, or, without that room, odd groups have their rows swapped in pairs.
  static constexpr int kGroupWords = (S * kPitch + (ALIGNED ? 0 : 64)) / 8;
  static constexpr int kWords = kGroups * kGroupWords;  // of a warp's rows

  // A lane's 8 bytes of the rows of a group; `from` is the global address of its first row's 64 bytes.
  struct Mine {
    const uint2 *even, *odd;  // ALIGNED
    // Otherwise where row i's bytes begin, less i rows: the shift repeats every kPeriod rows.  16-bit types read the words that
    // hold them and shift by the rest.
    static constexpr int kPeriod = ALIGNED ? 1 : 16 / static_cast<int>(sizeof(io_t));
    unsigned at[kPeriod], shift[2];

    __device__ __forceinline__ Lanes<V> operator[](int i) const { return unpack<io_t>(words(i)); }
    __device__ __forceinline__ uint2 words(int i) const {
      if constexpr (ALIGNED) {
        return (i & 1 ? odd : even)[i * kLanes];
      } else {
        unsigned w[3] = {0, 0, 0};
#pragma unroll
        for (int k = 0; k < (sizeof(io_t) == 4 ? 2 : 3); ++k)
          asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[k]) : "r"(at[i % kPeriod] + i * kPitch + 4 * k) : "memory");
        if constexpr (sizeof(io_t) == 4) return make_uint2(w[0], w[1]);
        return make_uint2(__funnelshift_r(w[0], w[1], shift[i & 1]), __funnelshift_r(w[1], w[2], shift[i & 1]));
      }
    }
  };
  static __device__ __forceinline__ Mine mine(const uint2* space, int group, const io_t* from, long long stride) {
    const uint2* at = space + group * kGroupWords;
    Mine m{};
    if constexpr (ALIGNED) {
      const int swap = (group & 1) * kLanes;
      m.even = at + static_cast<int>(threadIdx.x) % kLanes + swap;
      m.odd = m.even - 2 * swap;
    } else {
      const unsigned start = static_cast<unsigned>(__cvta_generic_to_shared(at)) + threadIdx.x % kLanes * 8;
      const unsigned first = static_cast<unsigned>(reinterpret_cast<uintptr_t>(from));
      const unsigned step = static_cast<unsigned>(stride) * static_cast<unsigned>(sizeof(io_t));
#pragma unroll
      for (int k = 0; k < Mine::kPeriod; ++k) m.at[k] = (start + ((first + k * step) & 15u)) & ~3u;
      m.shift[0] = (first & 2u) * 8u;
      m.shift[1] = ((first + step) & 2u) * 8u;
    }
    return m;
  }

  static __device__ __forceinline__ void copy(unsigned to, const void* from, int bytes) {  // 16 bytes, of which `bytes` exist
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" : : "r"(to), "l"(from), "r"(bytes) : "memory");
  }
  // A 16-byte piece of a row: nothing behind `end` is read, and nothing before the tensor's first element.
  static __device__ __forceinline__ void piece(unsigned to, uintptr_t from, uintptr_t end, const io_t* tensor) {
    const uintptr_t begin = reinterpret_cast<uintptr_t>(tensor);
    if (from >= end) return;
    if (from >= begin) {
      copy(to, reinterpret_cast<const void*>(from), end - from < 16 ? static_cast<int>(end - from) : 16);
    } else {  // the first piece of a tensor that begins inside it
      for (unsigned k = static_cast<unsigned>(begin - from); k < 16 && from + k < end; k += sizeof(io_t)) {
        const io_t value = *reinterpret_cast<const io_t*>(from + k);
        if constexpr (sizeof(io_t) == 4) asm volatile("st.shared.f32 [%0], %1;" : : "r"(to + k), "f"(value) : "memory");
        else asm volatile("st.shared.u16 [%0], %1;" : : "r"(to + k), "h"(*reinterpret_cast<const unsigned short*>(&value)) : "memory");
      }
    }
  }
  // Rows [0, rows) of `base` + row * stride (for this warp), `channels` of the block's 8 * V; what does not exist is not read.
  // FULL: all of them exist and lie 16 bytes or more behind the tensor's beginning.  `tensor` is its first element.
  template <bool FULL>
  static __device__ __forceinline__ void fetch(uint2* space, const io_t* base, long long stride, int rows, int channels, const io_t* tensor) {
    const int lane = threadIdx.x & 31;
    const int part = lane & 3, first = lane >> 2;  // four pieces of eight rows at once
    const unsigned to = static_cast<unsigned>(__cvta_generic_to_shared(space));
    static_assert(S % 8 == 0, "eight rows at once are of one group");
    if constexpr (ALIGNED) {
      // kParts accesses a row, kAtOnce rows at once, which are of one group and whole pairs
      constexpr int kElements = ALIGN / static_cast<int>(sizeof(io_t)), kParts = 64 / ALIGN, kAtOnce = 32 / kParts;
      const int access = lane % kParts, at_once = lane / kParts;
      const io_t* from = base + at_once * stride + access * kElements;
      const bool in = access * kElements < channels;
#pragma unroll
      for (int i = 0; i < kGroups * S / kAtOnce; ++i) {
        const int group = i * kAtOnce / S;
        const unsigned at = to + group * kGroupWords * 8 + (i * kAtOnce - group * S) * 64 + (at_once ^ (group & 1)) * 64 + access * ALIGN;
        const bool there = FULL || (in && i * kAtOnce + at_once < rows);
        if constexpr (ALIGN == 16)
          copy(at, there ? from : tensor, there ? 16 : 0);
        else
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" : : "r"(at), "l"(there ? from : tensor), "r"(there ? 4 : 0) : "memory");
        from += kAtOnce * stride;
      }
    } else {
      if constexpr (FULL) {
        const auto row_pieces = [&](unsigned at, const io_t* from, int which) {
          const uintptr_t address = reinterpret_cast<uintptr_t>(from);
          copy(at + which * 16, reinterpret_cast<const char*>(address & ~uintptr_t{15}) + which * 16,
               which < 4 ? 16 : static_cast<int>(address & 15));
        };
        const io_t* from = base + first * stride;
#pragma unroll
        for (int i = 0; i < kGroups * S / 8; ++i) {
          const int group = i * 8 / S;
          row_pieces(to + group * kGroupWords * 8 + (i * 8 - group * S + first) * kPitch, from, part);
          from += 8 * stride;
        }
        from = base + lane * stride;
#pragma unroll
        for (int i = 0; i < kGroups * S / 32; ++i) {
          const int group = (i * 32 + lane) / S;
          row_pieces(to + group * kGroupWords * 8 + (i * 32 + lane - group * S) * kPitch, from, 4);
          from += 32 * stride;
        }
      } else {
        const int bytes = min(channels, 8 * V) * static_cast<int>(sizeof(io_t));
        for (int i = lane; i < kGroups * S * 5; i += 32) {
          const int row = i / 5, which = i - 5 * row, group = row / S;
          if (row >= rows) break;
          const uintptr_t from = reinterpret_cast<uintptr_t>(base + row * stride);
          piece(to + group * kGroupWords * 8 + (row - group * S) * kPitch + which * 16, (from & ~uintptr_t{15}) + which * 16,
                from + bytes, tensor);
        }
      }
    }
  }
  template <bool FULL> static __device__ __forceinline__ void store(io_t* to, const Lanes<V>& a, int count) {
    const uint2 w = pack<io_t>(a);
    if constexpr (ALIGN == 16) {
      if (FULL || count > 0) __stcs(reinterpret_cast<uint2*>(to), w);
    } else if (FULL || count >= V) {
      if (sizeof(io_t) == 4 || (reinterpret_cast<uintptr_t>(to) & 2) == 0) {
        __stcs(reinterpret_cast<unsigned*>(to), w.x);
        __stcs(reinterpret_cast<unsigned*>(to) + 1, w.y);
      } else {
        unsigned short* half = reinterpret_cast<unsigned short*>(to);
        half[0] = static_cast<unsigned short>(w.x);
        __stcs(reinterpret_cast<unsigned*>(half + 1), __funnelshift_r(w.x, w.y, 16));
        half[3] = static_cast<unsigned short>(w.y >> 16);
      }
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

// The same where a lane's states are known to exist and to be aligned to their size.
template <int V> __device__ __forceinline__ Lanes<V> load_states_whole(const float* from) {
  Lanes<V> r;
  if constexpr (V == 4) {
    const float4 w = __ldcs(reinterpret_cast<const float4*>(from));
    r.v[0] = make_float2(w.x, w.y);
    r.v[1] = make_float2(w.z, w.w);
  } else {
    r.v[0] = __ldcs(reinterpret_cast<const float2*>(from));
  }
  return r;
}
template <int V> __device__ __forceinline__ void store_states_whole(float* to, const Lanes<V>& a) {
  if constexpr (V == 4) __stcs(reinterpret_cast<float4*>(to), make_float4(a.v[0].x, a.v[0].y, a.v[1].x, a.v[1].y));
  else __stcs(reinterpret_cast<float2*>(to), a.v[0]);
}

// ---- gate

// What a token does to the state.  LOGITS keeps rho - 1, otherwise rho is kept (see the top of the file).
template <bool LOGITS, bool COMPLEMENT, int V> struct Decay {
  using L = Lanes<V>;

  // The SFU's exp2 and reciprocal: errors of 2^-22 and 2^-23, those of exp2f and nearly those of a division (what they flush to
  // zero is far below what is added to it).
  static __device__ __forceinline__ L exp2(const L& x) {
    return each([](float v) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }, x);
  }
  static __device__ __forceinline__ L reciprocal(const L& x) {
    return each([](float v) { float r; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }, x);
  }
  // e = exp(-(raw + bias)) from bias * -log2 e; the sigmoid is 1 / (1 + e)
  static __device__ __forceinline__ L exponential(const L& raw, const L& bias) { return exp2(fma(raw, L::all(-kLog2e), bias)); }
  static __device__ __forceinline__ L sigmoid_of(const L& e) { return reciprocal(add(e, L::all(1.0f))); }
  static __device__ __forceinline__ L sigmoid(const L& raw, const L& bias) { return sigmoid_of(exponential(raw, bias)); }
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
  // d rho / d raw from e and g = 1 / (1 + e): -c g (1 - g) rho.  1 - g is e g, which loses nothing where g is nearly one (1 - g
  // would be 6 % off for a logit of 16); e is infinite, or so large that g was flushed to zero, only where the slope is zero.
  static __device__ __forceinline__ L slope(const L& e, const L& g, const L& kept) {
    const L rest = mul(each([](float v) { return fminf(v, 0x1p126f); }, e), g);
    return mul(mul(rest, fma(kept, L::all(-kRate), L::all(-kRate))), g);
  }
};

// ---- affine maps h -> a h + b
//
// a is the product of the rho of up to 2048 tokens, and the carried state passes through one for each 16 of them.  As one fp32
// number it would be rounded at every token, by up to 2^-25 where its distance to one may be a millionth, and with a steady
// decay to the same side each time (16384 tokens with 1 - rho = 1.2e-5: 1.2e-4 rms of the values, walked token by token 1.5e-6).
// So the maps carry a as a sum of two numbers (1.8e-7).  It begins with a lane's tokens, whose product is known well in two
// ways: as a - 1 where that is small, and as a where that is.

// The product of the rho of a lane's tokens: from logits exp(-c times the sum of their sigmoids), else multiplied out, with the
// sum of what each token takes away.
template <bool LOGITS, int V> struct Fade;

template <int V> struct Fade<true, V> {
  using L = Lanes<V>;
  L gates;

  static __device__ __forceinline__ Fade none() { return Fade{L::all(0.0f)}; }
  __device__ __forceinline__ void take(const L& sigmoid, const L&) { gates = add(gates, sigmoid); }
  __device__ __forceinline__ L product() const { return Decay<true, false, V>::exp2(mul(gates, L::all(-kRateLog2e))); }
  __device__ __forceinline__ L fall() const { return Decay<true, false, V>::keep_gate(gates); }  // product - 1
  __device__ __forceinline__ L trifle() const { return L::all(0x1p-100f); }  // positive, and nothing beside a product of 16 rho
  __device__ __forceinline__ L choice() const { return gates; }
  static __device__ __forceinline__ bool is_slow(float gates) { return gates <= 1.0f; }  // fall() is good
};

template <int V> struct Fade<false, V> {
  using L = Lanes<V>;
  L a, less;

  static __device__ __forceinline__ Fade none() { return Fade{L::all(1.0f), L::all(0.0f)}; }
  __device__ __forceinline__ void take(const L&, const L& rho) {
    less = fma(minus(rho, L::all(1.0f)), a, less);
    a = mul(rho, a);
  }
  __device__ __forceinline__ L product() const { return a; }
  __device__ __forceinline__ L fall() const { return less; }
  __device__ __forceinline__ L trifle() const { return mul(a, L::all(0x1p-30f)); }
  __device__ __forceinline__ L choice() const { return a; }
  static __device__ __forceinline__ bool is_slow(float a) { return a >= 0.5f; }
};

// `low` has a's sign and is zero only with it (so an infinite state stays one, and does not become infinity less infinity):
// what is rounded is rounded towards zero, and where nothing is left over it is a trifle.
template <int V> struct Map {
  Lanes<V> a, low, b;  // a + low, b

  template <bool LOGITS> static __device__ __forceinline__ Map of(const Fade<LOGITS, V>& fade, const Lanes<V>& b) {
    const Lanes<V> one = Lanes<V>::all(1.0f), fall = fade.fall(), choice = fade.choice();
    Lanes<V> sum;
#pragma unroll
    for (int i = 0; i < V / 2; ++i) sum.v[i] = __fadd2_rz(one.v[i], fall.v[i]);
    const Lanes<V> rest = add(minus(fall, minus(sum, one)), Lanes<V>::all(0x1p-50f));
    Map m{fade.product(), fade.trifle(), b};
    const auto choose = [](float by, float& a, float& low, float sum, float rest) {
      const bool slow = Fade<LOGITS, V>::is_slow(by);
      a = slow ? sum : a;
      low = slow ? rest : low;
    };
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      choose(choice.v[i].x, m.a.v[i].x, m.low.v[i].x, sum.v[i].x, rest.v[i].x);
      choose(choice.v[i].y, m.a.v[i].y, m.low.v[i].y, sum.v[i].y, rest.v[i].y);
    }
    return m;
  }
  __device__ __forceinline__ Lanes<V> apply(const Lanes<V>& h) const { return fma(a, h, fma(low, h, b)); }
  // this map, then `next`
  __device__ __forceinline__ void then(const Map& next) {
    Lanes<V> product;
#pragma unroll
    for (int i = 0; i < V / 2; ++i) product.v[i] = __fmul2_rz(a.v[i], next.a.v[i]);
    const Lanes<V> rest = fma(a, next.a, mul(product, Lanes<V>::all(-1.0f)));
    b = next.apply(b);
    low = fma(a, next.low, fma(low, next.a, rest));
    a = product;
  }
};

template <int V> __device__ __forceinline__ Lanes<V> shuffle_up(const Lanes<V>& x, int lanes) {
  Lanes<V> r;
#pragma unroll
  for (int i = 0; i < V / 2; ++i)
    r.v[i] = make_float2(__shfl_up_sync(0xffffffffu, x.v[i].x, lanes), __shfl_up_sync(0xffffffffu, x.v[i].y, lanes));
  return r;
}

}  // namespace frwkv
