// Rotation of value pairs, shared by the rotary kernel and the paged append
// (a key rotated on its way into the cache has the bits of one rotated alone).
//
// The angle p f, its sine and cosine and the products are formed in 64 bits:
// at position 10^6 a 32-bit angle is off by up to 0.03 radians, and a key that
// a 32-bit product puts on the other side of a rounding border changes a code
// of the cache by a whole step.  One rounding to 32 bits and, for 16-bit
// types, one to the type follow, as torch's conversion from double does.  The
// sines, which cost most, are formed once per token and pair and shared by all
// heads through LDS.  What 64 bits cost: 7 us of the 36 of a prompt's append
// (16,381 tokens of 8 kv heads), nothing of the rotary kernel, which waits for
// memory.
#pragma once

#include "quant_ops.hpp"

namespace kvssd {

struct Turn {
  double c, s;  // magnitude times cosine and sine
};

__device__ __forceinline__ Turn make_turn(double position, double frequency, double magnitude, int inverse) {
  double s, c;
  sincos(position * frequency, &s, &c);
  return Turn{magnitude * c, inverse ? -(magnitude * s) : magnitude * s};
}

// A token's turns in LDS, one place left free after every 8: lanes that read the turns of words or items 8 pairs apart
// then meet no bank twice (16 bytes each, 64 banks of 4; a prompt's append 45.4 -> 41.7 us).
__host__ __device__ constexpr int turn_place(int pair) { return pair + pair / 8; }

// (a, b) turned: a c - b s and b c + a s
__device__ __forceinline__ float turn_low(double a, double b, Turn t) {
  return static_cast<float>(__builtin_fma(a, t.c, -(b * t.s)));
}
__device__ __forceinline__ float turn_high(double a, double b, Turn t) {
  return static_cast<float>(__builtin_fma(b, t.c, a * t.s));
}

template <typename T, int N>
__device__ __forceinline__ void load_values(const T* src, T (&v)[N]) {
  if constexpr (sizeof(T) * N >= 16) {
    __builtin_memcpy(v, __builtin_assume_aligned(src, 16), sizeof(v));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = src[i];
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_values(T* dst, const T (&v)[N]) {
  if constexpr (sizeof(T) * N >= 16) {
    __builtin_memcpy(__builtin_assume_aligned(dst, 16), v, sizeof(v));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) dst[i] = v[i];
  }
}

// What the host works out about a rotation of heads of `head_dim` values.
struct RotaryShape {
  int head_dim, pairs, interleaved;
  int turn_items, items;  // per head: items of PV pairs, then items of PV values passed through
};

inline RotaryShape rotary_shape(const kvssd_rotary_spec& r, int pv) {
  RotaryShape s{};
  s.head_dim = r.head_dim;
  s.pairs = r.rotary_dim / 2;
  s.interleaved = r.interleaved;
  s.turn_items = s.pairs / pv;
  s.items = s.turn_items + (r.head_dim - r.rotary_dim) / pv;
  return s;
}

// x in type T, rounded to nearest even (a NaN stays one).  x is rounded to 32 bits already, and kept from the compiler,
// which may otherwise round the 64-bit value before it to 16 bits at once: another result in 2^-17 of the values.
template <typename T>
__device__ __forceinline__ T round_to(float x) {
  if constexpr (sizeof(T) == 2) asm("" : "+v"(x));
  if constexpr (__is_same(T, uint16_t)) return __builtin_bit_cast(uint16_t, static_cast<__bf16>(x));
  else return static_cast<T>(x);
}

// One item of a head: PV pairs to turn, or PV values to pass through (a alone; none where y is x).  Every value is
// read and written by one thread only, so y may be x.
template <typename T, int PV>
struct RotaryItem {
  T a[PV], b[PV];

  static __device__ __forceinline__ int first(const RotaryShape& s, int item) {
    return item >= s.turn_items ? 2 * s.pairs + (item - s.turn_items) * PV : s.interleaved ? 2 * item * PV : item * PV;
  }
  __device__ __forceinline__ void load(const RotaryShape& s, int item, const T* x, bool in_place) {
    const int at = first(s, item);
    if (item < s.turn_items) load_values(x + at + (s.interleaved ? PV : s.pairs), b);
    if (item < s.turn_items || !in_place) load_values(x + at, a);
  }
  // `turns` of the item's token
  __device__ __forceinline__ void store(const RotaryShape& s, int item, T* y, const Turn* turns, bool in_place) {
    const int at = first(s, item);
    if (item >= s.turn_items) {
      if (!in_place) store_values(y + at, a);
      return;
    }
    const Turn* turn = turns + turn_place(item * PV);  // (PV pairs without a free place among them)
    T lo[PV], hi[PV];
    if (s.interleaved) {
#pragma unroll
      for (int i = 0; i < PV; ++i) {
        const float va = to_f32(2 * i < PV ? a[(2 * i) % PV] : b[(2 * i) % PV]);
        const float vb = to_f32(2 * i + 1 < PV ? a[(2 * i + 1) % PV] : b[(2 * i + 1) % PV]);
        const T l = round_to<T>(turn_low(va, vb, turn[i])), h = round_to<T>(turn_high(va, vb, turn[i]));
        if (2 * i < PV) lo[(2 * i) % PV] = l;
        else hi[(2 * i) % PV] = l;
        if (2 * i + 1 < PV) lo[(2 * i + 1) % PV] = h;
        else hi[(2 * i + 1) % PV] = h;
      }
    } else {
#pragma unroll
      for (int i = 0; i < PV; ++i) {
        lo[i] = round_to<T>(turn_low(to_f32(a[i]), to_f32(b[i]), turn[i]));
        hi[i] = round_to<T>(turn_high(to_f32(a[i]), to_f32(b[i]), turn[i]));
      }
    }
    store_values(y + at, lo);
    store_values(y + at + (s.interleaved ? PV : s.pairs), hi);
  }
};

// Division of 32-bit numbers by one that the host knows.
struct Divisor {
  uint32_t d, m;  // m = 2^32 / d, rounded up
  __device__ __forceinline__ uint32_t quotient(uint32_t x) const {
    if (d == 1) return x;
    const uint32_t q = __umulhi(x, m);  // right or one too many: x m / 2^32 is past x / d by less than 1
    return q * d > x ? q - 1 : q;
  }
};
inline Divisor divisor(int64_t d) {
  return Divisor{static_cast<uint32_t>(d), d > 1 ? static_cast<uint32_t>(((uint64_t{1} << 32) + d - 1) / d) : 0};
}

// 16-byte loads of a heads tensor's values: its addresses and strides allow them
inline bool heads_vector(const kvssd_heads& h, size_t item, bool with_out) {
  auto whole = [&](const void* p, int64_t t, int64_t s) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (t * static_cast<int64_t>(item)) % 16 == 0 &&
           (s * static_cast<int64_t>(item)) % 16 == 0;
  };
  return whole(h.data, h.token_stride, h.head_stride) &&
         (!with_out || whole(h.out, h.out_token_stride, h.out_head_stride));
}

}  // namespace kvssd
