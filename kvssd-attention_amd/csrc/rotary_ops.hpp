// Rotation of value pairs, shared by the rotary kernel and the paged append
// (a key rotated on its way into the cache has the bits of one rotated alone).
//
// The angle p f, its sine and cosine and the products are formed in 64 bits:
// at position 10^6 a 32-bit angle is off by up to 0.03 radians, and a key that
// a 32-bit product puts on the other side of a rounding border changes a code
// of the cache by a whole step.  One rounding to 32 bits and, for 16-bit
// types, one to the type follow, as torch's conversion from double does.  The
// sines, which cost most, are formed once per token and pair and shared by all
// heads through LDS.
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

// One item of a head: PV pairs turned (`turns` of the token), or PV values
// passed through.  Every value is read and written by one thread only, so y
// may be x.
template <typename T, int PV>
__device__ __forceinline__ void rotary_item(const RotaryShape& s, int item, const T* x, T* y, const Turn* turns) {
  if (item >= s.turn_items) {
    const int at = 2 * s.pairs + (item - s.turn_items) * PV;
    if (x == y) return;
    T v[PV];
    load_values(x + at, v);
    store_values(y + at, v);
    return;
  }
  const int p0 = item * PV;
  T a[PV], b[PV];
  const int at0 = s.interleaved ? 2 * p0 : p0;
  const int at1 = s.interleaved ? 2 * p0 + PV : s.pairs + p0;
  load_values(x + at0, a);
  load_values(x + at1, b);
  T lo[PV], hi[PV];
  if (s.interleaved) {
#pragma unroll
    for (int i = 0; i < PV; ++i) {
      const T va = 2 * i < PV ? a[(2 * i) % PV] : b[(2 * i) % PV];
      const T vb = 2 * i + 1 < PV ? a[(2 * i + 1) % PV] : b[(2 * i + 1) % PV];
      const Turn t = turns[p0 + i];
      const T l = store_cast<T>(turn_low(to_f32(va), to_f32(vb), t));
      const T h = store_cast<T>(turn_high(to_f32(va), to_f32(vb), t));
      if (2 * i < PV) lo[(2 * i) % PV] = l;
      else hi[(2 * i) % PV] = l;
      if (2 * i + 1 < PV) lo[(2 * i + 1) % PV] = h;
      else hi[(2 * i + 1) % PV] = h;
    }
  } else {
#pragma unroll
    for (int i = 0; i < PV; ++i) {
      const Turn t = turns[p0 + i];
      lo[i] = store_cast<T>(turn_low(to_f32(a[i]), to_f32(b[i]), t));
      hi[i] = store_cast<T>(turn_high(to_f32(a[i]), to_f32(b[i]), t));
    }
  }
  store_values(y + at0, lo);
  store_values(y + at1, hi);
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
