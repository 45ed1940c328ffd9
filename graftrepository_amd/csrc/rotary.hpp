// rotary.hpp -- rotary positions: a pair (a, b) of channels at position p
// becomes
//
//   (a cos t - b sin t, b cos t + a sin t) * magnitude,  t = 2 pi p turns[pair].
//
// No table of sines is kept: p * turns in 64 bits less its whole turns is
// exact to 2^-53 of p * turns, whatever the position, and the rest, in
// (-1/2, 1/2], goes on in 32 bits (an angle is off by 2 pi 2^-26 at most).
#pragma once

#include "kv_common.hpp"

namespace grm {
namespace kv {

constexpr int kMaxPairs = 128;
constexpr int kHalf = 0, kNeighbours = 1;  // layouts

// By value in a kernel's arguments.
struct Rotary {
  double turns[kMaxPairs];
  float magnitude;
  int32_t dim, layout;
};

int rotary_of(const grm_rotary_desc* d, int channels, Rotary* out);

struct CosSin {
  float cos, sin;
};

__device__ inline CosSin angle(const Rotary& r, int pair, int position) {
  const double t = static_cast<double>(position) * r.turns[pair];
  const float part = static_cast<float>(t - rint(t));
  CosSin a;
  sincospif(2.0f * part, &a.sin, &a.cos);
  a.cos *= r.magnitude;
  a.sin *= r.magnitude;
  return a;
}

__device__ inline void turn(const CosSin& t, float& a, float& b) {
  const float x = a, y = b;
  a = fmaf(x, t.cos, -(y * t.sin));
  b = fmaf(y, t.cos, x * t.sin);
}

// The pair that channel d of the turned ones is in, and the other channel.
__device__ inline int pair_of(int layout, int half, int d, int* other) {
  if (layout == kHalf) {
    *other = d < half ? d + half : d - half;
    return d < half ? d : d - half;
  }
  *other = d ^ 1;
  return d >> 1;
}

// Sixteen channels that are turned together, as two runs of eight: unit u of a
// head has eight pairs.  Halves: channels 8 u and half + 8 u on; neighbours: 16
// on from 16 u.
__device__ inline void unit_channels(int layout, int half, int u, int* first, int* second) {
  *first = layout == kHalf ? 8 * u : 16 * u;
  *second = layout == kHalf ? half + 8 * u : 16 * u + 8;
}

template <class Angle>
__device__ inline void turn_unit(int layout, float (&x)[2][8], Angle angle_of) {
  // by selected values: branches of the two layouts end as one with selected
  // addresses, and the array in scratch memory
  const bool half = layout == kHalf;
  float a[8], b[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    a[e] = half ? x[0][e] : x[e / 4][e % 4 * 2];
    b[e] = half ? x[1][e] : x[e / 4][e % 4 * 2 + 1];
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) turn(angle_of(e), a[e], b[e]);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    x[0][e] = half ? a[e] : e % 2 ? b[e / 2] : a[e / 2];
    x[1][e] = half ? b[e] : e % 2 ? b[4 + e / 2] : a[4 + e / 2];
  }
}

// Whether heads of this rotary are whole units.
inline bool whole_units(const Rotary& r) { return r.dim % 16 == 0; }

// Eight values, 16 bytes at a time where their address allows it.
template <class T, bool ALIGNED>
__device__ inline void get8(const typename T::store* p, float (&x)[8]) {
  if constexpr (!ALIGNED) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = T::get(p[e]);
  } else if constexpr (T::code == kF32) {
    const f32x4 a = reinterpret_cast<const f32x4*>(p)[0], b = reinterpret_cast<const f32x4*>(p)[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = a[e];
      x[4 + e] = b[e];
    }
  } else {
    const u32x4 w = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = T::get(static_cast<uint16_t>((w[e / 2] >> (16 * (e & 1))) & 0xffffu));
    }
  }
}

template <class T, bool ALIGNED>
__device__ inline void put8(typename T::store* p, const float (&x)[8]) {
  if constexpr (!ALIGNED) {
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = T::put(x[e]);
  } else if constexpr (T::code == kF32) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = x[4 * k + e];
      reinterpret_cast<f32x4*>(p)[k] = v;
    }
  } else {
    u32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t lo = T::put(x[2 * e]), hi = T::put(x[2 * e + 1]);
      v[e] = lo | (hi << 16);
    }
    *reinterpret_cast<u32x4*>(p) = v;
  }
}

}  // namespace kv
}  // namespace grm
