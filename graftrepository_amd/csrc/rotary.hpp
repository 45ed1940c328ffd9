// rotary.hpp -- rotary positions: a pair (a, b) of channels at position p
// becomes
//
//   (a cos t - b sin t, b cos t + a sin t) * magnitude,  t = pi / 2 p quarters[pair].
//
// No table of sines is kept: p * quarters in 64 bits less its whole part is
// rounded once, whatever the position, and the rest, x in [-1/2, 1/2], goes on in 32
// bits (off by 2^-26: an angle by 2^-25.3).  There the sine and cosine of pi/2 x are
// their power series, to x^9 and x^10 (what is left out is below 2^-29), a third of
// the instructions of a library's call: an append of 14151 turned tokens, which
// vector instructions bound, took 33 us with that and takes 31.
#pragma once

#include "kv_common.hpp"

namespace grm {
namespace kv {

constexpr int kMaxPairs = 128;
constexpr int kHalf = 0, kNeighbours = 1;  // layouts

// By value in a kernel's arguments.
struct Rotary {
  double quarters[kMaxPairs];  // of a turn, a position
  float magnitude;
  int32_t dim, layout;
};

int rotary_of(const grm_rotary_desc* d, int channels, Rotary* out);

struct CosSin {
  float cos, sin;
};

__device__ inline CosSin angle(const Rotary& r, int pair, int position) {
  // (added to this, a number's whole part is in the low bits)
  constexpr double kWhole = 6755399441055744.0;  // 1.5 * 2^52
  const double p = static_cast<double>(position), quarters = r.quarters[pair];
  const double at = fma(p, quarters, kWhole);
  const float x = static_cast<float>(fma(p, quarters, kWhole - at));
  const uint32_t quarter = static_cast<uint32_t>(__double2loint(at));
  // (pi/2)^n / n!
  const float y = x * x;
  float sin = fmaf(y, 1.6044118e-4f, -4.6817541e-3f);
  sin = fmaf(y, sin, 7.9692626e-2f);
  sin = fmaf(y, sin, -6.4596410e-1f);
  sin = x * fmaf(y, sin, 1.5707963f);
  float cos = fmaf(y, -2.5202042e-5f, 9.1926027e-4f);
  cos = fmaf(y, cos, -2.0863480e-2f);
  cos = fmaf(y, cos, 2.5366951e-1f);
  cos = fmaf(y, cos, -1.2337006f);
  cos = fmaf(y, cos, 1.0f);
  // a quarter on: (cos, sin) becomes (-sin, cos)
  const bool odd = quarter & 1u;
  const float c = odd ? sin : cos, s = odd ? cos : sin;
  CosSin a;
  a.cos = __uint_as_float(__float_as_uint(c) ^ ((quarter + 1u) << 30 & 0x80000000u)) * r.magnitude;
  a.sin = __uint_as_float(__float_as_uint(s) ^ (quarter << 30 & 0x80000000u)) * r.magnitude;
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
