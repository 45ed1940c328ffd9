// kv_attend.hpp -- what the attention kernels of the 8-bit key/value cache
// share: their arguments, codes and queries as operands of the matrix cores,
// and the last step of a row.
#pragma once

#include "kv_common.hpp"

namespace grm {
namespace kv {

struct AttendArgs {
  const int8_t* k_codes;
  const int8_t* v_codes;
  const float* k_scales;
  const float* v_scales;
  const void* q;
  void* out;
  float* lse;
  const int32_t* ctx_lens;
  const int32_t* cu_new;
  const int32_t* table;
  const char* work;
  float* parts;
  int64_t q_token_stride, q_head_stride, out_token_stride, out_head_stride;
  uint64_t blocks, at_units, at_tiles, at_run_units, at_items, at_joins;
  float scale;
  int32_t requests, width, tokens, window;
  int32_t heads, kv_heads, group, head_dim, block_log2;
  int32_t cols;       // columns a narrow unit may have
  int32_t whole;      // each block of the narrow kernel takes a whole unit
  int32_t cap_parts;  // wide partial results to a kv head
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Blocks of the narrow kernel to a CU: what its registers allow.
__host__ __device__ constexpr int narrow_blocks_per_cu(int dtype, int head_dim) {
  return head_dim == 256 || (dtype == kF32 && head_dim == 128) ? 1 : 2;
}

// Floats of one partial result of the narrow kernel: its columns' sums of
// weights times codes, then their maxima, their sums of probabilities and the
// powers of two that the sums are in.
__host__ __device__ constexpr int narrow_part_floats(int head_dim) {
  return kNarrowCols * (head_dim + 3);
}

// A run has at most two partial results: of its first unit and of its last.
__device__ inline size_t narrow_part(int g, int runs, int run, int which) {
  return (static_cast<size_t>(g) * runs + run) * 2 + which;
}

// A lane's eight values of an operand, all fp16 or (BF) all bf16.
template <bool BF>
__device__ inline f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (BF) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
}
template <bool BF>
__device__ inline f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (BF) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
}

// The upper halves of two words: two fp32 values as bf16, cut.
__device__ inline uint32_t upper_halves(uint32_t lo, uint32_t hi) {
  return __builtin_amdgcn_perm(hi, lo, 0x07060302u);
}

// Eight codes, exactly.  fp16: a byte under the exponent of 1024 is 1024 + u,
// and u = code + 128.  bf16: by fp32, of which an integer below 256 needs the
// upper half only (12 instructions against 10).
template <bool BF>
__device__ inline u32x4 codes_as(uint32_t first, uint32_t second) {
  u32x4 out;
  if constexpr (BF) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t w = k < 2 ? first : second;
      out[k] = upper_halves(__float_as_uint(static_cast<float>(code_at(w, 2 * (k & 1)))),
                            __float_as_uint(static_cast<float>(code_at(w, 2 * (k & 1) + 1))));
    }
  } else {
    const f16x2 off = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint32_t u = (k ? second : first) ^ 0x80808080u;
      const uint32_t lo = __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u);
      const uint32_t hi = __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u);
      out[2 * k] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, lo) + off);
      out[2 * k + 1] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, hi) + off);
    }
  }
  return out;
}

template <bool BF>
__device__ inline void codes_as(u32x4 w, u32x4 (&out)[2]) {
  out[0] = codes_as<BF>(w[0], w[1]);
  out[1] = codes_as<BF>(w[2], w[3]);
}

// A product as fp32 holds it.  Left open, the compiler rounds it to fp16 from
// its exact value in one place and from fp32 in another, and where the two
// differ the rest that is taken of one is a unit off the other.
__device__ inline float as_rounded(float v) {
  asm("" : "+v"(v));
  return v;
}

// Two values as N bf16 terms of eight bits, cut: what is left is exact, and of
// three terms nothing is.
template <int N>
__device__ inline void bf16_terms(float a, float b, uint32_t (&t)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n) {
    t[n] = upper_halves(__float_as_uint(a), __float_as_uint(b));
    a -= __uint_as_float(__float_as_uint(a) & 0xffff0000u);
    b -= __uint_as_float(__float_as_uint(b) & 0xffff0000u);
  }
}

// Two values as two fp16 terms: both rounded in one instruction, and what that
// leaves of each (exact) with the conversion back in one.  Spelt out, since the
// compiler rounds each of them a second time for the conversion back: 112
// instructions more to a tile of the wide kernel's against 48.
__device__ inline void fp16_terms(float a, float b, uint32_t (&t)[2]) {
  f16x2 v;
  v[0] = static_cast<_Float16>(a);
  v[1] = static_cast<_Float16>(b);
  t[0] = __builtin_bit_cast(uint32_t, v);
  float left[2];
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[0,0,0] op_sel_hi:[1,0,0]"
      : "=v"(left[0]) : "v"(t[0]), "v"(a));
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]"
      : "=v"(left[1]) : "v"(t[0]), "v"(b));
  v[0] = static_cast<_Float16>(left[0]);
  v[1] = static_cast<_Float16>(left[1]);
  t[1] = __builtin_bit_cast(uint32_t, v);
}

// A weight's terms in the second product: whole for fp32 outputs, 22 bits for
// 16-bit ones.
template <class T>
__host__ __device__ constexpr bool weight_bf16() { return T::code == kF32; }
template <class T>
__host__ __device__ constexpr int weight_terms() { return T::code == kF32 ? 3 : 2; }

template <class T>
__device__ inline void split_weights(float a, float b, uint32_t (&t)[weight_terms<T>()]) {
  if constexpr (weight_bf16<T>()) bf16_terms(a, b, t);
  else fp16_terms(a, b, t);
}

template <class T>
__device__ inline void load8(const typename T::store* p, float (&x)[8]) {
  if constexpr (T::code == kF32) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p);
    const f32x4 b = *reinterpret_cast<const f32x4*>(p + 4);
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

// Query values as terms of the first product.  fp16 is taken as it is.  bf16
// and fp32 go as bf16 (one term, three), which holds every bit of channels of
// any size beside each other: a key may have nothing in the largest.  They are
// in units of a power of two that brings the column's largest (`top`) into
// [1/2, 1), for sums that stay in range.  Returns `scale` times the unit.
template <class T>
__host__ __device__ constexpr bool query_bf16() { return T::code != kF16; }

template <class T, int N, int TERMS>
__device__ inline float split_query(const float (&x)[N][8], float top, float scale,
                                    u32x4 (&q)[TERMS][N]) {
  int unit = 0;
  if constexpr (query_bf16<T>()) {
    if (top > 0.0f && top <= 3.4028235e38f) unit = __builtin_amdgcn_frexp_expf(top);
  }
#pragma unroll
  for (int s = 0; s < N; ++s) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      if constexpr (query_bf16<T>()) {
        uint32_t t[TERMS];
        bf16_terms(__builtin_amdgcn_ldexpf(x[s][e], -unit),
                   __builtin_amdgcn_ldexpf(x[s][e + 1], -unit), t);
#pragma unroll
        for (int n = 0; n < TERMS; ++n) q[n][s][e / 2] = t[n];
      } else {
        f16x2 v;
        v[0] = static_cast<_Float16>(x[s][e]);
        v[1] = static_cast<_Float16>(x[s][e + 1]);
        q[0][s][e / 2] = __builtin_bit_cast(uint32_t, v);
      }
    }
  }
  return __builtin_amdgcn_ldexpf(scale, unit);
}

// The power of two at or above a positive finite number.
__device__ inline float power_above(float v) {
  // frexp: v = f 2^e with f in [1/2, 1), so 2^e > v; kept where its
  // reciprocal is a number too
  const int e = __builtin_amdgcn_frexp_expf(v);
  return __builtin_amdgcn_ldexpf(1.0f, e > 127 ? 127 : e < -120 ? -120 : e);
}

// Log2 of what probabilities are scaled by on their way into fp16.
__host__ __device__ constexpr float weight_bias(int dtype) { return dtype == kF32 ? 0.0f : 13.0f; }

// What takes sums in units of `from` to units of `to`, a power of two no less
// (0: nothing was summed).
__device__ inline float unit_change(float from, float to) { return to > 0.0f ? from / to : 1.0f; }

// Four values of a finished row: o / l, which is a mean, times the power of two
// it is in, so that nothing passes fp32's range before (a sum of large values
// would), rounded once; and the row's log-sum-exp by the thread of its first
// column.  m in log2 units, l and o biased.
template <class T>
__device__ inline void finish4(const AttendArgs& a, int row, int h, int d, f32x4 o, float m,
                               float l, float ref) {
  const bool empty = m == -INFINITY && l == 0.0f;
  const float inv = 1.0f / l;
  typename T::store* out = static_cast<typename T::store*>(a.out) +
                           static_cast<int64_t>(row) * a.out_token_stride +
                           static_cast<int64_t>(h) * a.out_head_stride + d;
  if constexpr (T::code == kF32) {
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = empty ? 0.0f : o[e] * inv * ref;
    *reinterpret_cast<f32x4*>(out) = v;
  } else {
    u32x2 v;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t lo = T::put(empty ? 0.0f : o[2 * e] * inv * ref);
      const uint32_t hi = T::put(empty ? 0.0f : o[2 * e + 1] * inv * ref);
      v[e] = lo | (hi << 16);
    }
    *reinterpret_cast<u32x2*>(out) = v;
  }
  if (a.lse && d == 0) {
    a.lse[static_cast<size_t>(row) * a.heads + h] =
        empty ? -INFINITY : (m - weight_bias(T::code) + __builtin_amdgcn_logf(l)) * kLn2;
  }
}

}  // namespace kv
}  // namespace grm
