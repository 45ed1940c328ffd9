// kv_wide.hpp -- attention of requests that bring many tokens (prompts and
// chunks of prompts).
//
// An item is up to 128 (token, head) columns of one kv head against a range
// of key tiles (64 tokens).  It is bound by the matrix cores and the vector
// unit beside them, so the codes are turned into fp16 once per block and tile:
// a block's four wavefronts load the next tile's codes to registers, write
// them to LDS as fp16 (exact) in the order in which the matrix instructions
// take them (16 bytes per lane, no bank conflicts), and each multiplies the
// tile with its own 32 columns (32x32x16).  Two LDS buffers, one barrier per
// tile; two blocks share a CU where registers allow, so that one's vector
// work runs beside the other's matrix work.
//
// Layout of the products (lane = c + 32 h):
//   S^T = K Q^T: row 8 m + 4 h' + j of a 32-key row tile is its key
//     16 h' + 4 m + j, so that a lane's 16 results are the neighbouring keys
//     16 h .. 16 h + 15 of column c;
//   O^T = V^T P^T: those are the lane's part of the B operand, 8 keys to an
//     instruction, and the A operand's lane holds the same keys of a value
//     column.
// The softmax is the narrow kernel's: one pass, scores and statistics in fp32,
// weights in fp16 (two terms for fp16 and fp32 outputs).
//
// Items of one kv head follow each other at a distance of kv_heads blocks, so
// with 8 kv heads an XCD's L2 serves one of them.
#pragma once

#include "kv_narrow.hpp"

namespace grm {
namespace kv {



// Blocks to a CU: registers (accumulators of 32 columns, twice for fp32) and
// the two LDS buffers.
__host__ __device__ constexpr int wide_blocks_per_cu(int dtype, int head_dim) {
  return head_dim == 256 || (dtype == kF32 && head_dim == 128) ? 1 : 2;
}

// Floats of one partial result: 128 columns, and their maxima and sums.
__host__ __device__ constexpr int wide_part_floats(int head_dim) {
  return kWideCols * (head_dim + 2);
}

template <class T, int D>
__global__ __launch_bounds__(256, wide_blocks_per_cu(T::code, D)) void attend_wide_kernel(
    AttendArgs a) {
  typedef NarrowState<T, D> State;  // its constants: terms and allowances
  constexpr int kSteps = D / 16;    // of the first product
  constexpr int kTilesD = D / 32;   // value row tiles
  constexpr int kChunks = D / 64;   // 16-byte chunks of keys, and of values, to a thread
  const int g = blockIdx.x;
  const auto* head = reinterpret_cast<ConstHead>(reinterpret_cast<uintptr_t>(a.work));
  if (static_cast<int>(blockIdx.y) >= head->items) return;
  const auto* item = reinterpret_cast<ConstItem>(reinterpret_cast<uintptr_t>(a.work) + a.at_items) +
                     blockIdx.y;
  if (item->tokens <= 0) return;
  const auto* table = reinterpret_cast<ConstInt>(reinterpret_cast<uintptr_t>(a.table));
  const int lane = __lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int c = lane & 31, h = lane >> 5;
  const int tile_lo = item->tile_lo, tile_hi = item->tile_hi;
  const int first_pos = item->pos, last_pos = first_pos + item->tokens - 1;
  const int cols = item->tokens * a.group;
  const size_t table_row = static_cast<size_t>(item->request) * a.width;
  const int bs = 1 << a.block_log2;
  const uint32_t cell_bytes = static_cast<uint32_t>(bs * D);

  __shared__ f16x8 s_k[2][2 * kSteps * kWave];       // [row tile][step][lane]
  __shared__ f16x8 s_v[2][kTilesD * 4 * kWave];      // [d tile][row tile][half][lane]
  __shared__ float s_scale[2][2][4];                 // [keys, values][group of 16]

  // ---- codes of a tile to registers
  u32x4 k_reg[kChunks], v_reg[kChunks];
  float scale_reg = 0.0f;
  int seen_reg = 0;  // groups whose block is there, as bits
  auto load_codes = [&](int tile) {
    const int first_seen = a.window > 0 ? max(0, first_pos + 1 - a.window) : 0;
    int id[4], seen = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int key = tile * kTile + 16 * k, at = key >> a.block_log2;
      const int raw = table[table_row + max(0, min(at, a.width - 1))];
      const bool there = key <= last_pos && key + 15 >= first_seen && at < a.width &&
                         static_cast<uint32_t>(raw) < a.blocks;
      id[k] = there ? raw : 0;
      seen |= there ? 1 << k : 0;
    }
    seen_reg = seen;
    auto cell_of = [&](int k) {
      const int lo = k & 1 ? id[1] : id[0], hi = k & 1 ? id[3] : id[2];
      return static_cast<uint32_t>(k & 2 ? hi : lo) * a.kv_heads + g;
    };
    // Keys: lane = 8 tokens x 8 chunks of a wave's group.
#pragma unroll
    for (int q = 0; q < kChunks; ++q) {
      const int n = q * 256 + static_cast<int>(threadIdx.x);
      const int t8 = n & 7, chunk = (n >> 3) % kSteps, grp = (n >> 3) / kSteps;
      const int key = 32 * (grp >> 2) + 16 * (t8 >> 2) + 4 * (grp & 3) + (t8 & 3);
      const int8_t* p = a.k_codes + static_cast<uint64_t>(cell_of(key >> 4)) * cell_bytes +
                        ((tile * kTile + key) & (bs - 1)) * D + 16 * chunk;
      k_reg[q] = *reinterpret_cast<const u32x4*>(p);
    }
    // Values: a wave's 16 tokens, a value column per lane.
#pragma unroll
    for (int q = 0; q < kChunks; ++q) {
      const int8_t* p = a.v_codes + static_cast<uint64_t>(cell_of(wave)) * cell_bytes +
                        static_cast<size_t>(q * kWave + lane) * bs +
                        ((tile * kTile + 16 * wave) & (bs - 1));
      v_reg[q] = *reinterpret_cast<const u32x4*>(p);
    }
    if (threadIdx.x < 8) {
      const int k = threadIdx.x & 3;
      const uint32_t cell = cell_of(k);
      scale_reg = seen >> k & 1 ? (threadIdx.x < 4 ? a.k_scales[cell] : a.v_scales[cell]) : 0.0f;
    }
  };
  auto store_codes = [&](int b) {
#pragma unroll
    for (int q = 0; q < kChunks; ++q) {
      const int n = q * 256 + static_cast<int>(threadIdx.x);
      const int t8 = n & 7, chunk = (n >> 3) % kSteps, grp = (n >> 3) / kSteps;
      f16x8 f[2];
      codes_to_f16(k_reg[q], f);
      f16x8* to = &s_k[b][((grp >> 2) * kSteps + chunk) * kWave + 8 * (grp & 3) + t8];
      to[0] = f[0];
      to[32] = f[1];
    }
#pragma unroll
    for (int q = 0; q < kChunks; ++q) {
      const int d = q * kWave + lane;
      f16x8 f[2];
      codes_to_f16(v_reg[q], f);
      f16x8* to = &s_v[b][(((d >> 5) * 2 + (wave >> 1)) * 2) * kWave + (d & 31) + 32 * (wave & 1)];
      to[0] = f[0];
      to[kWave] = f[1];
    }
    if (threadIdx.x < 8) s_scale[b][threadIdx.x >> 2][threadIdx.x & 3] = scale_reg;
  };

  // ---- the wave's columns
  const int col = 32 * wave + c;
  const bool mine = col < cols;
  const int token = mine ? col / a.group : item->tokens - 1;
  const int q_head = g * a.group + (mine ? col - token * a.group : 0);
  const int pos = first_pos + token;
  const int seen_from = a.window > 0 ? max(0, pos + 1 - a.window) : 0;
  // the wave's first and last token: what all and what any of its columns see
  const int wave_first = first_pos + min(32 * wave, cols - 1) / a.group;
  const int wave_last = first_pos + min(32 * wave + 31, cols - 1) / a.group;
  const int all_from = a.window > 0 ? max(0, wave_last + 1 - a.window) : 0;
  const int any_from = a.window > 0 ? max(0, wave_first + 1 - a.window) : 0;
  const bool busy = 32 * wave < cols;

  if (tile_lo < tile_hi) load_codes(tile_lo);
  f16x8 q[State::kTerms][kSteps];
  float col_scale;
  {
    const typename T::store* from = static_cast<const typename T::store*>(a.q) +
                                    static_cast<int64_t>(min(item->row + token, a.tokens - 1)) *
                                        a.q_token_stride +
                                    static_cast<int64_t>(q_head) * a.q_head_stride + 8 * h;
    float x[kSteps][8];
    float top = 0.0f;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      load8<T>(from + 16 * s, x[s]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[s][e] = mine ? x[s][e] : 0.0f;
        top = fmaxf(top, fabsf(x[s][e]));
      }
    }
    top = fmaxf(top, __shfl_xor(top, 32));
    col_scale = split_query<T, kSteps>(x, top, a.scale * kLog2e, q);
  }

  f32x16 o[kTilesD], rest[State::kApart ? kTilesD : 1];
#pragma unroll
  for (int d = 0; d < kTilesD; ++d) {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      o[d][e] = 0.0f;
      if constexpr (State::kApart) rest[d][e] = 0.0f;
    }
  }
  float m = -INFINITY, l = 0.0f, v_ref = 0.0f, v_inv = 0.0f;

  int seen = 0;
  if (tile_lo < tile_hi) {
    store_codes(0);
    seen = seen_reg;
    if (tile_lo + 1 < tile_hi) load_codes(tile_lo + 1);
  }
  for (int tile = tile_lo; tile < tile_hi; ++tile) {
    const int b = (tile - tile_lo) & 1;
    __syncthreads();  // the tile is in LDS; the other buffer is read
    const int seen_now = seen;
    if (tile + 1 < tile_hi) {
      store_codes(b ^ 1);
      seen = seen_reg;
      if (tile + 2 < tile_hi) load_codes(tile + 2);
    }
    const int key0 = tile * kTile;
    if (!busy || key0 > wave_last || key0 + kTile - 1 < any_from || seen_now == 0) continue;

    f32x16 s[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[r][e] = 0.0f;
    }
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const f16x8 f = s_k[b][(r * kSteps + k) * kWave + lane];
#pragma unroll
        for (int e = 0; e < State::kTerms; ++e) {
          s[r] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f, q[e][k], s[r], 0, 0, 0);
        }
      }
    }

    // scales of keys 16 h .. 16 h + 15 of the row tiles
    float kscale[2], vscale[2], top[2], v_top[2], mul[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      kscale[r] = s_scale[b][0][2 * r + h] * col_scale;
      vscale[r] = s_scale[b][1][2 * r + h];
    }
    const bool whole = key0 >= all_from && key0 + kTile - 1 <= wave_first && seen_now == 15;
    if (whole && __all(!(kscale[0] < 0.0f || kscale[1] < 0.0f))) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        top[r] = s[r][0];
#pragma unroll
        for (int e = 1; e < 16; ++e) top[r] = fmaxf(top[r], s[r][e]);
        top[r] *= kscale[r];
        v_top[r] = vscale[r];
        mul[r] = kscale[r];
      }
    } else {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int key = key0 + 32 * r + 16 * h;
        const bool some = (seen_now >> (2 * r + h) & 1) && key <= pos && key + 15 >= seen_from;
        top[r] = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int k = key + e;
          s[r][e] = some && k <= pos && k >= seen_from ? s[r][e] * kscale[r] : -INFINITY;
          top[r] = fmaxf(top[r], s[r][e]);
        }
        v_top[r] = some ? vscale[r] : 0.0f;
        mul[r] = 1.0f;
      }
    }
    const float t_top = fmaxf(top[0], top[1]);
    const float t_v =
        fmaxf(v_top[0] <= 3.0e38f ? v_top[0] : 0.0f, v_top[1] <= 3.0e38f ? v_top[1] : 0.0f);
    if (__any(t_top > m + State::kRescale || t_v > v_ref)) {
      float m2 = fmaxf(m, t_top);
      m2 = fmaxf(m2, __shfl_xor(m2, 32));
      float v2 = fmaxf(v_ref, t_v);
      v2 = fmaxf(v2, __shfl_xor(v2, 32));
      const float ref = v2 > v_ref ? power_above(v2) : v_ref;
      const float keep = m2 == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - m2);
      const float keep_o = ref > 0.0f ? keep * (v_ref / ref) : 1.0f;
      l *= keep;
#pragma unroll
      for (int d = 0; d < kTilesD; ++d) {
        o[d] *= keep_o;
        if constexpr (State::kApart) rest[d] *= keep_o;
      }
      m = m2;
      v_ref = ref;
      v_inv = ref > 0.0f ? 1.0f / ref : 0.0f;
    }
    const float shift = weight_bias(T::code) - (m == -INFINITY ? 0.0f : m);
    const float v_factor[2] = {vscale[0] * v_inv, vscale[1] * v_inv};
    f16x8 w[2][2], w_rest[2][2];
    auto weights = [&](auto some_hidden) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float p[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float sc = s[r][8 * k + e];
            p[e] = __builtin_amdgcn_exp2f(fmaf(sc, mul[r], shift));
            float v = p[e] * v_factor[r];
            if constexpr (decltype(some_hidden)::value) v = sc == -INFINITY ? 0.0f : v;
            w[r][k][e] = static_cast<_Float16>(v);
            if constexpr (State::kRest) {
              w_rest[r][k][e] =
                  static_cast<_Float16>((v - static_cast<float>(w[r][k][e])) * State::kRestScale);
            }
          }
          l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
        }
      }
    };
    if (!whole && __any(!(fabsf(v_factor[0]) <= 3.0e38f && fabsf(v_factor[1]) <= 3.0e38f))) {
      weights(std::true_type{});
    } else {
      weights(std::false_type{});
    }

#pragma unroll
    for (int r = 0; r < 2; ++r) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int d = 0; d < kTilesD; ++d) {
          const f16x8 f = s_v[b][((d * 2 + r) * 2 + k) * kWave + lane];
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f, w[r][k], o[d], 0, 0, 0);
          if constexpr (State::kRest) {
            f32x16& to = State::kApart ? rest[d] : o[d];
            to = __builtin_amdgcn_mfma_f32_32x32x16_f16(f, w_rest[r][k], to, 0, 0, 0);
          }
        }
      }
    }
  }

  if (!busy) return;
  l += __shfl_xor(l, 32);
  if (!mine) return;
  const int part = item->part;
  float* to = a.parts + (static_cast<size_t>(g) * a.cap_parts + max(0, part)) * wide_part_floats(D);
#pragma unroll
  for (int d = 0; d < kTilesD; ++d) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = o[d][4 * k + e];
        if constexpr (State::kApart) v[e] += rest[d][4 * k + e] * (1.0f / State::kRestScale);
        v[e] *= v_ref;
      }
      const int at = 32 * d + 8 * k + 4 * h;
      if (part < 0) finish4<T>(a, item->row + token, q_head, at, v, m, l);
      else *reinterpret_cast<f32x4*>(to + col * D + at) = v;
    }
  }
  if (part >= 0 && h == 0) {
    to[kWideCols * D + col] = m;
    to[kWideCols * (D + 1) + col] = l;
  }
}

// Joins the parts of cut units: a block per kv head, unit and 16 columns.
template <class T, int D>
__global__ __launch_bounds__(256) void join_wide_kernel(AttendArgs a) {
  constexpr int kVecs = D / 4, kGroups = 256 / kVecs;
  const int g = blockIdx.x;
  const SchedHead* head = reinterpret_cast<const SchedHead*>(a.work);
  if (static_cast<int>(blockIdx.y) >= head->joins) return;
  const WideJoin j = reinterpret_cast<const WideJoin*>(a.work + a.at_joins)[blockIdx.y];
  const int cols = j.tokens * a.group, d = threadIdx.x % kVecs * 4;
  const float* from =
      a.parts + (static_cast<size_t>(g) * a.cap_parts + j.part) * wide_part_floats(D);
  const int stop = min(cols, static_cast<int>(blockIdx.z + 1) * 16);
  for (int c = blockIdx.z * 16 + threadIdx.x / kVecs; c < stop; c += kGroups) {
    float m = -INFINITY;
    for (int p = 0; p < j.parts; ++p) {
      m = fmaxf(m, from[static_cast<size_t>(p) * wide_part_floats(D) + kWideCols * D + c]);
    }
    f32x4 o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float l = 0.0f;
#pragma unroll 4
    for (int p = 0; p < j.parts; ++p) {
      const float* q = from + static_cast<size_t>(p) * wide_part_floats(D);
      const float pm = q[kWideCols * D + c], pl = q[kWideCols * (D + 1) + c];
      const f32x4 po = *reinterpret_cast<const f32x4*>(q + c * D + d);
      const float f = pm == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(pm - m);
      o += po * f;
      l += pl * f;
    }
    finish4<T>(a, j.row + c / a.group, g * a.group + c % a.group, d, o, m, l);
  }
}

}  // namespace kv
}  // namespace grm
