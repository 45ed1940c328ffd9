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

#include <type_traits>

#include "kv_narrow.hpp"

namespace grm {
namespace kv {


// Columns of a wavefront.  32 read a tile half as often from LDS as 16; 16
// need half the registers, and are taken where 32 would fill more than a
// half of a SIMD's, with one wavefront that nothing covers (attend of 1021
// tokens on 14011, head_dim 256 in fp16: OLD us with 32, NEW with 16).
__host__ __device__ constexpr int wide_wave_cols(int dtype, int head_dim) {
  return head_dim == 256 || (dtype == kF32 && head_dim == 128) ? 16 : 32;
}

__host__ __device__ constexpr int wide_threads(int dtype, int head_dim) {
  return kWideCols / wide_wave_cols(dtype, head_dim) * kWave;
}

// Floats of one partial result: 128 columns, and their maxima and sums.
__host__ __device__ constexpr int wide_part_floats(int head_dim) {
  return kWideCols * (head_dim + 2);
}

// Scales of 16 tokens, 0 where they have no block or none of the item's
// columns sees them.
struct __align__(16) GroupScale {
  float k, v;
  int there, pad;
};

// A value joined over the lanes of a column.
template <int W, class F>
__device__ inline float across(float v, F join) {
#pragma unroll
  for (int by = W; by < kWave; by *= 2) v = join(v, __shfl_xor(v, by));
  return v;
}

__device__ inline f32x16 wide_mul(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ inline f32x4 wide_mul(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// The order of a product's reads from LDS and matrix instructions (MULS for
// each of READS reads): reads run kAhead before what needs them.
template <int READS, int MULS>
__device__ inline void feed() {
  constexpr int kAhead = 6, kMul = 0x8, kRead = 0x100;
  __builtin_amdgcn_sched_group_barrier(kRead, kAhead, 0);
#pragma unroll
  for (int i = 0; i < READS; ++i) {
    __builtin_amdgcn_sched_group_barrier(kMul, MULS, 0);
    if (i + kAhead < READS) __builtin_amdgcn_sched_group_barrier(kRead, 1, 0);
  }
}

template <class T, int D>
__global__ __launch_bounds__(wide_threads(T::code, D), 2) void attend_wide_kernel(AttendArgs a) {
  typedef NarrowState<T, D> State;  // its constants: terms and allowances
  constexpr int W = wide_wave_cols(T::code, D);
  constexpr int kWaves = kWideCols / W, kLanes = kWave / W;  // lanes of a column
  constexpr int kStepD = 8 * kLanes, kSteps = D / kStepD;    // of the first product
  constexpr int kTilesD = D / W;                             // value row tiles
  constexpr int kLoads = 16 * D * 4 / (kWaves * kWave * 16);  // 16 bytes of keys to a lane
  constexpr int kPer = W / 2, kHalves = 32 / W;  // scores, accumulators of 32 keys to a lane
  constexpr int kAcc = W * W / kWave;
  typedef typename std::conditional<W == 32, f32x16, f32x4>::type Acc;
  const int g = blockIdx.x;
  const auto* head = reinterpret_cast<ConstHead>(reinterpret_cast<uintptr_t>(a.work));
  if (static_cast<int>(blockIdx.y) >= head->items) return;
  const auto* item = reinterpret_cast<ConstItem>(reinterpret_cast<uintptr_t>(a.work) + a.at_items) +
                     blockIdx.y;
  if (item->tokens <= 0) return;
  const int lane = __lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int c = lane % W, h = lane / W;
  const int tile_lo = item->tile_lo, tile_hi = item->tile_hi;
  const int first_pos = item->pos, last_pos = first_pos + item->tokens - 1;
  const int cols = item->tokens * a.group;
  const size_t table_row = static_cast<size_t>(item->request) * a.width;
  const int bs = 1 << a.block_log2;
  const uint32_t cell_bytes = static_cast<uint32_t>(bs * D);

  // a lane's eight values of the instruction's operand
  __shared__ f16x8 s_k[2][2 * kHalves * kSteps * kWave];  // [row tile][step][lane]
  __shared__ f16x8 s_v[2][kTilesD * 2 * kPer / 8 * kWave];  // [d tile][32 keys][lane]
  __shared__ GroupScale s_scale[2][4];                      // of a group of 16 tokens

  // ---- codes of a tile to registers: a wavefront (or two) loads 16 of its
  // tokens, which lie in one block, so that addresses are a scalar base and a
  // lane's fixed offset.  The block's id is loaded a tile ahead.
  const int grp = wave * 4 / kWaves, part_of = wave % (kWaves / 4);
  u32x4 k_reg[kLoads], v_reg[kLoads];
  float k_scale_reg, v_scale_reg;
  int raw_id, there_reg;
  const int first_seen = a.window > 0 ? max(0, first_pos + 1 - a.window) : 0;
  // Keys: 8 tokens by 8 chunks of 16 values to a load (of 32 columns and
  // head_dim 64, 16 tokens by 4); with two wavefronts the second has the
  // tokens of the other row tile.
  constexpr int kChunks = D / 16;
  const int token = W == 32 ? (lane & 7) + (lane >> 3) / kChunks * 8
                            : (lane & 3) + 2 * (lane & 4) + 4 * part_of;
  const uint32_t k_at = static_cast<uint32_t>(token * D + (lane >> 3) % kChunks * 16);
  const uint32_t v_at = static_cast<uint32_t>((part_of * (D / 2) + lane) * bs);
  auto load_id = [&](int tile) {
    const int at = (tile * kTile + 16 * grp) >> a.block_log2;
    raw_id = a.table[table_row + max(0, min(at, a.width - 1))];
  };
  auto load_codes = [&](int tile) {
    const int key = tile * kTile + 16 * grp;
    const int raw = __builtin_amdgcn_readfirstlane(raw_id);
    const bool there = key <= last_pos && key + 15 >= first_seen &&
                       (key >> a.block_log2) < a.width && static_cast<uint32_t>(raw) < a.blocks;
    const uint32_t cell = static_cast<uint32_t>(there ? raw : 0) * a.kv_heads + g;
    const uint64_t base = static_cast<uint64_t>(cell) * cell_bytes;
    const int place = key & (bs - 1);
    const int8_t* k_base = a.k_codes + base + place * D;
    const int8_t* v_base = a.v_codes + base + place;
#pragma unroll
    for (int q = 0; q < kLoads; ++q) {
      const int chunk = 8 * q % kChunks, token8 = 8 * q / kChunks;
      k_reg[q] = *reinterpret_cast<const u32x4*>(k_base + chunk * 16 + token8 * 8 * D + k_at);
    }
#pragma unroll
    for (int q = 0; q < kLoads; ++q) {
      v_reg[q] = *reinterpret_cast<const u32x4*>(v_base + q * kWave * bs + v_at);
    }
    k_scale_reg = a.k_scales[cell];
    v_scale_reg = a.v_scales[cell];
    there_reg = there ? 1 : 0;
  };
  // Eight lanes write rows of eight different bank groups: with 32 columns
  // their rows have one bit 2, which rows of odd eights therefore turn over.
  const int k_slot = W == 32
                         ? 8 * (lane >> 2 & 1) + 4 * ((wave ^ lane >> 2) & 1) + (lane & 3)
                         : 8 * (grp & 1) + (lane & 7);
  const int k_read = W == 32 ? 32 * h + (c ^ (c >> 3 & 1) << 2) : lane;
  auto store_codes = [&](int b) {
#pragma unroll
    for (int q = 0; q < kLoads; ++q) {
      const int at = 8 * q + (lane >> 3), chunk = at % kChunks, token8 = at / kChunks;
      f16x8 f[2];
      codes_to_f16(k_reg[q], f);
      const int row_tile = W == 32 ? grp >> 1 : 2 * (grp >> 1) + part_of;
      const int step = chunk * 16 / kStepD, half = chunk * 16 % kStepD / 8;
      f16x8* to = &s_k[b][(row_tile * kSteps + step) * kWave + half * W +
                          (W == 32 ? 16 * token8 : 0) + k_slot];
      to[0] = f[0];
      to[W] = f[1];
    }
#pragma unroll
    for (int q = 0; q < kLoads; ++q) {
      const int d = part_of * (D / 2) + q * kWave + lane;
      f16x8 f[2];
      codes_to_f16(v_reg[q], f);
      f16x8* to =
          W == 32 ? &s_v[b][((d / 32 * 2 + (grp >> 1)) * 2) * kWave + d % 32 + 32 * (grp & 1)]
                  : &s_v[b][(d / 16 * 2 + (grp >> 1)) * kWave + d % 16 + 32 * (grp & 1)];
      to[0] = f[0];
      to[W == 32 ? kWave : 16] = f[1];
    }
    if (part_of == 0 && lane == 0) {
      s_scale[b][grp] = {there_reg ? k_scale_reg : 0.0f, there_reg ? v_scale_reg : 0.0f,
                         there_reg, 0};
    }
  };

  // ---- the wave's columns
  const int col = W * wave + c;
  const bool mine = col < cols;
  const int row = mine ? col / a.group : item->tokens - 1;
  const int q_head = g * a.group + (mine ? col - row * a.group : 0);
  const int pos = first_pos + row;
  const int seen_from = a.window > 0 ? max(0, pos + 1 - a.window) : 0;
  // the wave's first and last token: what all and what any of its columns see
  const int wave_first = first_pos + min(W * wave, cols - 1) / a.group;
  const int wave_last = first_pos + min(W * wave + W - 1, cols - 1) / a.group;
  const int all_from = a.window > 0 ? max(0, wave_last + 1 - a.window) : 0;
  const int any_from = a.window > 0 ? max(0, wave_first + 1 - a.window) : 0;
  const bool busy = W * wave < cols;

  const int tile_last = tile_hi - 1;
  if (tile_lo < tile_hi) {
    load_id(tile_lo);
    load_codes(tile_lo);
    load_id(min(tile_lo + 1, tile_last));
  }
  f16x8 q[State::kTerms][kSteps];
  float col_scale;
  {
    const typename T::store* from = static_cast<const typename T::store*>(a.q) +
                                    static_cast<int64_t>(min(item->row + row, a.tokens - 1)) *
                                        a.q_token_stride +
                                    static_cast<int64_t>(q_head) * a.q_head_stride + 8 * h;
    float x[kSteps][8];
    float top = 0.0f;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      load8<T>(from + kStepD * s, x[s]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[s][e] = mine ? x[s][e] : 0.0f;
        top = fmaxf(top, fabsf(x[s][e]));
      }
    }
    top = across<W>(top, [](float x, float y) { return fmaxf(x, y); });
    col_scale = split_query<T, kSteps>(x, top, a.scale * kLog2e, q);
  }

  Acc o[kTilesD], rest[State::kApart ? kTilesD : 1];
#pragma unroll
  for (int d = 0; d < kTilesD; ++d) {
#pragma unroll
    for (int e = 0; e < kAcc; ++e) {
      o[d][e] = 0.0f;
      if constexpr (State::kApart) rest[d][e] = 0.0f;
    }
  }
  float m = -INFINITY, l = 0.0f, v_ref = 0.0f, v_inv = 0.0f;

  if (tile_lo < tile_hi) {
    store_codes(0);
    load_codes(min(tile_lo + 1, tile_last));
    load_id(min(tile_lo + 2, tile_last));
  }
  for (int tile = tile_lo; tile < tile_hi; ++tile) {
    const int b = (tile - tile_lo) & 1;
    __syncthreads();  // the tile is in LDS; the other buffer is read
    Acc s[2][kHalves];  // of 32 keys each
#pragma unroll
    for (int r = 0; r < 2 * kHalves; ++r) {
#pragma unroll
      for (int e = 0; e < kAcc; ++e) s[r / kHalves][r % kHalves][e] = 0.0f;
    }
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
#pragma unroll
      for (int r = 0; r < 2 * kHalves; ++r) {
        const f16x8 f = s_k[b][(r * kSteps + k) * kWave + k_read];
        Acc& to = s[r / kHalves][r % kHalves];
#pragma unroll
        for (int e = 0; e < State::kTerms; ++e) to = wide_mul(f, q[e][k], to);
      }
    }
    feed<2 * kHalves * kSteps, State::kTerms>();
    auto score = [&](int r, int e) { return s[r][e / kAcc][e % kAcc]; };
    store_codes(b ^ 1);  // past the last tile: what nobody reads
    load_codes(min(tile + 2, tile_last));
    load_id(min(tile + 3, tile_last));
    const GroupScale of[2] = {s_scale[b][h * kPer / 16], s_scale[b][2 + h * kPer / 16]};
    const int seen_0 = s_scale[b][0].there, seen_1 = s_scale[b][1].there;
    const int seen_2 = s_scale[b][2].there, seen_3 = s_scale[b][3].there;
    const int seen_now =
        __builtin_amdgcn_readfirstlane(seen_0 | seen_1 << 1 | seen_2 << 2 | seen_3 << 3);
    const int key0 = tile * kTile;
    if (!busy || key0 > wave_last || key0 + kTile - 1 < any_from || seen_now == 0) continue;

    // a lane's keys: kPer neighbours of either 32, which share their scales
    float kscale[2], vscale[2], top[2], v_top[2], mul[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      kscale[r] = of[r].k * col_scale;
      vscale[r] = of[r].v;
    }
    const bool whole = key0 >= all_from && key0 + kTile - 1 <= wave_first && seen_now == 15;
    if (whole && __all(!(kscale[0] < 0.0f || kscale[1] < 0.0f))) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        top[r] = score(r, 0);
#pragma unroll
        for (int e = 1; e < kPer; ++e) top[r] = fmaxf(top[r], score(r, e));
        top[r] *= kscale[r];
        v_top[r] = vscale[r];
        mul[r] = kscale[r];
      }
    } else {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int key = key0 + 32 * r + kPer * h;
        const bool some = of[r].there && key <= pos && key + kPer - 1 >= seen_from;
        top[r] = -INFINITY;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          const int k = key + e;
          const float sc = some && k <= pos && k >= seen_from ? score(r, e) * kscale[r] : -INFINITY;
          s[r][e / kAcc][e % kAcc] = sc;
          top[r] = fmaxf(top[r], sc);
        }
        v_top[r] = some ? vscale[r] : 0.0f;
        mul[r] = 1.0f;
      }
    }
    const float t_top = fmaxf(top[0], top[1]);
    const float t_v =
        fmaxf(v_top[0] <= 3.0e38f ? v_top[0] : 0.0f, v_top[1] <= 3.0e38f ? v_top[1] : 0.0f);
    if (__any(t_top > m + State::kRescale || t_v > v_ref)) {
      const auto larger = [](float x, float y) { return fmaxf(x, y); };
      const float m2 = across<W>(fmaxf(m, t_top), larger);
      const float v2 = across<W>(fmaxf(v_ref, t_v), larger);
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
    f16x8 w[2][kPer / 8], w_rest[2][kPer / 8];
    auto weights = [&](auto some_hidden) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
#pragma unroll
        for (int k = 0; k < kPer / 8; ++k) {
          float p[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float sc = score(r, 8 * k + e);
            p[e] = __builtin_amdgcn_exp2f(fmaf(sc, mul[r], shift));
            float v = p[e] * v_factor[r];
            if constexpr (decltype(some_hidden)::value) v = sc == -INFINITY ? 0.0f : v;
            if constexpr (State::kRest) v = as_rounded(v);
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
      for (int k = 0; k < kPer / 8; ++k) {
#pragma unroll
        for (int d = 0; d < kTilesD; ++d) {
          const f16x8 f = s_v[b][((d * 2 + r) * (kPer / 8) + k) * kWave + lane];
          o[d] = wide_mul(f, w[r][k], o[d]);
          if constexpr (State::kRest) {
            Acc& to = State::kApart ? rest[d] : o[d];
            to = wide_mul(f, w_rest[r][k], to);
          }
        }
      }
    }
    feed<2 * kPer / 8 * kTilesD, State::kRest ? 2 : 1>();
  }

  if (!busy) return;
  l = across<W>(l, [](float x, float y) { return x + y; });
  if (!mine) return;
  const int part = item->part;
  float* to = a.parts + (static_cast<size_t>(g) * a.cap_parts + max(0, part)) * wide_part_floats(D);
#pragma unroll
  for (int d = 0; d < kTilesD; ++d) {
#pragma unroll
    for (int k = 0; k < kAcc / 4; ++k) {
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = o[d][4 * k + e];
        if constexpr (State::kApart) v[e] += rest[d][4 * k + e] * (1.0f / State::kRestScale);
        v[e] *= v_ref;
      }
      const int at = W * d + 4 * kLanes * k + 4 * h;
      if (part < 0) finish4<T>(a, item->row + row, q_head, at, v, m, l);
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
