// kv_wide.hpp -- attention of requests that bring many tokens (prompts and
// chunks of prompts).
//
// An item is up to 128 (token, head) columns of one kv head against a range
// of key tiles (64 tokens).  A block turns each tile's codes into fp16 or bf16
// once: its wavefronts load the next tiles' codes to registers and write them to
// LDS as such (exact) in the order in which the matrix instructions take them (16
// bytes per lane, no bank conflicts); each multiplies the tile with its own
// columns.  Two LDS buffers, one barrier per tile.
//
// In a wavefront, vector work stands beside matrix work: the codes are turned
// between the instructions of the first product, and the tile's weights are
// made between those of the last tile's second product (values are stored a
// tile later than keys for that).  Two wavefronts share a SIMD.
//
// Bound by the vector unit and the matrix cores together.  Prompts of 333 to
// 4100 tokens (32 heads on 8, head_dim 128, bf16, 167 GFLOP and half as many
// again for the second term of the weights): a call of 283 us, 0.89 PFLOP/s with
// that term; the vector unit is busy for 66 % of the cycles and the matrix cores
// for 49 %.  A chunk of 1021 tokens on 14011 (16 heads on 4, head_dim 256, fp16,
// 243 GFLOP and half as many again): 342 us; 41 % and 50 %.
//
// Layout of the products (W columns to a wavefront, lane = c + W h):
//   S^T = K Q^T, 32 columns (32x32x16): row 8 m + 4 h' + j of a 32-key row
//     tile is its key 16 h' + 4 m + j, so that a lane's 16 results are the
//     neighbouring keys 16 h .. 16 h + 15 of column c; 16 columns (16x16x32):
//     row 4 h' + j of 16-row tile r is key 8 h' + 4 r + j of 32 keys, and a
//     lane has keys 8 h .. 8 h + 7 of each 32;
//   O^T = V^T P^T: those are the lane's part of the B operand, 8 keys to an
//     instruction, and the A operand's lane holds the same keys of a value
//     column.
// The softmax is the narrow kernel's: one pass, scores and statistics in fp32,
// weights as two fp16 terms, or three bf16 ones.
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
// tokens on 14011, head_dim 256 in fp16: 865 us with 32, 488 with 16; at
// head_dim 128 32 columns are faster, four prompts in bf16 262 us against 328).
__host__ __device__ constexpr int wide_wave_cols(int dtype, int head_dim) {
  return head_dim == 256 || (dtype == kF32 && head_dim == 128) ? 16 : 32;
}

__host__ __device__ constexpr int wide_threads(int dtype, int head_dim) {
  return kWideCols / wide_wave_cols(dtype, head_dim) * kWave;
}

// Floats of one partial result: 128 columns, as in the narrow kernel's.
__host__ __device__ constexpr int wide_part_floats(int head_dim) {
  return kWideCols * (head_dim + 3);
}

// Scales of 16 tokens, 0 where they have no block or none of the item's
// columns sees them.
struct __align__(16) GroupScale {
  float k, v;
  int there, pad;
};

constexpr float kLargest = 3.0e38f;  // below are numbers

// A value joined over the lanes of a column.
template <int W, class F>
__device__ inline float across(float v, F join) {
#pragma unroll
  for (int by = W; by < kWave; by *= 2) v = join(v, __shfl_xor(v, by));
  return v;
}

// A product's reads from LDS and what is done with each, in this order: reads
// run kAhead before their use, and what `use` does beside the matrix
// instruction stays beside it.
template <int READS, class Read, class Use>
__device__ inline void in_step(Read read, Use use) {
  constexpr int kAhead = 4;
  u32x4 f[READS];
#pragma unroll
  for (int i = 0; i < kAhead && i < READS; ++i) f[i] = read(i);
#pragma unroll
  for (int i = 0; i < READS; ++i) {
    if (i + kAhead < READS) f[i + kAhead] = read(i + kAhead);
    use(i, f);
    if (i % 2) __builtin_amdgcn_sched_barrier(0);  // two at a time
  }
}

template <class T, int D>
struct WideShape {
  typedef NarrowState<T, D> State;  // its constants: terms and allowances
  static constexpr int W = wide_wave_cols(T::code, D);
  static constexpr int kWaves = kWideCols / W, kLanes = kWave / W;  // lanes of a column
  static constexpr int kStepD = 8 * kLanes, kSteps = D / kStepD;    // of the first product
  static constexpr int kTilesD = D / W;                             // value row tiles
  static constexpr int kLoads = 16 * D * 4 / (kWaves * kWave * 16);  // 16 bytes of keys to a lane
  static constexpr int kPer = W / 2, kHalves = 32 / W;  // scores, accumulators of 32 keys to a lane
  static constexpr int kAcc = W * W / kWave;
  typedef typename std::conditional<W == 32, f32x16, f32x4>::type Acc;

  // a lane's eight values of an instruction's operand
  u32x4 k[2][2 * kHalves * kSteps * kWave];       // [row tile][step][lane]
  u32x4 v[2][kTilesD * 2 * kPer / 8 * kWave];     // [d tile][32 keys][lane]
  GroupScale scale[2][4];                         // of a group of 16 tokens
};

// One item's tiles up to tile_hi, which may be the next item's.
template <class T, int D>
__device__ inline void wide_item(const AttendArgs& a, ConstItem item, int tile_hi,
                                 int g, WideShape<T, D>& lds) {
  typedef WideShape<T, D> S;
  typedef typename S::State State;
  typedef typename S::Acc Acc;
  constexpr int W = S::W, kWaves = S::kWaves, kLanes = S::kLanes, kStepD = S::kStepD;
  constexpr int kSteps = S::kSteps, kTilesD = S::kTilesD, kLoads = S::kLoads;
  constexpr int kPer = S::kPer, kHalves = S::kHalves, kAcc = S::kAcc;
  auto& s_k = lds.k;
  auto& s_v = lds.v;
  auto& s_scale = lds.scale;
  const int lane = __lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int c = lane % W, h = lane / W;
  const int tile_lo = item->tile_lo;
  const int first_pos = item->pos, last_pos = first_pos + item->tokens - 1;
  const int cols = item->tokens * a.group;
  const size_t table_row = static_cast<size_t>(item->request) * a.width;
  const int bs = 1 << a.block_log2;
  const uint32_t cell_bytes = static_cast<uint32_t>(bs * D);

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
  int32_t v_cell = 0, v_place = 0;
  auto load_keys = [&](int tile) {
    const int key = tile * kTile + 16 * grp;
    const int raw = __builtin_amdgcn_readfirstlane(raw_id);
    const bool there = key <= last_pos && key + 15 >= first_seen &&
                       (key >> a.block_log2) < a.width && static_cast<uint32_t>(raw) < a.blocks;
    const uint32_t cell = static_cast<uint32_t>(there ? raw : 0) * a.kv_heads + g;
    const int place = key & (bs - 1);
    const int8_t* k_base = a.k_codes + static_cast<uint64_t>(cell) * cell_bytes + place * D;
#pragma unroll
    for (int q = 0; q < kLoads; ++q) {
      const int chunk = 8 * q % kChunks, token8 = 8 * q / kChunks;
      k_reg[q] = *reinterpret_cast<const u32x4*>(k_base + chunk * 16 + token8 * 8 * D + k_at);
    }
    k_scale_reg = a.k_scales[cell];
    v_scale_reg = a.v_scales[cell];
    there_reg = there ? 1 : 0;
    v_cell = cell;
    v_place = place;
  };
  auto load_values = [&]() {  // of the tile whose keys were loaded last
    const int8_t* v_base = a.v_codes + static_cast<uint64_t>(static_cast<uint32_t>(v_cell)) * cell_bytes + v_place;
#pragma unroll
    for (int q = 0; q < kLoads; ++q) {
      v_reg[q] = *reinterpret_cast<const u32x4*>(v_base + q * kWave * bs + v_at);
    }
  };
  // Eight lanes write rows of eight different bank groups: with 32 columns
  // their rows have one bit 2, which rows of odd eights therefore turn over.
  const int k_slot = W == 32
                         ? 8 * (lane >> 2 & 1) + 4 * ((wave ^ lane >> 2) & 1) + (lane & 3)
                         : 8 * (grp & 1) + (lane & 7);
  const int k_read = W == 32 ? 32 * h + (c ^ (c >> 3 & 1) << 2) : lane;
  // Half a register's codes at a time, so that the products' instructions have
  // something beside each: kPieces of a tile's keys and the one's before values.
  constexpr int kPieces = 4 * kLoads;
  auto store_piece = [&](int piece, int b) {
    const int q = piece / 2 % kLoads, half = piece % 2;
    if (piece < 2 * kLoads) {
      const int at = 8 * q + (lane >> 3), chunk = at % kChunks, token8 = at / kChunks;
      const int row_tile = W == 32 ? grp >> 1 : 2 * (grp >> 1) + part_of;
      const int step = chunk * 16 / kStepD, first = chunk * 16 % kStepD / 8;
      s_k[b ^ 1][(row_tile * kSteps + step) * kWave + (first + half) * W +
                 (W == 32 ? 16 * token8 : 0) + k_slot] =
          codes_as<query_bf16<T>()>(k_reg[q][2 * half], k_reg[q][2 * half + 1]);
    } else {
      const int d = part_of * (D / 2) + q * kWave + lane;
      const int at =
          W == 32 ? ((d / 32 * 2 + (grp >> 1)) * 2 + half) * kWave + d % 32 + 32 * (grp & 1)
                  : (d / 16 * 2 + (grp >> 1)) * kWave + d % 16 + 32 * (grp & 1) + 16 * half;
      s_v[b][at] = codes_as<weight_bf16<T>()>(v_reg[q][2 * half], v_reg[q][2 * half + 1]);
    }
  };
  auto store_scales = [&](int b) {
    if (part_of == 0 && lane == 0) {
      s_scale[b][grp] = {there_reg ? k_scale_reg : 0.0f, there_reg ? v_scale_reg : 0.0f, there_reg,
                         0};
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
  const bool busy = W * wave < cols;

  const int tile_last = tile_hi - 1;
  if (tile_lo < tile_hi) {
    load_id(tile_lo);
    load_keys(tile_lo);
    load_values();
    load_id(min(tile_lo + 1, tile_last));
  }
  u32x4 q[State::kTerms][kSteps];
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
  float m = -INFINITY, l = 0.0f, v_ref = 0.0f, v_inv = 0.0f, poison = 0.0f;
  // The sums of the tiles so far take a change of the references with them
  // when the next tile's scores are there: then their products are done.
  bool moves = false;
  float keep_o = 1.0f;
  auto rescale = [&]() {
    if (moves) {
#pragma unroll
      for (int d = 0; d < kTilesD; ++d) {
        o[d] *= keep_o;
        if constexpr (State::kApart) rest[d] *= keep_o;
      }
    }
  };

  auto next_codes = [&](int tile) {
    load_values();
    load_keys(min(tile + 2, tile_last));
    load_id(min(tile + 3, tile_last));
  };
  if (tile_lo < tile_hi) {
    // the values go where the first product, with weights of 0, reads them
#pragma unroll
    for (int piece = 0; piece < kPieces; ++piece) store_piece(piece, 1);
    store_scales(0);
    load_keys(min(tile_lo + 1, tile_last));
    load_id(min(tile_lo + 2, tile_last));
  }
  // kept as halves: as words they spill more (fp16, head_dim 128: 35 registers
  // against 14, prompts in 307 us against 243)
  f16x8 w[State::kWeights][2][kPer / 8] = {};
  // Weights of a tile times its values.
  constexpr int kValueReads = 2 * kPer / 8 * kTilesD;
  auto multiply = [&](int b, auto beside) {
    in_step<kValueReads>([&](int i) { return s_v[b][(i % kTilesD * 2 * (kPer / 8) + i / kTilesD) * kWave + lane]; },
        [&](int i, const u32x4(&f)[kValueReads]) {
          const int d = i % kTilesD, rk = i / kTilesD;
#pragma unroll
          for (int n = 0; n < State::kWeights; ++n) {
            Acc& to = n && State::kApart ? rest[d] : o[d];
            to = mfma<weight_bf16<T>()>(
                f[i], __builtin_bit_cast(u32x4, w[n][rk / (kPer / 8)][rk % (kPer / 8)]), to);
          }
          beside(i);
        });
  };

  if (!busy) {  // loads its share of the codes
    for (int tile = tile_lo; tile < tile_hi; ++tile) {
      const int b = (tile - tile_lo) & 1;
      __syncthreads();
#pragma unroll
      for (int piece = 0; piece < kPieces; ++piece) store_piece(piece, b);
      store_scales(b ^ 1);
      next_codes(tile);
    }
    __syncthreads();
    return;
  }
  for (int tile = tile_lo; tile < tile_hi; ++tile) {
    const int b = (tile - tile_lo) & 1;
    __syncthreads();  // the tile is in LDS; the other buffer is read
    const GroupScale of[2] = {s_scale[b][h * kPer / 16], s_scale[b][2 + h * kPer / 16]};
    Acc s[2][kHalves];  // of 32 keys each
    constexpr bool kLesser = State::kTerms > 1;  // a query's lesser terms are summed apart
    Acc lesser[kLesser ? 2 * kHalves : 1];
#pragma unroll
    for (int r = 0; r < 2 * kHalves; ++r) {
#pragma unroll
      for (int e = 0; e < kAcc; ++e) {
        s[r / kHalves][r % kHalves][e] = 0.0f;
        if constexpr (kLesser) lesser[r][e] = 0.0f;
      }
    }
    constexpr int kKeyReads = 2 * kHalves * kSteps;
    in_step<kKeyReads>(
        [&](int i) {
          return s_k[b][(i % (2 * kHalves) * kSteps + i / (2 * kHalves)) * kWave + k_read];
        },
        [&](int i, const u32x4(&f)[kKeyReads]) {
          constexpr int kRows = 2 * kHalves;
#pragma unroll
          for (int e = 0; e < State::kTerms; ++e) {
            Acc& to = e ? lesser[i % kRows * kLesser] : s[i % kRows / kHalves][i % kHalves];
            to = mfma<query_bf16<T>()>(f[i], q[e][i / kRows], to);
          }
#pragma unroll
          for (int piece = i * kPieces / kKeyReads; piece < (i + 1) * kPieces / kKeyReads;
               ++piece) {
            store_piece(piece, b);  // past the last tile: what nobody reads
          }
        });
    store_scales(b ^ 1);
    next_codes(tile);
    if constexpr (kLesser) {
#pragma unroll
      for (int r = 0; r < 2 * kHalves; ++r) s[r / kHalves][r % kHalves] += lesser[r];
    }
    auto score = [&](int r, int e) { return s[r][e / kAcc][e % kAcc]; };
    const int key0 = tile * kTile;
    // a lane's keys: kPer neighbours of either 32, which share their scales
    float kscale[2], top[2], v_top[2], mul[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      kscale[r] = of[r].k * col_scale;
      v_top[r] = of[r].v;
    }
    const bool whole = key0 >= all_from && key0 + kTile - 1 <= wave_first;
    if (whole && __all(of[0].there && of[1].there && !(kscale[0] < 0.0f || kscale[1] < 0.0f))) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        top[r] = score(r, 0);
#pragma unroll
        for (int e = 1; e < kPer; ++e) top[r] = fmaxf(top[r], score(r, e));
        top[r] *= kscale[r];
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
        if (!some) v_top[r] = 0.0f;
        mul[r] = 1.0f;
      }
    }
    const float t_top = fmaxf(top[0], top[1]);
    const float t_v =
        fmaxf(v_top[0] <= kLargest ? v_top[0] : 0.0f, v_top[1] <= kLargest ? v_top[1] : 0.0f);
    rescale();
    moves = __any(t_top > m + State::kRescale || t_v > v_ref);
    if (moves) {
      const auto larger = [](float x, float y) { return fmaxf(x, y); };
      const float m2 = across<W>(fmaxf(m, t_top), larger);
      const float v2 = across<W>(fmaxf(v_ref, t_v), larger);
      const float ref = v2 > v_ref ? power_above(v2) : v_ref;
      const float keep = m2 == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - m2);
      keep_o = ref > 0.0f ? keep * (v_ref / ref) : 1.0f;
      l *= keep;
      m = m2;
      v_ref = ref;
      v_inv = ref > 0.0f ? 1.0f / ref : 0.0f;
    }
    const float shift = weight_bias(T::code) - (m == -INFINITY ? 0.0f : m);
    // A value scale that is no number makes its columns so at the end.  (As a
    // logarithm in the exponent a scale would cost a product less to a weight,
    // but its own rounding, which grows with its distance from 1.)
    float v_factor[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      poison += v_top[r] <= kLargest ? 0.0f : NAN;
      v_factor[r] = v_top[r] <= kLargest ? v_top[r] * v_inv : 0.0f;
    }
    // The last tile's product runs beside this tile's weights.
    u32x4 w2[State::kWeights][2][kPer / 8];
    float sum[2] = {0.0f, 0.0f};
    multiply(b ^ 1, [&](int i) {
      // two weights at a time, spread over the reads
      constexpr int kEvery = kValueReads > kPer ? kValueReads / kPer : 1;
      constexpr int kCount = kPer > kValueReads ? kPer / kValueReads : 1;
      if ((i + 1) % kEvery != 0) return;
#pragma unroll
      for (int u = 0; u < kCount; ++u) {
        const int j = ((i + 1) / kEvery - 1) * kCount + u, r = 2 * j / kPer;
        const int e = 2 * j % kPer;
        const float p[2] = {__builtin_amdgcn_exp2f(fmaf(score(r, e), mul[r], shift)),
                            __builtin_amdgcn_exp2f(fmaf(score(r, e + 1), mul[r], shift))};
        uint32_t t[State::kWeights];
        split_weights<T>(as_rounded(p[0] * v_factor[r]), as_rounded(p[1] * v_factor[r]), t);
#pragma unroll
        for (int n = 0; n < State::kWeights; ++n) w2[n][r][e / 8][e % 8 / 2] = t[n];
        sum[r] += p[0];
        sum[r] += p[1];
      }
    });
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l += sum[r];
#pragma unroll
      for (int k = 0; k < kPer / 8; ++k) {
#pragma unroll
        for (int n = 0; n < State::kWeights; ++n) w[n][r][k] = __builtin_bit_cast(f16x8, w2[n][r][k]);
      }
    }
  }
  __syncthreads();
  rescale();
  if (tile_lo < tile_hi) multiply((tile_last - tile_lo) & 1, [](int) {});

  const auto sum_of = [](float x, float y) { return x + y; };
  l = across<W>(l, sum_of);
  poison = across<W>(poison, sum_of);
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
        if constexpr (State::kApart) v[e] += rest[d][4 * k + e];
        v[e] += poison;
      }
      const int at = W * d + 4 * kLanes * k + 4 * h;
      if (part < 0) finish4<T>(a, item->row + row, q_head, at, v, m, l, v_ref);
      else *reinterpret_cast<f32x4*>(to + col * D + at) = v;
    }
  }
  if (part >= 0 && h == 0) {
    to[kWideCols * D + col] = m;
    to[kWideCols * (D + 1) + col] = l;
    to[kWideCols * (D + 2) + col] = v_ref;
    if (tile_hi != item->tile_hi) {  // the next item's part has nothing left
      to[wide_part_floats(D) + kWideCols * D + col] = -INFINITY;
      to[wide_part_floats(D) + kWideCols * (D + 1) + col] = 0.0f;
      to[wide_part_floats(D) + kWideCols * (D + 2) + col] = 0.0f;
    }
  }
}

// Items to a block.  The plan cuts for two blocks to a CU; where one fits, it
// takes two items, as one where they are neighbours of one unit.
__host__ __device__ constexpr int wide_items(int dtype, int head_dim) {
  return 32 / wide_wave_cols(dtype, head_dim);
}

template <class T, int D>
__global__ __launch_bounds__(wide_threads(T::code, D), 2) void attend_wide_kernel(AttendArgs a) {
  constexpr int kItems = wide_items(T::code, D);
  __shared__ WideShape<T, D> lds;
  const auto* head = reinterpret_cast<ConstHead>(reinterpret_cast<uintptr_t>(a.work));
  // in one dimension, which alone has room for millions of tokens
  const int g = static_cast<int>(blockIdx.x) % a.kv_heads;
  const int items = head->items, first = static_cast<int>(blockIdx.x) / a.kv_heads * kItems;
  for (int n = first; n < min(items, first + kItems); ++n) {
    const auto* item =
        reinterpret_cast<ConstItem>(reinterpret_cast<uintptr_t>(a.work) + a.at_items) + n;
    int tile_hi = item->tile_hi;
    const bool two = kItems == 2 && n == first && n + 1 < items && item->part >= 0 &&
                     item[1].part == item->part + 1 && item[1].row == item->row;
    if (two) tile_hi = item[1].tile_hi;
    if (n > first) __syncthreads();  // the item before has read its tiles
    if (item->tokens > 0) wide_item<T, D>(a, item, tile_hi, g, lds);
    if (two) break;
  }
}

// Joins the parts of cut units: four values of a column to a thread.
template <int D>
__host__ __device__ constexpr int join_wide_cols() {
  return 256 / (D / 4);
}

template <class T, int D>
__device__ inline void join_wide(const AttendArgs& a, const float* parts, int unit, int piece) {
  constexpr int kVecs = D / 4;
  const int g = blockIdx.y;
  const WideJoin j = reinterpret_cast<const WideJoin*>(a.work + a.at_joins)[unit];
  const int c = piece * join_wide_cols<D>() + threadIdx.x / kVecs;
  const int d = threadIdx.x % kVecs * 4;
  if (c >= j.tokens * a.group) return;
  const float* from = parts + (static_cast<size_t>(g) * a.cap_parts + j.part) * wide_part_floats(D);
  float m = -INFINITY, l = 0.0f, ref = 0.0f;
  f32x4 o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  constexpr int kBatch = 4;  // parts whose loads go out together
  for (int p0 = 0; p0 < j.parts; p0 += kBatch) {
    float pm[kBatch], pl[kBatch], pr[kBatch];
    f32x4 po[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const float* q = from + static_cast<size_t>(min(p0 + u, j.parts - 1)) * wide_part_floats(D);
      pm[u] = q[kWideCols * D + c];
      pl[u] = p0 + u < j.parts ? q[kWideCols * (D + 1) + c] : 0.0f;
      pr[u] = q[kWideCols * (D + 2) + c];
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      // no keys, or the part before has them: then nothing was written
      po[u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if (pl[u] != 0.0f) {
        const float* q = from + static_cast<size_t>(p0 + u) * wide_part_floats(D);
        po[u] = *reinterpret_cast<const f32x4*>(q + c * D + d);
      }
    }
    float m2 = m, ref2 = ref;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      m2 = p0 + u < j.parts ? fmaxf(m2, pm[u]) : m2;
      ref2 = p0 + u < j.parts ? fmaxf(ref2, pr[u]) : ref2;
    }
    const float keep = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - m2);
    o *= keep * unit_change(ref, ref2);
    l *= keep;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const float f = pm[u] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(pm[u] - m2);
      o += po[u] * (f * unit_change(pr[u], ref2));
      l += pl[u] * f;
    }
    m = m2;
    ref = ref2;
  }
  finish4<T>(a, j.row + c / a.group, g * a.group + c % a.group, d, o, m, l, ref);
}

// What joins the parts of both kernels, in one launch (one for each took 4.5 us
// more, also where there was nothing to join): `narrow` blocks of narrow units
// to a kv head, then blocks that go through what the plan cut of wide ones.
struct JoinShape {
  const float* wide_parts;
  int narrow, runs, by_unit, cols;
};

template <class T, int D>
__global__ __launch_bounds__(256) void join_kernel(AttendArgs a, JoinShape s) {
  const int at = blockIdx.x;
  if (at < s.narrow) {
    join_narrow<T, D>(a, s.runs, s.by_unit, at / s.cols, at % s.cols, s.cols);
    return;
  }
  constexpr int kPieces = kWideCols / join_wide_cols<D>();
  const auto* head = reinterpret_cast<ConstHead>(reinterpret_cast<uintptr_t>(a.work));
  const int all = head->joins * kPieces, blocks = gridDim.x - s.narrow;
  for (int k = at - s.narrow; k < all; k += blocks) {
    join_wide<T, D>(a, s.wide_parts, k / kPieces, k % kPieces);
  }
}

}  // namespace kv
}  // namespace grm
