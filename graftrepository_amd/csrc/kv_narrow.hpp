// kv_narrow.hpp -- attention of requests that bring few tokens (a decode
// step): at most 16 (token, head) columns to a kv head.
//
// The work is one pass over the request's codes, so it is cut by bytes: the
// key tiles (64 tokens) of all requests, in order, are dealt to the
// wavefronts of a kv head in equal runs, whatever request they belong to.  A
// wavefront streams its run without a pause: while one tile is computed the
// next one's codes are in flight (each register is loaded again as soon as
// it is used up) and the block ids of the one after, across request
// boundaries too.  Of a run at most the first and the last request are
// shared with a neighbour; their partial results (maximum, sum, unnormalised
// output) go to scratch, and the join kernel adds them in order.  Where the
// four runs of a block lie in one request, the block adds them itself.
//
// Inside a tile both products run on the matrix cores in fp16, where an int8
// code is exact (16x16x32; rows: 16 keys or 16 value columns, columns: the
// queries):
//   S^T = K Q^T: lane (i, G) = (lane % 16, lane / 16) loads 16 bytes of one
//     key: code row 16 (i / 4) + 4 t + i % 4 of the tile for row tile t, so
//     that results 4 t + j of the lane belong to keys 16 G + 4 t + j: each
//     lane ends up with 16 neighbouring keys of column i;
//   O^T = V^T P^T: those 16 are the lane's part of the B operand as they
//     are, and the A operand is 16 neighbouring tokens of one value column,
//     one 16-byte load of the transposed value codes.
// Nothing crosses lanes until the end, and nothing goes through LDS.  The 16
// keys lie in one block of the cache, so a lane has one key scale and one
// value scale per tile.
//
// Probabilities enter the second product as fp16(2^7 p vs / v), with v a
// power of two no less than any value scale the column has met: they stay
// below 2^15, and 2^-21 of the largest is still a normal number.  The
// running maximum follows only when a score passes it by more than 8
// (log2 units); until then nothing is rescaled.
//
// For fp32 and fp16 outputs the probabilities are two fp16 terms: the second
// is what the first leaves, scaled and summed apart (one term alone is off by
// 2.4e-4 of a flat row, more than the rounding to fp16).  For fp16 it is
// scaled by 2^11, which keeps it below 2^15.  For fp32 the scale is 2^19 and
// the maximum follows at once, so both terms stay below 2^15 and reach 2^-51
// of the largest; fp32 queries are two terms too.
#pragma once

#include "kv_attend.hpp"

namespace grm {
namespace kv {

// The last unit whose first tile is not past t (wave-uniform; first tiles
// ascend).  64 entries a step.
__device__ inline int find_unit(const int32_t* first, int n, int t) {
  const int lane = __lane_id();
  int lo = 0;
  while (true) {
    const int step = (n + kWave - 1) / kWave;
    const int at = lane * step;
    const bool le = at < n && first[lo + at] <= t;
    const int k = __popcll(__ballot(le)) - 1;
    lo += k * step;
    if (step == 1) return lo;
    n = min(step, n - k * step);
  }
}

constexpr float kWeightBias = 7.0f;

// Everything one wave carries for one unit.
template <class T, int D>
struct NarrowState {
  static constexpr int kTerms = T::code == kF32 ? 2 : 1;        // of a query
  static constexpr bool kRest = T::code != kBF16;               // of a probability
  static constexpr float kRestScale = T::code == kF32 ? 524288.0f : 2048.0f;
  static constexpr float kRescale = T::code == kF32 ? 0.0f : 8.0f;
  f16x8 q[kTerms][D / 32];
  float col_scale;  // softmax scale, log2 e and the query's own power of two
  f32x4 o[D / 16];
  f32x4 rest[kRest ? D / 16 : 1];
  float m, l;       // running maximum and this lane's sum of 2^(s - m + 7)
  float v_ref, v_inv;
};

// A unit and its tiles [first, end) in the order of all tiles.
struct UnitView {
  int at, first, end, request, row, tokens, tile_lo, ctx;
};

template <class T, int D>
__device__ inline void narrow_query(const AttendArgs& a, const UnitView& u, int g,
                                    NarrowState<T, D>& st) {
  const int lane = __lane_id(), i = lane & 15, G = lane >> 4;
  const bool mine = i < u.tokens * a.group;
  const int t = mine ? i / a.group : 0, h = mine ? i % a.group : 0;
  const typename T::store* q = static_cast<const typename T::store*>(a.q) +
                               static_cast<int64_t>(min(u.row + t, a.tokens - 1)) * a.q_token_stride +
                               static_cast<int64_t>(g * a.group + h) * a.q_head_stride + 16 * G;
  float x[D / 32][8];
  float top = 0.0f;
#pragma unroll
  for (int s = 0; s < D / 32; ++s) {
    load8<T>(q + 64 * (s >> 1) + 8 * (s & 1), x[s]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[s][e] = mine ? x[s][e] : 0.0f;
      top = fmaxf(top, fabsf(x[s][e]));
    }
  }
  top = fmaxf(top, __shfl_xor(top, 16));
  top = fmaxf(top, __shfl_xor(top, 32));
  st.col_scale = split_query<T, D / 32>(x, top, a.scale * kLog2e, st.q);
}

template <class T, int D>
__global__ __launch_bounds__(256, D > 128 ? 1 : 2) void attend_narrow_kernel(AttendArgs a) {
  typedef NarrowState<T, D> State;
  constexpr int kPieces = D / 64;   // 64-byte pieces of a key
  constexpr int kValueTiles = D / 16;
  const int g = blockIdx.x;
  const int lane = __lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int i = lane & 15, G = lane >> 4;
  const SchedHead* head = reinterpret_cast<const SchedHead*>(a.work);
  const NarrowUnit* units = reinterpret_cast<const NarrowUnit*>(a.work + a.at_units);
  const int32_t* first = reinterpret_cast<const int32_t*>(a.work + a.at_tiles);
  const int total = __builtin_amdgcn_readfirstlane(head->narrow_tiles);
  const int n_units = __builtin_amdgcn_readfirstlane(head->units);
  const int share = narrow_share(total, 4 * gridDim.y);
  const int run = 4 * blockIdx.y + wave;
  const int block_begin = 4 * blockIdx.y * share;
  if (block_begin >= total) return;
  const int block_end = min(total, block_begin + 4 * share);
  const int begin = min(total, run * share), end = min(total, begin + share);
  const int bs = 1 << a.block_log2;
  const size_t cell_bytes = static_cast<size_t>(bs) * D;

  auto unit_at = [&](int at) {
    const NarrowUnit u = units[at];
    UnitView v;
    v.at = at;
    v.first = __builtin_amdgcn_readfirstlane(first[at]);
    v.end = __builtin_amdgcn_readfirstlane(first[at + 1]);
    v.request = __builtin_amdgcn_readfirstlane(u.request);
    v.row = __builtin_amdgcn_readfirstlane(u.row);
    v.tokens = __builtin_amdgcn_readfirstlane(u.tokens);
    v.tile_lo = __builtin_amdgcn_readfirstlane(u.tile_lo);
    v.ctx = __builtin_amdgcn_readfirstlane(u.ctx);
    return v;
  };

  u32x4 kr[4][kPieces], vr[kValueTiles];
  float ks = 0.0f, vs = 0.0f;
  // Block of the 16 keys from `key` on; -1 where no column sees any of them.
  auto block_of = [&](const UnitView& u, int key) {
    const int last_pos = u.ctx + u.tokens - 1;
    const int first_seen = a.window > 0 ? max(0, u.ctx + 1 - a.window) : 0;
    const int j = key >> a.block_log2;
    int b = -1;
    if (key <= last_pos && key + 15 >= first_seen && j < a.width) {
      b = a.table[static_cast<size_t>(u.request) * a.width + j];
    }
    return static_cast<uint64_t>(static_cast<int64_t>(b)) < a.blocks ? b : -1;
  };
  auto load_k = [&](int tile, int kb) {
    const int key = tile * kTile + 16 * (i >> 2);
    const int8_t* k = a.k_codes +
                      (static_cast<size_t>(kb < 0 ? 0 : kb) * a.kv_heads + g) * cell_bytes +
                      ((key & (bs - 1)) + (i & 3)) * D + 16 * G;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
#pragma unroll
      for (int p = 0; p < kPieces; ++p) {
        kr[r][p] = __builtin_nontemporal_load(
            reinterpret_cast<const u32x4*>(k + 4 * r * D + 64 * p));
      }
    }
  };
  auto load_v = [&](int tile, int vb) {
    const int key = tile * kTile + 16 * G;
    const int8_t* v = a.v_codes +
                      (static_cast<size_t>(vb < 0 ? 0 : vb) * a.kv_heads + g) * cell_bytes +
                      static_cast<size_t>(i) * bs + (key & (bs - 1));
#pragma unroll
    for (int d = 0; d < kValueTiles; ++d) {
      vr[d] = __builtin_nontemporal_load(
          reinterpret_cast<const u32x4*>(v + static_cast<size_t>(16 * d) * bs));
    }
  };
  auto load_scales = [&](int vb) {
    const size_t cell = static_cast<size_t>(vb < 0 ? 0 : vb) * a.kv_heads + g;
    ks = vb < 0 ? 0.0f : a.k_scales[cell];
    vs = vb < 0 ? 0.0f : a.v_scales[cell];
  };

  State st;
  auto reset = [&]() {
#pragma unroll
    for (int d = 0; d < kValueTiles; ++d) {
      st.o[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if constexpr (State::kRest) st.rest[d] = st.o[d];
    }
    st.m = -INFINITY;
    st.l = 0.0f;
    st.v_ref = 0.0f;
    st.v_inv = 0.0f;
  };
  reset();

  // One unit may span the whole block: its waves then add up in LDS.
  UnitView now{};
  bool spans = false;
  if (begin < end) {
    now = unit_at(find_unit(first, n_units, begin));
    spans = now.first <= block_begin && now.end >= block_end;
    UnitView next = now;  // the unit of tile x + 1
    int vb = -1, kb1 = -1, vb1 = -1;
    {
      const int tile = now.tile_lo + begin - now.first;
      const int kb = block_of(now, tile * kTile + 16 * (i >> 2));
      vb = block_of(now, tile * kTile + 16 * G);
      load_k(tile, kb);
      load_scales(vb);
      load_v(tile, vb);
      if (begin + 1 < end) {
        if (begin + 1 >= next.end) next = unit_at(next.at + 1);
        const int tile1 = next.tile_lo + begin + 1 - next.first;
        kb1 = block_of(next, tile1 * kTile + 16 * (i >> 2));
        vb1 = block_of(next, tile1 * kTile + 16 * G);
      }
    }
    narrow_query<T, D>(a, now, g, st);
    for (int x = begin; x < end; ++x) {
      const int tile = now.tile_lo + x - now.first;
      const bool more = x + 1 < end;
      const int tile1 = next.tile_lo + x + 1 - next.first;
      // the block ids of the tile after the next one
      UnitView after = next;
      int kb2 = -1, vb2 = -1;
      if (x + 2 < end) {
        if (x + 2 >= after.end) after = unit_at(after.at + 1);
        const int tile2 = after.tile_lo + x + 2 - after.first;
        kb2 = block_of(after, tile2 * kTile + 16 * (i >> 2));
        vb2 = block_of(after, tile2 * kTile + 16 * G);
      }
      const int cols = now.tokens * a.group;
      const int pos = now.ctx + (i < cols ? i / a.group : 0);
      const int seen = a.window > 0 ? max(0, pos + 1 - a.window) : 0;  // first key it sees
      const int all_from = a.window > 0 ? max(0, now.ctx + now.tokens - a.window) : 0;

      // scores of keys 16 G + 4 r + j
      f32x4 s[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[r] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int p = 0; p < kPieces; ++p) {
          f16x8 c[2];
          codes_to_f16(kr[r][p], c);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int e = 0; e < State::kTerms; ++e) {
              s[r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(c[h], st.q[e][2 * p + h], s[r], 0, 0, 0);
            }
          }
        }
      }
      const float kscale = ks * st.col_scale, vscale = vs;
      if (more) {
        load_k(tile1, kb1);
        load_scales(vb1);
      }
      const int key = tile * kTile + 16 * G;
      const bool whole = tile * kTile >= all_from && tile * kTile + kTile - 1 <= now.ctx &&
                         __all(vb >= 0);
      float top = -INFINITY, v_top = 0.0f;
      if (whole) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            s[r][j] *= kscale;
            top = fmaxf(top, s[r][j]);
          }
        }
        v_top = vscale;
      } else {
        const bool some = vb >= 0 && key <= pos && key + 15 >= seen;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int k = key + 4 * r + j;
            s[r][j] = some && k <= pos && k >= seen ? s[r][j] * kscale : -INFINITY;
            top = fmaxf(top, s[r][j]);
          }
        }
        v_top = some ? vscale : 0.0f;
      }
      // a scale that is not finite makes the products what they should be,
      // but is no reference for others
      v_top = v_top <= 3.0e38f ? v_top : 0.0f;
      if (__any(top > st.m + State::kRescale || v_top > st.v_ref)) {
        float m2 = fmaxf(st.m, top);
        m2 = fmaxf(m2, __shfl_xor(m2, 16));
        m2 = fmaxf(m2, __shfl_xor(m2, 32));
        float v2 = fmaxf(st.v_ref, v_top);
        v2 = fmaxf(v2, __shfl_xor(v2, 16));
        v2 = fmaxf(v2, __shfl_xor(v2, 32));
        const float ref = v2 > st.v_ref ? power_above(v2) : st.v_ref;
        const float keep = m2 == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(st.m - m2);
        const float keep_o = ref > 0.0f ? keep * (st.v_ref / ref) : 1.0f;
        st.l *= keep;
#pragma unroll
        for (int d = 0; d < kValueTiles; ++d) {
          st.o[d] *= keep_o;
          if constexpr (State::kRest) st.rest[d] *= keep_o;
        }
        st.m = m2;
        st.v_ref = ref;
        st.v_inv = ref > 0.0f ? 1.0f / ref : 0.0f;
      }
      const float shift = (st.m == -INFINITY ? 0.0f : st.m) - kWeightBias;
      const float v_factor = vscale * st.v_inv;
      f16x8 w[2], w_rest[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float sc = s[2 * h + (e >> 2)][e & 3];
          const float p = __builtin_amdgcn_exp2f(sc - shift);
          st.l += p;
          const float v = whole || sc != -INFINITY ? p * v_factor : 0.0f;
          w[h][e] = static_cast<_Float16>(v);
          if constexpr (State::kRest) {
            w_rest[h][e] =
                static_cast<_Float16>((v - static_cast<float>(w[h][e])) * State::kRestScale);
          }
        }
      }
#pragma unroll
      for (int d = 0; d < kValueTiles; ++d) {
        f16x8 c[2];
        codes_to_f16(vr[d], c);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          st.o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(c[h], w[h], st.o[d], 0, 0, 0);
          if constexpr (State::kRest) {
            st.rest[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(c[h], w_rest[h], st.rest[d], 0, 0, 0);
          }
        }
      }
      if (more) load_v(tile1, vb1);

      if (!spans && (x + 1 == now.end || !more)) {
        // the unit, or this run's share of it, is done
        float l = st.l + __shfl_xor(st.l, 16);
        l += __shfl_xor(l, 32);
        const bool alone = now.first >= begin && now.end <= end;
        float* part = a.parts + narrow_part(g, 4 * gridDim.y, run, now.first <= begin ? 0 : 1) *
                                    (kNarrowCols * (D + 2));
        if (i < cols) {
          const int row = now.row + i / a.group, h = g * a.group + i % a.group;
#pragma unroll
          for (int d = 0; d < kValueTiles; ++d) {
            f32x4 o = st.o[d];
            if constexpr (State::kRest) o += st.rest[d] * (1.0f / State::kRestScale);
            o *= st.v_ref;
            if (alone) finish4<T>(a, row, h, 16 * d + 4 * G, o, st.m, l);
            else *reinterpret_cast<f32x4*>(part + i * D + 16 * d + 4 * G) = o;
          }
          if (!alone && G == 0) {
            part[kNarrowCols * D + i] = st.m;
            part[kNarrowCols * (D + 1) + i] = l;
          }
        }
        if (more) {
          reset();
          narrow_query<T, D>(a, next, g, st);
        }
      }
      now = next;
      next = after;
      vb = vb1;
      kb1 = kb2;
      vb1 = vb2;
    }
  }

  // The block's first tile decides for all four waves alike; a wave without
  // a run of its own adds nothing.
  __shared__ float s_ml[2][4][16];
  __shared__ float s_o[4][16][D];
  __shared__ int s_unit[2];  // wave 0 has the first run
  if (threadIdx.x == 0) {
    s_unit[0] = spans;
    s_unit[1] = now.at;
  }
  __syncthreads();
  if (!s_unit[0]) return;
  const UnitView u = unit_at(__builtin_amdgcn_readfirstlane(s_unit[1]));
  const int cols = u.tokens * a.group;
  st.l += __shfl_xor(st.l, 16);
  st.l += __shfl_xor(st.l, 32);
  if (G == 0) {
    s_ml[0][wave][i] = st.m;
    s_ml[1][wave][i] = st.l;
  }
  __syncthreads();
  float top = s_ml[0][0][i];
#pragma unroll
  for (int w = 1; w < 4; ++w) top = fmaxf(top, s_ml[0][w][i]);
  const float mine = st.m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(st.m - top) * st.v_ref;
  if (i < cols) {
#pragma unroll
    for (int d = 0; d < kValueTiles; ++d) {
      f32x4 o = st.o[d];
      if constexpr (State::kRest) o += st.rest[d] * (1.0f / State::kRestScale);
      *reinterpret_cast<f32x4*>(&s_o[wave][i][16 * d + 4 * G]) = o * mine;
    }
  }
  __syncthreads();
  const bool alone = u.first == block_begin && u.end == block_end;
  float* part = a.parts + narrow_part(g, 4 * gridDim.y, 4 * blockIdx.y, 0) * (kNarrowCols * (D + 2));
  for (int e = threadIdx.x; e < cols * (D / 4); e += 256) {
    const int c = e / (D / 4), d = e % (D / 4) * 4;
    f32x4 o = *reinterpret_cast<const f32x4*>(&s_o[0][c][d]);
#pragma unroll
    for (int w = 1; w < 4; ++w) o += *reinterpret_cast<const f32x4*>(&s_o[w][c][d]);
    float m = s_ml[0][0][c], l = 0.0f;
#pragma unroll
    for (int w = 1; w < 4; ++w) m = fmaxf(m, s_ml[0][w][c]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      l += s_ml[0][w][c] == -INFINITY ? s_ml[1][w][c]
                                      : s_ml[1][w][c] * __builtin_amdgcn_exp2f(s_ml[0][w][c] - m);
    }
    if (alone) {
      finish4<T>(a, u.row + c / a.group, g * a.group + c % a.group, d, o, m, l);
    } else {
      *reinterpret_cast<f32x4*>(part + c * D + d) = o;
      if (d == 0) {
        part[kNarrowCols * D + c] = m;
        part[kNarrowCols * (D + 1) + c] = l;
      }
    }
  }
}

// Joins the parts of units that several runs share: one block per kv head,
// column, and unit (or, where there are more units than runs, per boundary
// between two runs; the first boundary inside a unit does it).  The threads
// take four output columns each, and the parts in 1024 / D groups.
template <class T, int D>
__global__ __launch_bounds__(256) void join_narrow_kernel(AttendArgs a, int runs, int by_unit) {
  constexpr int kVecs = D / 4, kGroups = 256 / kVecs;
  const int g = blockIdx.x, c = blockIdx.z;
  const SchedHead* head = reinterpret_cast<const SchedHead*>(a.work);
  const NarrowUnit* units = reinterpret_cast<const NarrowUnit*>(a.work + a.at_units);
  const int32_t* first = reinterpret_cast<const int32_t*>(a.work + a.at_tiles);
  const int total = head->narrow_tiles, n_units = head->units;
  const int share = narrow_share(total, runs);
  int at = blockIdx.y;
  if (by_unit) {
    if (at >= n_units) return;
  } else {
    const int t = (blockIdx.y + 1) * share;
    if (t >= total) return;
    at = find_unit(first, n_units, t);
    if (first[at] >= t || first[at] < t - share) return;  // not cut here, or cut before
  }
  const int from = first[at], to = first[at + 1];
  const NarrowUnit u = units[at];
  if (to <= from || c >= u.tokens * a.group) return;
  const int r0 = from / share, r1 = (to - 1) / share;
  if (r0 == r1) return;
  // One block held all of it: finished there.
  if (r0 / 4 * 4 * share == from && min(total, (r0 / 4 + 1) * 4 * share) == to) return;
  // Parts in order: a whole block's, or a run's.
  auto part_of = [&](int r) -> const float* {
    const int b0 = r / 4 * 4 * share, b1 = min(total, (r / 4 + 1) * 4 * share);
    if (from <= b0 && to >= b1) return r % 4 ? nullptr : a.parts + narrow_part(g, runs, r, 0) * (kNarrowCols * (D + 2));
    return a.parts + narrow_part(g, runs, r, from > r * share ? 1 : 0) * (kNarrowCols * (D + 2));
  };
  __shared__ float s_top[4];
  __shared__ float s_l[kGroups];
  __shared__ f32x4 s_o[kGroups][kVecs];
  float m = -INFINITY;
  for (int r = r0 + static_cast<int>(threadIdx.x); r <= r1; r += 256) {
    const float* p = part_of(r);
    if (p) m = fmaxf(m, p[kNarrowCols * D + c]);
  }
#pragma unroll
  for (int d = kWave / 2; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
  if (__lane_id() == 0) s_top[threadIdx.x / kWave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(s_top[0], s_top[1]), fmaxf(s_top[2], s_top[3]));
  const int group = threadIdx.x / kVecs, d = threadIdx.x % kVecs;
  f32x4 o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float l = 0.0f;
#pragma unroll 4
  for (int r = r0 + group; r <= r1; r += kGroups) {
    const float* p = part_of(r);
    if (!p) continue;
    const float pm = p[kNarrowCols * D + c], pl = p[kNarrowCols * (D + 1) + c];
    const f32x4 po = *reinterpret_cast<const f32x4*>(p + c * D + 4 * d);
    const float f = pm == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(pm - m);
    o += po * f;
    l += pl * f;
  }
  s_o[group][d] = o;
  if (d == 0) s_l[group] = l;
  __syncthreads();
  if (group == 0) {
#pragma unroll
    for (int k = 1; k < kGroups; ++k) {
      o += s_o[k][d];
      l += s_l[k];
    }
    finish4<T>(a, u.row + c / a.group, g * a.group + c % a.group, 4 * d, o, m, l);
  }
}

}  // namespace kv
}  // namespace grm
