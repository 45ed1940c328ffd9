// kv_narrow.hpp -- attention of requests that bring few tokens (a decode
// step): at most 16 (token, head) columns to a kv head.
//
// The work is one pass over the request's codes, so it is cut by bytes: the
// key tiles (64 tokens) of all requests, in order, are dealt to the
// wavefronts of a kv head in equal runs, whatever request they belong to.  A
// wavefront streams its run across request boundaries: the codes of the next
// half tile are in flight while one is computed (each register is loaded
// again as soon as it is used up), and the block ids and scales of the next
// tile.  Of a run at most the first and the last request are shared with a
// neighbour; their partial results (maximum, sum, unnormalised output) go to
// scratch, and the join kernel adds them in order.  Where the four runs of a
// block lie in one request, the block adds them itself; where requests are
// known to be short, each has a block, and there is no join.  The plan leaves a
// unit that each run begins in, so a wave is three loads from its codes.
//
// Bound by bytes where there are many: each further byte comes at 6.5 TB/s
// (bf16, head_dim 128, blocks of 64).  Start, end and join are about 12 us of
// a call: a step of 32 sessions of 190 to 8150 tokens (32 heads on 8, 167 MB)
// takes 33 us here and 6 in the join; one session of 131071 tokens (268 MB) 54
// and 5; 48 sessions of 32 to 4095 tokens at head_dim 256 (77 MB) 29 and 6.
// Codes through LDS by direct loads measured 4.35 TB/s instead.
//
// Inside a tile both products run on the matrix cores in fp16 or bf16, where an
// int8 code is exact (16x16x32; rows: 16 keys or 16 value columns, columns: the
// queries):
//   S^T = K Q^T: lane (i, G) = (lane % 16, lane / 16) loads 16 bytes of one
//     key: of half h of the tile, code row 16 (i / 4) + 4 t + i % 4 for row
//     tile t, so that results 4 t + j of the lane belong to the half's keys
//     16 G + 4 t + j: each lane ends up with 16 neighbouring keys of column i;
//   O^T = V^T P^T: those 16 are the lane's part of the B operand as they
//     are, and the A operand is 16 neighbouring tokens of one value column,
//     one 16-byte load of the transposed value codes.
// Nothing crosses lanes and nothing goes through LDS until the end.  The 16
// keys lie in one block of the cache, so a lane has one key scale and one
// value scale.  With 128-token blocks a tile is two such halves, and the two
// halves of a value column, one 128-byte line, are read together (tiles of 64
// tokens fetched 1.4 times the bytes there).
//
// Probabilities enter the second product as p vs / v, with v a power of two no
// less than any value scale the column has met and at most twice the largest.
// For 16-bit outputs they are two fp16 terms of 2^13 times that, the second
// what the first leaves: one term alone is off by up to 2^-12 of each value,
// which shows in every output whose values cancel.  The running maximum follows
// only when a score passes it by more than 2 (log2 units), so weights stay
// below 2^15; 2^-27 of the largest probability is still a normal number, and
// what is lost below that is 2^-38 of it.  (An allowance of 8 would rescale
// less often, but lose 2^-32.)  For fp32 outputs they are three bf16 terms,
// which hold all 24 bits and fp32's range; the lesser two are summed apart, so
// that the sums that grow round no more often than fp32's own would.
#pragma once

#include "kv_attend.hpp"

#include <type_traits>

namespace grm {
namespace kv {

// The kernel's arguments, read again where they are used: kept in scalar
// registers through the loop, those of a unit's begin and end would push out
// the loop's own.
__device__ __forceinline__ const AttendArgs& late_args() {
  typedef const __attribute__((address_space(4))) AttendArgs* ConstArgs;
  uintptr_t p = reinterpret_cast<uintptr_t>(__builtin_amdgcn_kernarg_segment_ptr());
  asm volatile("" : "+s"(p));
  return *(const AttendArgs*)(ConstArgs)p;
}

// Everything one wave carries for one unit.
template <class T, int D>
struct NarrowState {
  static constexpr int kTerms = T::code == kF32 ? 3 : 1;  // of a query
  static constexpr int kWeights = weight_terms<T>();      // of a probability
  static constexpr bool kApart = T::code == kF32;  // the lesser ones are summed apart
  static constexpr float kRescale = 2.0f;
  float col_scale;  // softmax scale, log2 e and the query's own power of two
  f32x4 o[D / 16];
  f32x4 rest[kApart ? D / 16 : 1];
  float m, l;       // running maximum and this lane's sum of 2^(s - m + bias)
  float v_ref, v_inv;
};

// A unit and its tiles [first, end) in the order of all tiles.
struct UnitView {
  int at, first, end, request, row, tokens, tile_lo, ctx;
};

template <class T, int D>
__device__ inline void narrow_query(const AttendArgs& a, const UnitView& u, int g,
                                    NarrowState<T, D>& st, u32x4* s_q) {
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
  u32x4 f[NarrowState<T, D>::kTerms][D / 32];
  st.col_scale = split_query<T, D / 32>(x, top, a.scale * kLog2e, f);
#pragma unroll
  for (int e = 0; e < NarrowState<T, D>::kTerms; ++e) {
#pragma unroll
    for (int s = 0; s < D / 32; ++s) s_q[(e * (D / 32) + s) * kWave + lane] = f[e][s];
  }
}

template <class T, int D, int H>
__global__ __launch_bounds__(256, narrow_blocks_per_cu(T::code, D)) void attend_narrow_kernel(AttendArgs a) {
  typedef NarrowState<T, D> State;
  constexpr int kPieces = D / 64;  // 64-byte pieces of a key
  constexpr int kValueTiles = D / 16;
  constexpr int kHeld = (T::code == kF32 && D == 256 ? 4 : kValueTiles) / H;
  constexpr int kNarrowTile = 64 * H;
  const int g = blockIdx.x;
  const int lane = __lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int i = lane & 15, G = lane >> 4, Gk = (lane & 15) >> 2;
  const auto* units = reinterpret_cast<ConstUnit>(reinterpret_cast<uintptr_t>(a.work) + a.at_units);
  const auto* first = reinterpret_cast<ConstInt>(reinterpret_cast<uintptr_t>(a.work) + a.at_tiles);
  const auto* table = reinterpret_cast<ConstInt>(reinterpret_cast<uintptr_t>(a.table));
  const auto* head = reinterpret_cast<ConstHead>(reinterpret_cast<uintptr_t>(a.work));
  const int run = 4 * blockIdx.y + wave, runs = 4 * gridDim.y;
  int start_unit, begin, end, block_begin, block_end;
  if (a.whole) {
    start_unit = blockIdx.y;
    if (start_unit >= head->units) return;
    block_begin = first[start_unit];
    block_end = first[start_unit + 1];
    const int each = (block_end - block_begin + 3) / 4;
    begin = min(block_end, block_begin + wave * each);
    end = min(block_end, begin + each);
  } else {
    start_unit = reinterpret_cast<ConstInt>(reinterpret_cast<uintptr_t>(a.work) +
                                            a.at_run_units)[run];
    const Deal deal(head->narrow_tiles, runs);
    begin = deal.begin(run);
    end = deal.begin(run + 1);
    block_begin = deal.begin(4 * blockIdx.y);
    block_end = deal.begin(4 * blockIdx.y + 4);
  }
  if (block_begin >= block_end) return;
  const int bs = 1 << a.block_log2;
  const uint32_t cell_bytes = static_cast<uint32_t>(bs * D);
  // a lane's column's token, and its part of a load's address
  const int col_token = i / a.group;
  const int8_t* k_lane = a.k_codes + (((16 * Gk) & (bs - 1)) + (i & 3)) * D + 16 * G;
  const int8_t* v_lane = a.v_codes + static_cast<size_t>(i) * bs + ((16 * G) & (bs - 1));

  auto unit_at = [&](int at) {
    UnitView v;
    v.at = at;
    v.first = first[at];
    v.end = first[at + 1];
    v.request = units[at].request;
    v.row = units[at].row;
    v.tokens = units[at].tokens;
    v.tile_lo = units[at].tile_lo;
    v.ctx = units[at].ctx;
    return v;
  };

  // Half a tile: where a lane's keys and values are.  `Asked` holds the
  // table's entries for its four groups of 16 keys on their way.
  struct Asked {
    int id[4], seen;
  };
  struct Half {
    bool all, here;  // every group has a block that some column sees; this lane's has
    const int8_t* k;
    const int8_t* v;
    uint32_t cell;
  };
  auto ask_half = [&](const UnitView& u, int key0) {
    const int last_pos = u.ctx + u.tokens - 1;
    const int first_seen = a.window > 0 ? max(0, u.ctx + 1 - a.window) : 0;
    const size_t row = static_cast<size_t>(u.request) * a.width;
    Asked r;
    r.seen = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int key = key0 + 16 * k, at = key >> a.block_log2;
      if (key <= last_pos && key + 15 >= first_seen && at < a.width) r.seen |= 1 << k;
      r.id[k] = table[row + max(0, min(at, a.width - 1))];
    }
    return r;
  };
  auto take = [&](const Asked& r, int h) {
    Half t;
    int id[4], ok = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool there = (r.seen >> k & 1) && static_cast<uint32_t>(r.id[k]) < a.blocks;
      id[k] = there ? r.id[k] : 0;  // no block: any one, what it gives is not used
      ok |= there ? 1 << k : 0;
    }
    auto cell_of = [&](int k) {
      const int lo = k & 1 ? id[1] : id[0], hi = k & 1 ? id[3] : id[2];
      return static_cast<uint32_t>(k & 2 ? hi : lo) * a.kv_heads + g;
    };
    t.all = ok == 15;
    t.here = ok >> G & 1;
    t.cell = cell_of(G);
    const int place = 64 * h & (bs - 1);  // the second half of a 128-token block
    t.k = k_lane + place * D + static_cast<uint64_t>(cell_of(Gk)) * cell_bytes;
    t.v = v_lane + place + static_cast<uint64_t>(t.cell) * cell_bytes;
    return t;
  };

  // Keys: four row tiles held, eight to a tile.  Values: half of the tile's
  // columns held, both halves of the tokens.
  u32x4 kr[4][kPieces], vr[kHeld][H];
  auto load_keys = [&](const Half& t, int r) {
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
      kr[r][p] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(t.k + 4 * r * D + 64 * p));
    }
  };
  auto load_values = [&](const Half (&t)[H], int d) {
#pragma unroll
    for (int h = 0; h < H; ++h) {
      vr[d % kHeld][h] = __builtin_nontemporal_load(
          reinterpret_cast<const u32x4*>(t[h].v + static_cast<size_t>(16 * d) * bs));
    }
  };

  // The unit's queries, as the lane's part of the B operands: in LDS, so that
  // they take registers during the first product only;
  // their memory is the outputs' when the waves are done with them.
  union Lds {
    u32x4 q[4][State::kTerms * (D / 32)][kWave];
    float o[4][16][D];
  };
  __shared__ Lds s_lds;
  u32x4* s_q = &s_lds.q[wave][0][0];

  State st;
  auto reset = [&]() {
#pragma unroll
    for (int d = 0; d < kValueTiles; ++d) {
      st.o[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if constexpr (State::kApart) st.rest[d] = st.o[d];
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
    now = unit_at(start_unit);
    spans = now.first <= block_begin && now.end >= block_end;
    UnitView ahead = now;  // the unit of the tile whose blocks were asked for last
    Half cur[H], nxt[H];
    float ks[H], vs[H];
    {
      const int key = (now.tile_lo + begin - now.first) * kNarrowTile;
      Asked asked[H];
#pragma unroll
      for (int h = 0; h < H; ++h) asked[h] = ask_half(now, key + 64 * h);
#pragma unroll
      for (int h = 0; h < H; ++h) cur[h] = take(asked[h], h);
#pragma unroll
      for (int r = 0; r < 4; ++r) load_keys(cur[0], r);
#pragma unroll
      for (int h = 0; h < H; ++h) {
        ks[h] = a.k_scales[cur[h].cell];
        vs[h] = a.v_scales[cur[h].cell];
      }
#pragma unroll
      for (int d = 0; d < kHeld; ++d) load_values(cur, d);
    }
    narrow_query<T, D>(late_args(), now, g, st, s_q);

    // Tile x of the run; MORE: another one follows.
    auto step = [&](int x, auto more_follow) {
      constexpr bool kMore = decltype(more_follow)::value;
      const int key0 = (now.tile_lo + x - now.first) * kNarrowTile;
      Asked asked[H];
      if constexpr (kMore) {
        if (x + 1 >= ahead.end) ahead = unit_at(ahead.at + 1);
        const int key = (ahead.tile_lo + x + 1 - ahead.first) * kNarrowTile;
#pragma unroll
        for (int h = 0; h < H; ++h) asked[h] = ask_half(ahead, key + 64 * h);
      }
      // products of the halves' keys 16 G + 4 r + j
      f32x4 s[H][4];
      u32x4 q[State::kTerms][D / 32];
#pragma unroll
      for (int e = 0; e < State::kTerms; ++e) {
#pragma unroll
        for (int k = 0; k < D / 32; ++k) q[e][k] = s_q[(e * (D / 32) + k) * kWave + lane];
      }
      auto multiply = [&](int h, int r) {
        // the lesser terms apart: their sums are small, and so is what they round
        f32x4 sum[2] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}, f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
        for (int p = 0; p < kPieces; ++p) {
          u32x4 c[2];
          codes_as<query_bf16<T>()>(kr[r][p], c);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
#pragma unroll
            for (int e = 0; e < State::kTerms; ++e) {
              f32x4& to = sum[e ? 1 : 0];
              to = mfma<query_bf16<T>()>(c[k], q[e][2 * p + k], to);
            }
          }
        }
        s[h][r] = State::kTerms > 1 ? sum[0] + sum[1] : sum[0];
      };
      if constexpr (H == 2) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          multiply(0, r);
          load_keys(cur[H - 1], r);
        }
      }
      float kscale[H], vscale[H];
#pragma unroll
      for (int h = 0; h < H; ++h) {
        kscale[h] = cur[h].here ? ks[h] * st.col_scale : 0.0f;
        vscale[h] = cur[h].here ? vs[h] : 0.0f;
      }
      if constexpr (kMore) {
#pragma unroll
        for (int h = 0; h < H; ++h) {
          nxt[h] = take(asked[h], h);
          ks[h] = a.k_scales[nxt[h].cell];
          vs[h] = a.v_scales[nxt[h].cell];
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        multiply(H - 1, r);
        if constexpr (kMore) load_keys(nxt[0], r);
      }

      const int all_from = a.window > 0 ? max(0, now.ctx + now.tokens - a.window) : 0;
      const bool whole =
          key0 >= all_from && key0 + kNarrowTile - 1 <= now.ctx && cur[0].all && cur[H - 1].all;
      // Scaling by what is not negative keeps the order, so the whole tile's
      // maximum is taken before it.  A partly seen tile is scaled first, and
      // what a column does not see is -inf.
      float top[H], v_top[H], mul[H];
      if (whole && __all(!(kscale[0] < 0.0f || kscale[H - 1] < 0.0f))) {
#pragma unroll
        for (int h = 0; h < H; ++h) {
          top[h] = s[h][0][0];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
#pragma unroll
            for (int j = 0; j < 4; ++j) top[h] = fmaxf(top[h], s[h][r][j]);
          }
          top[h] *= kscale[h];
          v_top[h] = vscale[h];
          mul[h] = kscale[h];
        }
      } else {
        const int pos = now.ctx + min(col_token, now.tokens - 1);
        const int seen = a.window > 0 ? max(0, pos + 1 - a.window) : 0;  // first key it sees
#pragma unroll
        for (int h = 0; h < H; ++h) {
          const int key = key0 + 64 * h + 16 * G;
          const bool some = cur[h].here && key <= pos && key + 15 >= seen;
          top[h] = -INFINITY;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int k = key + 4 * r + j;
              s[h][r][j] = some && k <= pos && k >= seen ? s[h][r][j] * kscale[h] : -INFINITY;
              top[h] = fmaxf(top[h], s[h][r][j]);
            }
          }
          v_top[h] = some ? vscale[h] : 0.0f;
          mul[h] = 1.0f;
        }
      }
      // a scale that is not finite makes the products what they should be,
      // but is no reference for others
      const float t_top = fmaxf(top[0], top[H - 1]);
      const float t_v = fmaxf(v_top[0] <= 3.0e38f ? v_top[0] : 0.0f,
                              v_top[H - 1] <= 3.0e38f ? v_top[H - 1] : 0.0f);
      if (__any(t_top > st.m + State::kRescale || t_v > st.v_ref)) {
        float m2 = fmaxf(st.m, t_top);
        m2 = fmaxf(m2, __shfl_xor(m2, 16));
        m2 = fmaxf(m2, __shfl_xor(m2, 32));
        float v2 = fmaxf(st.v_ref, t_v);
        v2 = fmaxf(v2, __shfl_xor(v2, 16));
        v2 = fmaxf(v2, __shfl_xor(v2, 32));
        const float ref = v2 > st.v_ref ? power_above(v2) : st.v_ref;
        const float keep = m2 == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(st.m - m2);
        const float keep_o = ref > 0.0f ? keep * (st.v_ref / ref) : 1.0f;
        st.l *= keep;
#pragma unroll
        for (int d = 0; d < kValueTiles; ++d) {
          st.o[d] *= keep_o;
          if constexpr (State::kApart) st.rest[d] *= keep_o;
        }
        st.m = m2;
        st.v_ref = ref;
        st.v_inv = ref > 0.0f ? 1.0f / ref : 0.0f;
      }
      const float shift = weight_bias(T::code) - (st.m == -INFINITY ? 0.0f : st.m);
      float v_factor[H];
#pragma unroll
      for (int h = 0; h < H; ++h) v_factor[h] = vscale[h] * st.v_inv;
      u32x4 w[State::kWeights][H][2];
      // probabilities and their weights; `some_hidden`: 0 times a scale that
      // is no number has to be 0
      auto weights = [&](auto some_hidden) {
#pragma unroll
        for (int h = 0; h < H; ++h) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float p[8], v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float sc = s[h][2 * k + (e >> 2)][e & 3];
              p[e] = __builtin_amdgcn_exp2f(fmaf(sc, mul[h], shift));
              v[e] = p[e] * v_factor[h];
              if constexpr (decltype(some_hidden)::value) v[e] = sc == -INFINITY ? 0.0f : v[e];
              v[e] = as_rounded(v[e]);
            }
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
              uint32_t t[State::kWeights];
              split_weights<T>(v[e], v[e + 1], t);
#pragma unroll
              for (int n = 0; n < State::kWeights; ++n) w[n][h][k][e / 2] = t[n];
            }
            st.l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
          }
        }
      };
      if (!whole && __any(!(fabsf(v_factor[0]) <= 3.0e38f && fabsf(v_factor[H - 1]) <= 3.0e38f))) {
        weights(std::true_type{});
      } else {
        weights(std::false_type{});
      }

#pragma unroll
      for (int d = 0; d < kValueTiles; ++d) {
        u32x4 c[H][2];
#pragma unroll
        for (int h = 0; h < H; ++h) codes_as<weight_bf16<T>()>(vr[d % kHeld][h], c[h]);
#pragma unroll
        for (int h = 0; h < H; ++h) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
#pragma unroll
            for (int n = 0; n < State::kWeights; ++n) {
              f32x4& o = n && State::kApart ? st.rest[d] : st.o[d];
              o = mfma<weight_bf16<T>()>(c[h][k], w[n][h][k], o);
            }
          }
        }
        if (d + kHeld < kValueTiles) load_values(cur, d + kHeld);
        else if constexpr (kMore) load_values(nxt, d + kHeld - kValueTiles);
      }

      if (!spans && (!kMore || x + 1 == now.end)) {
        // the unit, or this run's share of it, is done
        const AttendArgs& b = late_args();
        const int cols = now.tokens * b.group;
        float l = st.l + __shfl_xor(st.l, 16);
        l += __shfl_xor(l, 32);
        const bool alone = now.first >= begin && now.end <= end;
        float* part = b.parts + narrow_part(g, runs, run, now.first <= begin ? 0 : 1) *
                                    narrow_part_floats(D);
        if (i < cols) {
          const int row = now.row + col_token, h = g * b.group + i - col_token * b.group;
#pragma unroll
          for (int d = 0; d < kValueTiles; ++d) {
            f32x4 o = st.o[d];
            if constexpr (State::kApart) o += st.rest[d];
            if (alone) finish4<T>(b, row, h, 16 * d + 4 * G, o, st.m, l, st.v_ref);
            else *reinterpret_cast<f32x4*>(part + i * D + 16 * d + 4 * G) = o;
          }
          if (!alone && G == 0) {
            part[kNarrowCols * D + i] = st.m;
            part[kNarrowCols * (D + 1) + i] = l;
            part[kNarrowCols * (D + 2) + i] = st.v_ref;
          }
        }
        if constexpr (kMore) {
          now = unit_at(now.at + 1);
          reset();
          narrow_query<T, D>(b, now, g, st, s_q);
        }
      }
      if constexpr (kMore) {
#pragma unroll
        for (int h = 0; h < H; ++h) cur[h] = nxt[h];
      }
    };
    int x = begin;
    for (; x + 1 < end; ++x) step(x, std::true_type{});
    step(x, std::false_type{});
  }

  // The block's first tile decides for all four waves alike; a wave without
  // a run of its own adds nothing.
  __shared__ float s_ml[3][4][16];
  auto& s_o = s_lds.o;
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
    s_ml[2][wave][i] = st.v_ref;
  }
  __syncthreads();
  float top = s_ml[0][0][i], ref = s_ml[2][0][i];
#pragma unroll
  for (int w = 1; w < 4; ++w) {
    top = fmaxf(top, s_ml[0][w][i]);
    ref = fmaxf(ref, s_ml[2][w][i]);
  }
  const float mine = st.m == -INFINITY
                         ? 0.0f : __builtin_amdgcn_exp2f(st.m - top) * unit_change(st.v_ref, ref);
  if (i < cols) {
#pragma unroll
    for (int d = 0; d < kValueTiles; ++d) {
      f32x4 o = st.o[d];
      if constexpr (State::kApart) o += st.rest[d];
      *reinterpret_cast<f32x4*>(&s_o[wave][i][16 * d + 4 * G]) = o * mine;
    }
  }
  __syncthreads();
  const bool alone = u.first == block_begin && u.end == block_end;
  float* part = a.parts + narrow_part(g, runs, 4 * blockIdx.y, 0) * narrow_part_floats(D);
  for (int e = threadIdx.x; e < cols * (D / 4); e += 256) {
    const int c = e / (D / 4), d = e % (D / 4) * 4;
    f32x4 o = *reinterpret_cast<const f32x4*>(&s_o[0][c][d]);
#pragma unroll
    for (int w = 1; w < 4; ++w) o += *reinterpret_cast<const f32x4*>(&s_o[w][c][d]);
    float m = s_ml[0][0][c], l = 0.0f, all_ref = s_ml[2][0][c];
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      m = fmaxf(m, s_ml[0][w][c]);
      all_ref = fmaxf(all_ref, s_ml[2][w][c]);
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      l += s_ml[0][w][c] == -INFINITY ? s_ml[1][w][c]
                                      : s_ml[1][w][c] * __builtin_amdgcn_exp2f(s_ml[0][w][c] - m);
    }
    if (alone) {
      finish4<T>(a, u.row + c / a.group, g * a.group + c % a.group, d, o, m, l, all_ref);
    } else {
      *reinterpret_cast<f32x4*>(part + c * D + d) = o;
      if (d == 0) {
        part[kNarrowCols * D + c] = m;
        part[kNarrowCols * (D + 1) + c] = l;
        part[kNarrowCols * (D + 2) + c] = all_ref;
      }
    }
  }
}

// Joins the parts of units that several runs share: one block per kv head and
// unit (or, where there are more units than runs, per boundary between two
// runs; the first boundary inside a unit does it) takes every `step`-th of the
// unit's columns.  The threads take four output columns each, and the parts in
// 1024 / D groups.
template <class T, int D>
__device__ inline void join_narrow(const AttendArgs& a, int runs, bool by_unit, int at,
                                   int first_col, int step) {
  constexpr int kVecs = D / 4, kGroups = 256 / kVecs;
  const int g = blockIdx.y;
  const SchedHead* head = reinterpret_cast<const SchedHead*>(a.work);
  const NarrowUnit* units = reinterpret_cast<const NarrowUnit*>(a.work + a.at_units);
  const int32_t* first = reinterpret_cast<const int32_t*>(a.work + a.at_tiles);
  const int total = head->narrow_tiles, n_units = head->units;
  const Deal deal(total, runs);
  if (by_unit) {
    if (at >= n_units) return;
  } else {
    const int t = deal.begin(at + 1), before = deal.begin(at);
    if (t >= total) return;
    at = find_unit(first, n_units, t);
    // not cut here, or cut before
    if (first[at] >= t || first[at] < before) return;
  }
  const int from = first[at], to = first[at + 1];
  const NarrowUnit u = units[at];
  if (to <= from) return;
  const int r0 = deal.run(from), r1 = deal.run(to - 1);
  if (r0 == r1) return;
  // One block held all of it: finished there.
  if (deal.begin(r0 / 4 * 4) == from && deal.begin(r0 / 4 * 4 + 4) == to) return;
  // Parts in order: runs up to the first block of runs that the unit holds
  // whole, a part to each such block, and runs behind them.
  const int b0 = from <= deal.begin(r0 / 4 * 4) ? r0 / 4 * 4 : r0 / 4 * 4 + 4;
  const int b1 = to >= deal.begin(r1 / 4 * 4 + 4) ? r1 / 4 * 4 + 4 : r1 / 4 * 4;
  const int lead = b0 < b1 ? b0 - r0 : r1 + 1 - r0, whole = b0 < b1 ? (b1 - b0) / 4 : 0;
  const int parts = lead + whole + (b0 < b1 ? max(0, r1 + 1 - b1) : 0);
  auto part_of = [&](int p) -> const float* {
    const int r = p < lead ? r0 + p : p < lead + whole ? b0 + 4 * (p - lead) : b1 + p - lead - whole;
    return a.parts +
           narrow_part(g, runs, r, from > deal.begin(r) ? 1 : 0) * narrow_part_floats(D);
  };
  __shared__ float s_top[2][4];
  __shared__ float s_l[kGroups];
  __shared__ f32x4 s_o[kGroups][kVecs];
  for (int c = first_col; c < u.tokens * a.group; c += step) {
    float m = -INFINITY, ref = 0.0f;
    for (int r = threadIdx.x; r < parts; r += 256) {
      const float* p = part_of(r);
      m = fmaxf(m, p[kNarrowCols * D + c]);
      ref = fmaxf(ref, p[kNarrowCols * (D + 2) + c]);
    }
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) {
      m = fmaxf(m, __shfl_xor(m, d));
      ref = fmaxf(ref, __shfl_xor(ref, d));
    }
    if (__lane_id() == 0) {
      s_top[0][threadIdx.x / kWave] = m;
      s_top[1][threadIdx.x / kWave] = ref;
    }
    __syncthreads();
    m = fmaxf(fmaxf(s_top[0][0], s_top[0][1]), fmaxf(s_top[0][2], s_top[0][3]));
    ref = fmaxf(fmaxf(s_top[1][0], s_top[1][1]), fmaxf(s_top[1][2], s_top[1][3]));
    const int group = threadIdx.x / kVecs, d = threadIdx.x % kVecs;
    f32x4 o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float l = 0.0f;
#pragma unroll 4
    for (int r = group; r < parts; r += kGroups) {
      const float* p = part_of(r);
      const float pm = p[kNarrowCols * D + c], pl = p[kNarrowCols * (D + 1) + c];
      const f32x4 po = *reinterpret_cast<const f32x4*>(p + c * D + 4 * d);
      const float f = pm == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(pm - m);
      o += po * (f * unit_change(p[kNarrowCols * (D + 2) + c], ref));
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
      finish4<T>(a, u.row + c / a.group, g * a.group + c % a.group, 4 * d, o, m, l, ref);
    }
    __syncthreads();  // what LDS holds has been read
  }
}

}  // namespace kv
}  // namespace grm
