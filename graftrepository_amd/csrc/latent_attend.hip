// latent_attend.hip -- the latent schedule of a step, and absorbed attention over
// the latent cache (see latent_attend.hpp).
#include "latent_attend.hpp"

namespace grm {
namespace kv {

int latent_layout_of(const grm_kv_batch_desc* b, LatentLayout* out) {
  LatentLayout l{};
  int cus = 0;
  GRM_CHECK_RC(device_cus(&cus));
  const uint64_t rows = static_cast<uint64_t>(b->tokens);
  const uint64_t reqs = static_cast<uint64_t>(b->requests);
  const uint64_t busy = std::min(rows, reqs);
  const int64_t most = static_cast<int64_t>(std::max(1, b->max_new)) * b->heads;
  l.cols = most <= 16 ? 16 : most <= 32 ? 32 : most <= 64 ? 64 : kLatentCols;
  l.unit_tokens = std::max(1, l.cols / b->heads);
  for (int k = 0; k < 2; ++k) {
    l.runs[k] = (k + 1) * cus;
    l.starts[k] = (l.runs[k] + 7) / 8 * 8;
  }
  l.cap_units = std::min(rows, rows / l.unit_tokens + busy);
  l.cap_rows = std::min(rows, rows / kRowUnit + busy);
  // Pieces of dense rows are no shorter than a fourth of the even share (all tiles x
  // heads / 2 blocks to a CU), and only longer units are cut: into two pieces or more, so
  // that pieces are at most twice the units' tiles over that fourth.  (Items have a few
  // more, for a share that is rounded down; parts past the end would be whole units.)
  // With as many heads as blocks no unit is longer than the even share.
  const uint64_t slots = 2 * static_cast<uint64_t>(cus), heads = static_cast<uint64_t>(b->heads);
  l.cap_items = l.cap_rows + 4 * (slots / heads + 1);
  l.cap_parts = heads < slots ? std::min(l.cap_items, 8 * slots / heads) : 0;
  l.cap_row_joins = std::min(l.cap_rows, l.cap_parts / 2);
  l.reach = static_cast<int32_t>(std::min<int64_t>(
      static_cast<int64_t>(b->table_width) * b->block_tokens, 2 * static_cast<int64_t>(kMaxLen)));
  auto place = [&l](uint64_t bytes) {
    const uint64_t at = l.bytes;
    l.bytes += (bytes + 63) / 64 * 64;
    return at;
  };
  place(sizeof(LatentHead));
  for (int k = 0; k < 2; ++k) {
    l.at_units[k] = place(l.cap_units * sizeof(LatentUnit));
    l.at_first[k] = place((l.cap_units + 1) * 8);
    // a join is of a unit of its own and has an end of a run
    l.joins[k] = static_cast<int>(std::min<uint64_t>(l.runs[k] - 1, l.cap_units));
    l.at_starts[k] = place(static_cast<uint64_t>(l.starts[k]) * sizeof(LatentStart));
    l.at_joins[k] = place(static_cast<uint64_t>(l.joins[k]) * sizeof(LatentJoin));
  }
  for (int k = 0; k < 3; ++k) l.at_scan[k] = place((reqs + 1) * 4);
  l.at_lengths = place(l.cap_rows * 4);
  l.at_cuts = place(l.cap_items * sizeof(RowItem));
  l.at_items = place(l.cap_items * sizeof(RowItem));
  l.at_row_joins = place(l.cap_row_joins * sizeof(RowJoin));
  *out = l;
  return 0;
}

// ------------------------------------------------------------------- plan

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / kWave;

struct LatentPlanArgs {
  const int32_t* ctx_lens;
  const int32_t* new_lens;
  const int32_t* cu_new;
  char* work;
  int32_t requests, tokens, window, reach, unit_tokens, cap_units, cap_rows;
  int32_t heads, slots, cap_items, cap_parts, cap_row_joins;
  int32_t runs[2], starts[2], joins[2];
  uint64_t at_units[2], at_first[2], at_starts[2], at_joins[2], at_scan[3], at_lengths, at_cuts, at_items,
      at_row_joins;
};

// Exclusive sum over the block; the total in *sum.  Two barriers.
template <class N>
__device__ inline N block_sum(N v, N* sum, N* scratch) {
  const int lane = __lane_id(), wave = threadIdx.x / kWave;
  const N own = v;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const N o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  if (lane == kWave - 1) scratch[wave] = v;
  __syncthreads();
  N before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kPlanWaves; ++w) {
    const N t = scratch[w];
    before += w < wave ? t : 0;
    all += t;
  }
  __syncthreads();
  *sum = all;
  return v - own + before;
}

// Largest i in [0, n) with pre[i] <= x.
template <class N>
__device__ inline int last_of(const N* pre, int n, N x) {
  int lo = 0, len = n;
  while (len > 1) {
    const int half = len >> 1;
    if (pre[lo + half] <= x) lo += half;
    len -= half;
  }
  return lo;
}

// Sums over the requests of their units of `each` tokens, exclusive, in `at`; the
// total (sums past an int end at the lists' ends, which are never that long).
__device__ inline int64_t scan_units(const LatentPlanArgs& a, int each, int* at, int64_t* scratch) {
  int64_t all = 0;
  for (int base = 0; base < a.requests; base += kPlanThreads) {
    const int r = base + threadIdx.x;
    const int fresh = r < a.requests ? clamp_len(a.new_lens[r]) : 0;
    int64_t sum;
    const int64_t v = block_sum<int64_t>((fresh + each - 1) / each, &sum, scratch);
    if (r < a.requests) at[r] = static_cast<int>(min(all + v, static_cast<int64_t>(0x7fffffff)));
    all += sum;
  }
  return all;
}

// Unit i's first token within its request, its rows and how many: those past the
// batch's rows are none.
template <class U>
__device__ inline void unit_of(const LatentPlanArgs& a, const int* at, int i, int each, U* u) {
  u->request = last_of(at, a.requests, i);
  const int t0 = (i - at[u->request]) * each;
  const int fresh = clamp_len(a.new_lens[u->request]);
  u->pos = clamp_len(a.ctx_lens[u->request]) + t0;
  const int64_t row = static_cast<int64_t>(a.cu_new[u->request]) + t0;
  u->row = static_cast<int>(min(row, static_cast<int64_t>(a.tokens)));
  u->tokens = max(0, min(min(each, fresh - t0), a.tokens - u->row));
}

// Attention over the cache with k + 1 blocks to a CU.
__device__ inline void plan_cache(const LatentPlanArgs& a, int k, int* at, int64_t* scratch) {
  const int tid = threadIdx.x;
  auto* units = reinterpret_cast<LatentUnit*>(a.work + a.at_units[k]);
  auto* firsts = reinterpret_cast<int64_t*>(a.work + a.at_first[k]);
  const int n_units = static_cast<int>(
      min(scan_units(a, a.unit_tokens, at, scratch), static_cast<int64_t>(a.cap_units)));
  __syncthreads();
  int64_t tiles = 0;
  for (int base = 0; base < n_units; base += kPlanThreads) {
    const int i = base + tid;
    int64_t mine = 0, sum;
    LatentUnit u{};
    if (i < n_units) {
      unit_of(a, at, i, a.unit_tokens, &u);
      const int first = a.window > 0 ? max(0, u.pos + 1 - a.window) : 0;
      u.tile_lo = first / kLatentTile;
      const int hi = (min(u.pos + u.tokens, a.reach) + kLatentTile - 1) / kLatentTile;
      mine = max(1, hi - u.tile_lo);
    }
    const int64_t v = block_sum<int64_t>(mine, &sum, scratch);
    if (i < n_units) {
      units[i] = u;
      firsts[i] = tiles + v;
    }
    tiles += sum;
  }
  if (tid == 0) firsts[n_units] = tiles;
  __syncthreads();  // the lists are read back by other threads of this block
  LatentDeal deal;
  const int64_t most = (tiles + kLatentLeast - 1) / kLatentLeast;
  deal.used = static_cast<int>(min(most, static_cast<int64_t>(a.runs[k])));
  deal.each = deal.used ? tiles / deal.used : 0;
  deal.rem = deal.used ? static_cast<int>(tiles - deal.each * deal.used) : 0;
  // Few units: each gets runs of its own, where the longest of those is at most
  // kLatentChange tiles longer than an even run (which changes from unit to unit
  // somewhere, with queries to fetch and one part more).  The length is the least of 16
  // candidates with which all fit: the last one does, since tiles / length + units of them
  // do.
  __shared__ int s_runs[kPlanWaves], s_piece[kPlanThreads];
  const int own = a.runs[k] - n_units;
  bool whole_runs = false;
  if (n_units > 0 && n_units <= kPlanThreads && own > 0) {
    const int wave = tid / kWave, lane = tid % kWave;
    const int64_t least = max(static_cast<int64_t>(kLatentLeast), (tiles + a.runs[k] - 1) / a.runs[k]);
    const int64_t most_len = max(least, (tiles + own - 1) / own);
    auto length = [&](int c) { return least + (most_len - least) * c / (kPlanWaves - 1); };
    int64_t count = 0;
    for (int i = lane; i < n_units; i += kWave) {
      count += (firsts[i + 1] - firsts[i] + length(wave) - 1) / length(wave);
    }
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) count += __shfl_xor(count, d);
    if (lane == 0) s_runs[wave] = static_cast<int>(min(count, static_cast<int64_t>(0x7fffffff)));
    __syncthreads();
    int c = 0;
    while (c < kPlanWaves - 1 && s_runs[c] > a.runs[k]) ++c;
    const int64_t even = deal.each + (deal.rem > 0);
    whole_runs = length(c) <= even + kLatentChange;
    if (whole_runs) {
      const int64_t mine = tid < n_units ? firsts[tid + 1] - firsts[tid] : 0;
      int64_t sum;
      const int64_t v = block_sum<int64_t>((mine + length(c) - 1) / length(c), &sum, scratch);
      s_piece[tid] = static_cast<int>(v);
      deal.used = static_cast<int>(sum);
      __syncthreads();
    }
  }
  auto pieces_of = [&](int u) { return (u + 1 < n_units ? s_piece[u + 1] : deal.used) - s_piece[u]; };
  auto* to = reinterpret_cast<LatentStart*>(a.work + a.at_starts[k]);
  for (int i = tid; i < a.starts[k]; i += kPlanThreads) {
    // neighbouring runs to one XCD, to which every eighth entry goes
    const int xcd = i % 8, nth = i / 8;
    LatentStart s{};
    s.run = -1;
    if (nth < deal.used / 8 + (xcd < deal.used % 8)) {
      s.run = xcd * (deal.used / 8) + min(xcd, deal.used % 8) + nth;
      if (whole_runs) {
        s.unit = last_of(s_piece, n_units, s.run);
        s.first = firsts[s.unit];
        s.last = firsts[s.unit + 1];
        const int pieces = pieces_of(s.unit), piece = s.run - s_piece[s.unit];
        s.begin = s.first + (s.last - s.first) * piece / pieces;
        s.end = s.first + (s.last - s.first) * (piece + 1) / pieces;
      } else {
        s.begin = deal.begin(s.run);
        s.end = deal.begin(s.run + 1);
        s.unit = last_of(firsts, n_units, s.begin);
        s.first = firsts[s.unit];
        s.last = firsts[s.unit + 1];
      }
      const LatentUnit u = units[s.unit];
      s.request = u.request;
      s.row = u.row;
      s.tokens = u.tokens;
      s.pos = u.pos;
      s.tile_lo = u.tile_lo;
    }
    to[i] = s;
  }
  // Units that are cut: those of more than one run, or ends of runs that are the first
  // in a unit.
  auto* joins = reinterpret_cast<LatentJoin*>(a.work + a.at_joins[k]);
  int done = 0;
  const int ends = whole_runs ? n_units : deal.used - 1;
  for (int base = 0; base < ends; base += kPlanThreads) {
    const int e = base + tid;
    LatentJoin j{};
    bool cuts = false;
    if (e < ends && whole_runs) {
      const int pieces = pieces_of(e);
      cuts = pieces > 1 && units[e].tokens > 0;
      j = LatentJoin{s_piece[e], s_piece[e] + pieces - 1, units[e].row, units[e].tokens};
    } else if (e < ends) {
      const int64_t end = deal.begin(e + 1);
      const int u = last_of(firsts, n_units, end);
      if (firsts[u] < end && firsts[u] >= deal.begin(e)) {
        cuts = units[u].tokens > 0;
        j.from = e;
        j.to = deal.run(firsts[u + 1] - 1);
        j.row = units[u].row;
        j.tokens = units[u].tokens;
      }
    }
    int64_t sum;
    const int64_t v = block_sum<int64_t>(cuts, &sum, scratch);
    if (cuts) joins[done + v] = j;
    done += static_cast<int>(sum);
  }
  for (int i = done + tid; i < a.joins[k]; i += kPlanThreads) joins[i] = LatentJoin{};
}

// Attention over dense rows.
__device__ inline void plan_rows(const LatentPlanArgs& a, int* at, int64_t* scratch) {
  const int tid = threadIdx.x;
  auto* head = reinterpret_cast<LatentHead*>(a.work);
  int* lengths = reinterpret_cast<int*>(a.work + a.at_lengths);
  auto* cuts = reinterpret_cast<RowItem*>(a.work + a.at_cuts);
  auto* items = reinterpret_cast<RowItem*>(a.work + a.at_items);
  auto* row_joins = reinterpret_cast<RowJoin*>(a.work + a.at_row_joins);
  auto row_unit = [&](int i, RowItem* u) {
    unit_of(a, at, i, kRowUnit, u);
    const int first = a.window > 0 ? max(0, u->pos + 1 - a.window) : 0;
    return u->tokens > 0 ? max(1, (u->pos + u->tokens - first / kLatentTile * kLatentTile + kLatentTile - 1) / kLatentTile) : 0;
  };
  const int n_rows = static_cast<int>(
      min(scan_units(a, kRowUnit, at, scratch), static_cast<int64_t>(a.cap_rows)));
  __syncthreads();
  int64_t all = 0, sum;
  int longest = 0;
  for (int i = tid; i < n_rows; i += kPlanThreads) {
    RowItem u;
    lengths[i] = row_unit(i, &u);
    all += lengths[i];
    longest = max(longest, lengths[i]);
  }
  __shared__ int s_count[8], s_high[8], s_low[8], s_longest;
  if (tid < 8) {
    s_count[tid] = 0;
    s_high[tid] = 0;
    s_low[tid] = kMaxLen;
  }
  if (tid == 0) s_longest = 0;
  block_sum<int64_t>(all, &all, scratch);
  atomicMax(&s_longest, longest);
  __syncthreads();
  longest = s_longest;
  // The longest share of a piece: of eight parts of the even share the one by which
  // blocks, that take pieces longest first, are through first (as the wide units of
  // the 8-bit cache are cut).  Four tiles are added to a piece for its start and
  // end, which a piece of several has more of.
  const float even = static_cast<float>(all) * a.heads / a.slots;
  const float kOf[8] = {1.25f, 1.0f, 0.75f, 0.625f, 0.5f, 0.4f, 1.0f / 3.0f, 0.25f};
  auto share_of = [&](int k) {
    return max(kRowLeast, static_cast<int>(ceilf(fmaxf(even * kOf[k], 1.0f))));
  };
  int share = longest;
  if (even < static_cast<float>(longest)) {
    const int k = tid / 128;
    const float part = 1.0f / static_cast<float>(share_of(k));
    int count = 0, high = 0, low = kMaxLen;
    for (int i = tid % 128; i < n_rows; i += 128) {
      if (lengths[i] == 0) continue;
      const float cut = fmaxf(1.0f, ceilf(static_cast<float>(lengths[i]) * part));
      const int each = static_cast<int>(ceilf(static_cast<float>(lengths[i]) / cut));
      count += static_cast<int>(cut);
      high = max(high, each);
      low = min(low, each);
    }
    atomicAdd(&s_count[k], count);
    atomicMax(&s_high[k], high);
    atomicMin(&s_low[k], low);
    __syncthreads();
    float best = INFINITY;
    for (int c = -1; c < 8; ++c) {  // (-1: none is cut)
      constexpr float kEnds = 4.0f, kJoin = 4.0f;
      const float n = c < 0 ? static_cast<float>(n_rows) * a.heads : static_cast<float>(s_count[c]) * a.heads;
      const float extra = c < 0 ? 0.0f : static_cast<float>(s_count[c] - n_rows) * a.heads;
      const float rounds = n / a.slots, open = ceilf(rounds) - rounds;
      const float low_of = c < 0 ? 1.0f : static_cast<float>(s_low[c]);
      const float est = fmaxf((static_cast<float>(all) * a.heads + kEnds * n + 2.0f * kJoin * extra) / a.slots +
                                  open * (low_of + kEnds),
                              static_cast<float>(c < 0 ? longest : s_high[c]) + kEnds);
      if (est < best) {
        best = est;
        share = c < 0 ? longest : share_of(c);
      }
    }
  }
  share = max(share, 1);
  int done_items = 0, done_parts = 0, done_joins = 0;
  for (int base = 0; base < n_rows; base += kPlanThreads) {
    const int i = base + tid;
    RowItem u{};
    int cut = 0, n = 0;
    if (i < n_rows) {
      n = row_unit(i, &u);
      cut = n > 0 ? (n + share - 1) / share : 0;
    }
    const int from = done_items + static_cast<int>(block_sum<int64_t>(cut, &sum, scratch));
    done_items += static_cast<int>(sum);
    const int part = done_parts + static_cast<int>(block_sum<int64_t>(cut > 1 ? cut : 0, &sum, scratch));
    done_parts += static_cast<int>(sum);
    const int join = done_joins + static_cast<int>(block_sum<int64_t>(cut > 1, &sum, scratch));
    done_joins += static_cast<int>(sum);
    // The even share bounds all three lists; a unit past them would be one piece.
    const bool whole = cut <= 1 || part + cut > a.cap_parts || join >= a.cap_row_joins;
    for (int p = 0; p < cut && from + p < a.cap_items; ++p) {
      RowItem v = u;
      v.piece = whole ? 0 : p;
      v.pieces = whole ? 1 : cut;
      v.part = whole ? -1 : part + p;
      v.tiles = whole ? n : (n + cut - 1) / cut;
      if (whole && p) v.tokens = 0;
      cuts[from + p] = v;
    }
    if (cut > 1 && join < a.cap_row_joins) row_joins[join] = RowJoin{u.row, whole ? 0 : u.tokens, part, whole ? 0 : cut};
  }
  __syncthreads();
  // Longest first, where a block can sort them.
  const int n_items = min(done_items, a.cap_items);
  __shared__ __align__(16) int keys[kPlanThreads];
  if (n_items <= kPlanThreads) {
    // all different; no list is so long that pieces reach the bound
    const int mine = tid < n_items ? min(cuts[tid].tiles, (1 << 21) - 1) * kPlanThreads + kPlanThreads - 1 - tid : -1;
    keys[tid] = mine;
    __syncthreads();
    if (tid < n_items) {
      int rank = 0;
      for (int i = 0; i < n_items; i += 4) {
        const auto k = *reinterpret_cast<const u32x4*>(keys + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) rank += static_cast<int>(k[e]) > mine;
      }
      items[rank] = cuts[tid];
    }
  } else {
    for (int i = tid; i < n_items; i += kPlanThreads) items[i] = cuts[n_items - 1 - i];
  }
  if (tid == 0) {
    head->row_items = n_items;
    head->row_joins = min(done_joins, a.cap_row_joins);
  }
}

// Three blocks, a plan to each: latency (a scan over the requests, one over the units,
// a search for each run; the cuts of dense rows and their order).
__global__ __launch_bounds__(kPlanThreads) void latent_plan_kernel(LatentPlanArgs a) {
  __shared__ int64_t scratch[kPlanWaves];
  constexpr int kHeld = 4096;  // requests whose sums stay in LDS
  __shared__ int s_at[kHeld + 1];
  const int k = blockIdx.x;
  int* at = a.requests <= kHeld ? s_at : reinterpret_cast<int*>(a.work + a.at_scan[k]);
  if (k < 2) plan_cache(a, k, at, scratch);
  else plan_rows(a, at, scratch);
}

// ------------------------------------------------------- any shape of row

// One block to a (token, head): each of its wavefronts takes 64 rows in turn, a row
// to a lane for the scores and eight columns to a lane for the values.  Rows are
// read once for each head.
template <class T>
__global__ __launch_bounds__(256) void latent_any_kernel(LatentArgs a) {
  const int row = blockIdx.x, h = blockIdx.y;
  const int lane = __lane_id(), wave = threadIdx.x / kWave;
  const int values = a.rank + a.rope, bs = 1 << a.block_log2;
  __shared__ float s_q[640];
  __shared__ float s_p[4][kWave];
  __shared__ int64_t s_row[4][kWave];
  __shared__ float s_o[4][512];
  __shared__ float s_m[4], s_l[4];
  if (row >= a.cu_new[a.requests]) return;
  const int r = last_not_past(a.cu_new, a.requests, row);
  const int pos = clamp_len(a.ctx_lens[r]) + row - a.cu_new[r];
  const int first = a.window > 0 ? max(0, pos + 1 - a.window) : 0;
  const auto* q = static_cast<const typename T::store*>(a.q) + static_cast<int64_t>(row) * a.q_token +
                  static_cast<int64_t>(h) * a.q_head;
  for (int d = threadIdx.x; d < values; d += 256) s_q[d] = T::get(q[d]);
  __syncthreads();
  const auto* rows = reinterpret_cast<const typename T::store*>(a.rows);
  float m = -INFINITY, l = 0.0f, o[8] = {};
  const int reach = static_cast<int>(min(static_cast<int64_t>(pos), (static_cast<int64_t>(a.width) << a.block_log2) - 1));
  for (int t0 = first / kWave * kWave + wave * kWave; t0 <= reach; t0 += 4 * kWave) {
    const int key = t0 + lane;
    int64_t at = -1;
    if (key >= first && key <= reach) {
      const int block = a.table[static_cast<size_t>(r) * a.width + (key >> a.block_log2)];
      if (static_cast<uint64_t>(static_cast<int64_t>(block)) < a.blocks) {
        at = (static_cast<int64_t>(block) << a.block_log2) + (key & (bs - 1));
      }
    }
    float s = -INFINITY;
    if (at >= 0) {
      float dot = 0.0f;
      for (int d = 0; d < values; d += 8) {
        float x[8];
        get8<T, true>(rows + at * values + d, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) dot = fmaf(s_q[d + e], x[e], dot);
      }
      s = dot * a.scale * kLog2e;
      if (!(fabsf(dot) <= 3.4028235e38f)) s = NAN;
    }
    float top = s;
    const bool odd = __any(s != s);
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
    const float m2 = fmaxf(m, top);
    if (odd) l = NAN;
    if (m2 == -INFINITY) continue;
    const float keep = __builtin_amdgcn_exp2f(m - m2);
    m = m2;
    const float p = at >= 0 && s == s ? __builtin_amdgcn_exp2f(s - m2) : 0.0f;
    float sum = p;
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
    l = l * keep + sum;
    s_p[wave][lane] = p * a.unit.down;
    s_row[wave][lane] = s == s ? at : -1;
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] *= keep;
    if (8 * lane < a.rank) {
      for (int k = 0; k < kWave; ++k) {
        const int64_t from = s_row[wave][k];
        if (from < 0) continue;
        const float w = s_p[wave][k];
        float x[8];
        get8<T, true>(rows + from * values + 8 * lane, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = fmaf(w, x[e], o[e]);
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
  if (8 * lane < a.rank) {
#pragma unroll
    for (int e = 0; e < 8; ++e) s_o[wave][8 * lane + e] = o[e];
  }
  if (lane == 0) {
    s_m[wave] = m;
    s_l[wave] = l;
  }
  __syncthreads();
  const float top = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  float total = 0.0f, f[4];
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    f[w] = s_m[w] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s_m[w] - top);
    total += s_l[w] != s_l[w] ? NAN : f[w] * s_l[w];
  }
  auto* out = static_cast<typename T::store*>(a.out) + static_cast<int64_t>(row) * a.out_token +
              static_cast<int64_t>(h) * a.out_head;
  for (int d = threadIdx.x; d < a.rank; d += 256) {
    const float v = f[0] * s_o[0][d] + f[1] * s_o[1][d] + f[2] * s_o[2][d] + f[3] * s_o[3][d];
    out[d] = T::put(total == 0.0f ? 0.0f : v / total * a.unit.up);
  }
  if (a.lse && threadIdx.x == 0) {
    a.lse[static_cast<size_t>(row) * a.heads + h] =
        total == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(total)) * kLn2;
  }
}

// ------------------------------------------------------------- dispatch

// The matrix cores' shapes: (rank, rope) of (512, 64) and (256, 32), up to 128
// heads.
static bool latent_cores(const grm_latent_desc* c, const grm_kv_batch_desc* b) {
  return b->heads <= kLatentCols &&
         ((c->rank == 512 && c->rope == 64) || (c->rank == 256 && c->rope == 32));
}

// Wavefronts to a block of so many columns, and blocks to a CU.
static int latent_waves(int rank, int cols) { return cols == kLatentCols || (rank == 512 && cols == 64) ? 8 : 4; }
static int latent_per(const LatentLayout& l, int rank) { return latent_per_cu(rank, latent_waves(rank, l.cols)); }

static uint64_t latent_scratch(const LatentLayout& l, int rank) {
  return static_cast<uint64_t>(l.runs[latent_per(l, rank) - 1]) * 2 *
         latent_part_floats(l.cols, rank) * 4;
}

template <class T, int R, int P, int G, int NW>
static void launch_cols(const LatentArgs& a, hipStream_t stream) {
  typedef LatentShape<T, R, P, G, NW> S;
  const auto blocks = static_cast<unsigned>((a.runs + 7) / 8 * 8);
  latent_attend_kernel<T, R, P, G, NW><<<blocks, S::kThreads, 0, stream>>>(a);
  // real columns of a unit: whole tokens'
  const int cols = std::max(1, S::kCols / a.heads) * a.heads;
  if (a.joins == 0) return;
  // Many parts to a unit: four wavefronts share them (32 sessions of 40 columns, 16
  // parts on the average and 46 at most: 15 us without).
  const bool split = a.runs > 12 * a.joins;
  const dim3 grid(static_cast<unsigned>(a.joins), static_cast<unsigned>((cols + 15) / 16),
                  split ? R / 16 : R / 64);
  if (split) latent_join_kernel<T, R, S::kCols, true><<<grid, 256, 0, stream>>>(a, S::kBias);
  else latent_join_kernel<T, R, S::kCols, false><<<grid, 256, 0, stream>>>(a, S::kBias);
}

template <class T, int R, int P>
static void launch_latent(const LatentArgs& a, int cols, hipStream_t stream) {
  if (cols == 16) launch_cols<T, R, P, 4, 4>(a, stream);
  else if (cols == 32) launch_cols<T, R, P, 2, 4>(a, stream);
  else if (cols == 64) launch_cols<T, R, P, R == 512 ? 2 : 1, R == 512 ? 8 : 4>(a, stream);
  else launch_cols<T, R, P, 1, 8>(a, stream);
}

template <class T>
static void launch_latent_any(const LatentArgs& a, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(a.tokens), static_cast<unsigned>(a.heads));
  latent_any_kernel<T><<<grid, 256, 0, stream>>>(a);
}

}  // namespace kv
}  // namespace grm

using namespace grm::kv;

extern "C" int grm_hip_latent_work_bytes(const grm_kv_batch_desc* batch, uint64_t* out_bytes) {
  if (!out_bytes) return grm::fail(-1, "null output pointer");
  GRM_CHECK_RC(check_batch(batch, false));
  LatentLayout l;
  GRM_CHECK_RC(latent_layout_of(batch, &l));
  *out_bytes = l.bytes;
  grm::clear_error();
  return 0;
}

extern "C" int grm_hip_latent_plan(const grm_kv_batch_desc* b, void* work, uint64_t work_bytes,
                                   void* stream) {
  GRM_CHECK_RC(check_batch(b, true));
  if (b->requests == 0) {
    grm::clear_error();
    return 0;
  }
  if (!work || !aligned16(work)) return grm::fail(-1, "latent work must be 16-byte aligned");
  LatentLayout l;
  GRM_CHECK_RC(latent_layout_of(b, &l));
  if (work_bytes < l.bytes) return grm::fail(-1, "work is smaller than grm_hip_latent_work_bytes");
  LatentPlanArgs a{};
  a.ctx_lens = b->ctx_lens;
  a.new_lens = b->new_lens;
  a.cu_new = b->cu_new;
  a.work = static_cast<char*>(work);
  a.requests = b->requests;
  a.tokens = b->tokens;
  a.window = b->window;
  a.reach = l.reach;
  a.unit_tokens = l.unit_tokens;
  a.cap_units = static_cast<int32_t>(l.cap_units);
  a.cap_rows = static_cast<int32_t>(l.cap_rows);
  a.heads = b->heads;
  a.slots = l.runs[1];
  a.cap_items = static_cast<int32_t>(l.cap_items);
  a.cap_parts = static_cast<int32_t>(l.cap_parts);
  a.cap_row_joins = static_cast<int32_t>(l.cap_row_joins);
  for (int k = 0; k < 2; ++k) {
    a.runs[k] = l.runs[k];
    a.starts[k] = l.starts[k];
    a.joins[k] = l.joins[k];
    a.at_units[k] = l.at_units[k];
    a.at_first[k] = l.at_first[k];
    a.at_starts[k] = l.at_starts[k];
    a.at_joins[k] = l.at_joins[k];
  }
  for (int k = 0; k < 3; ++k) a.at_scan[k] = l.at_scan[k];
  a.at_lengths = l.at_lengths;
  a.at_cuts = l.at_cuts;
  a.at_items = l.at_items;
  a.at_row_joins = l.at_row_joins;
  latent_plan_kernel<<<3, kPlanThreads, 0, static_cast<hipStream_t>(stream)>>>(a);
  GRM_HIP_CHECK(hipGetLastError());
  grm::clear_error();
  return 0;
}

extern "C" int grm_hip_latent_attend_bytes(const grm_latent_desc* c, const grm_kv_batch_desc* b,
                                           uint64_t* out_bytes) {
  if (!out_bytes) return grm::fail(-1, "null output pointer");
  GRM_CHECK_RC(check_latent_pair(c, b, false));
  LatentLayout l;
  GRM_CHECK_RC(latent_layout_of(b, &l));
  *out_bytes = latent_cores(c, b) ? latent_scratch(l, c->rank) : 0;
  grm::clear_error();
  return 0;
}

extern "C" int grm_hip_latent_attend(const grm_latent_desc* c, const grm_kv_batch_desc* b,
                                     const void* work, uint64_t work_bytes, const void* q,
                                     int64_t q_token_stride, int64_t q_head_stride, void* out,
                                     int64_t out_token_stride, int64_t out_head_stride, float* lse,
                                     float softmax_scale, void* scratch, uint64_t scratch_bytes,
                                     void* stream) {
  GRM_CHECK_RC(check_latent_pair(c, b, true));
  if (!(softmax_scale - softmax_scale == 0.0f)) return grm::fail(-1, "softmax_scale must be finite");
  if (b->requests == 0 || b->tokens == 0) {
    grm::clear_error();
    return 0;
  }
  if (!q || !out) return grm::fail(-1, "null queries or output");
  if (!aligned16(q) || !aligned16(out) ||
      (q_token_stride | q_head_stride | out_token_stride | out_head_stride) % 8 != 0) {
    return grm::fail(-1, "queries and output: 16-byte aligned rows");
  }
  const bool cores = latent_cores(c, b);
  if (!cores) GRM_CHECK_RC(check_blocks(static_cast<uint64_t>(b->tokens)));
  if (cores && (!work || !aligned16(work))) {
    return grm::fail(-1, "latent work must be 16-byte aligned");
  }
  LatentLayout l;
  GRM_CHECK_RC(latent_layout_of(b, &l));
  const int per = latent_per(l, c->rank);
  if (cores) {
    if (work_bytes < l.bytes) return grm::fail(-1, "work is smaller than grm_hip_latent_work_bytes");
    if (!scratch || !aligned16(scratch) || scratch_bytes < latent_scratch(l, c->rank)) {
      return grm::fail(-1, "scratch is smaller than grm_hip_latent_attend_bytes, or not 16-byte aligned");
    }
  }
  LatentArgs a{};
  a.rows = static_cast<const char*>(c->rows);
  a.q = q;
  a.out = out;
  a.lse = lse;
  a.cu_new = b->cu_new;
  a.ctx_lens = b->ctx_lens;
  a.table = b->table_width ? b->block_table : b->cu_new;  // entry 0 is asked for all the same
  a.work = static_cast<const char*>(work);
  a.parts = static_cast<float*>(scratch);
  a.q_token = q_token_stride;
  a.q_head = q_head_stride;
  a.out_token = out_token_stride;
  a.out_head = out_head_stride;
  a.blocks = c->blocks;
  a.at_units = l.at_units[per - 1];
  a.at_first = l.at_first[per - 1];
  a.at_starts = l.at_starts[per - 1];
  a.at_joins = l.at_joins[per - 1];
  a.unit = sum_unit(c->dtype, l.reach);
  a.scale = softmax_scale;
  a.requests = b->requests;
  a.width = b->table_width;
  a.tokens = b->tokens;
  a.window = b->window;
  a.heads = b->heads;
  a.rank = c->rank;
  a.rope = c->rope;
  a.block_log2 = block_log2(c->block_tokens);
  a.runs = l.runs[per - 1];
  a.joins = l.joins[per - 1];
  const auto s = static_cast<hipStream_t>(stream);
  const bool bf = c->dtype == grm::kBF16;
  if (!cores) {
    if (bf) launch_latent_any<BF16>(a, s);
    else launch_latent_any<F16>(a, s);
  } else if (c->rank == 512) {
    if (bf) launch_latent<BF16, 512, 64>(a, l.cols, s);
    else launch_latent<F16, 512, 64>(a, l.cols, s);
  } else {
    if (bf) launch_latent<BF16, 256, 32>(a, l.cols, s);
    else launch_latent<F16, 256, 32>(a, l.cols, s);
  }
  GRM_HIP_CHECK(hipGetLastError());
  grm::clear_error();
  return 0;
}
