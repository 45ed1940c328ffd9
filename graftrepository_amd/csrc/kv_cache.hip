// kv_cache.hip -- the 8-bit key/value cache: a step's plan (block tables,
// slot map, schedule), the quantising append, and the dense read back.
//
// The cache's law is the header's (include/grm_hip_router.h).  The plan is
// latency, the append and the read are bytes: append reads the new values
// once, and writes a byte for each; read loads a byte per value and writes
// two or four.

#include "rotary.hpp"

#include <mutex>
#include <type_traits>

namespace grm {
namespace kv {

// ------------------------------------------------------------ descriptors

int device_cus(int* out) {
  static std::mutex m;
  static int cus[64] = {0};
  int dev = 0;
  GRM_HIP_CHECK(hipGetDevice(&dev));
  if (dev < 0 || dev >= 64) return fail(-1, "device index past 63");
  std::lock_guard<std::mutex> lock(m);
  if (cus[dev] == 0) {
    int n = 0;
    GRM_HIP_CHECK(hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev));
    cus[dev] = n;
  }
  *out = cus[dev];
  return 0;
}

static bool good_block(int n) { return n == 16 || n == 32 || n == 64 || n == 128; }

int check_batch(const grm_kv_batch_desc* b, bool with_arrays) {
  if (!b) return fail(-1, "null batch");
  if (b->requests < 0 || b->tokens < 0 || b->max_new < 0 || b->table_width < 0 || b->window < 0) {
    return fail(-1, "negative size in the batch");
  }
  if (b->requests > (1 << 24) || b->tokens > kMaxLen || b->table_width > (1 << 26)) {
    return fail(-1, "batch too large");
  }
  if (!good_block(b->block_tokens)) return fail(-1, "block_tokens must be 16, 32, 64 or 128");
  if (b->kv_heads <= 0 || b->heads <= 0 || b->heads % b->kv_heads != 0) {
    return fail(-1, "heads must be a positive multiple of kv_heads");
  }
  if (b->heads > 65535) return fail(-1, "more than 65535 heads");
  const int64_t columns = static_cast<int64_t>(b->table_width) * b->block_tokens / kTile + 2;
  if (columns * b->requests > 0x7fffffff) return fail(-1, "batch too large");
  if (!with_arrays || b->requests == 0) return 0;
  if (!b->ctx_lens || !b->new_lens || !b->cu_new || !b->work) {
    return fail(-1, "null array in the batch");
  }
  if (b->table_width > 0 && !b->block_table) return fail(-1, "null block table");
  if (!aligned16(b->work)) return fail(-1, "work must be 16-byte aligned");
  if (b->free_count > 0x7fffffffull) return fail(-1, "free list too long");
  if (b->free_list || b->free_head) {
    if (!b->free_list && b->free_count) return fail(-1, "null free list");
    if (!b->free_head || !b->free_head_out) return fail(-1, "a free list needs both heads");
    if (b->free_head == b->free_head_out) {
      return fail(-1, "free_head_out must not be free_head: other blocks still read it");
    }
  }
  return 0;
}

int check_cache(const grm_kv_cache_desc* c) {
  if (!c) return fail(-1, "null cache");
  if (!good_block(c->block_tokens)) return fail(-1, "block_tokens must be 16, 32, 64 or 128");
  if (c->kv_heads <= 0 || c->kv_heads > 65535) return fail(-1, "bad kv_heads");
  if (c->head_dim <= 0 || c->head_dim > 256 || c->head_dim % 16 != 0) {
    return fail(-1, "head_dim must be a multiple of 16, at most 256");
  }
  if (c->blocks == 0 || c->blocks > 0x7fffffffull) return fail(-1, "bad block count");
  if (!c->k_codes || !c->v_codes || !c->k_scales || !c->v_scales) {
    return fail(-1, "null array in the cache");
  }
  if (!aligned16(c->k_codes) || !aligned16(c->v_codes)) {
    return fail(-1, "code arrays must be 16-byte aligned");
  }
  return 0;
}

int check_pair(const grm_kv_cache_desc* c, const grm_kv_batch_desc* b, bool with_arrays) {
  GRM_CHECK_RC(check_cache(c));
  GRM_CHECK_RC(check_batch(b, with_arrays));
  if (c->block_tokens != b->block_tokens || c->kv_heads != b->kv_heads) {
    return fail(-1, "cache and batch differ in block_tokens or kv_heads");
  }
  return 0;
}

int layout_of(const grm_kv_batch_desc* b, Layout* out) {
  Layout l{};
  int cus = 0;
  GRM_CHECK_RC(device_cus(&cus));
  l.group = b->heads / b->kv_heads;
  l.reach = static_cast<int32_t>(std::min<int64_t>(
      static_cast<int64_t>(b->table_width) * b->block_tokens, 2 * static_cast<int64_t>(kMaxLen)));
  const uint64_t rows = static_cast<uint64_t>(b->tokens);
  const uint64_t reqs = static_cast<uint64_t>(b->requests);
  const uint64_t busy = std::min(rows, reqs);  // requests that bring tokens
  // A request of n tokens touches at most n / block_tokens + 2 blocks, and
  // no more than n.
  l.cap_append = std::min(rows, rows / b->block_tokens + 2 * busy);
  l.cap_units = l.group <= kNarrowCols ? busy : 0;
  l.wide_blocks = std::max(1, 2 * cus / b->kv_heads);
  for (int k = 0; k < 2; ++k) l.runs[k] = narrow_runs(cus, b->kv_heads, k + 1);
  const bool wide = static_cast<int64_t>(b->max_new) * l.group > kNarrowCols;
  l.wide_tokens = wide && l.group <= kWideCols ? kWideCols / l.group : 0;
  if (l.wide_tokens) {
    l.cap_wide = rows / l.wide_tokens + busy;
    // Only units longer than the share C = all / (4 x blocks) are cut, into
    // at most 2 x length / C parts; and only into parts of kLeastShare tiles.
    // A unit's tiles are the table's or, with a window, what it spans.
    uint64_t tiles = (static_cast<uint64_t>(l.reach) + kTile - 1) / kTile;
    if (b->window) {
      tiles = std::min(tiles, (static_cast<uint64_t>(b->window) + l.wide_tokens + 2 * kTile) / kTile);
    }
    if (tiles > kLeastShare) {
      l.cap_parts = std::min(8 * static_cast<uint64_t>(l.wide_blocks) + 8,
                             l.cap_wide * ((tiles + kLeastShare - 1) / kLeastShare));
    }
    l.cap_joins = l.cap_parts / 2;
    l.cap_items = l.cap_wide + l.cap_parts;
  }
  auto place = [&l](uint64_t bytes) {
    const uint64_t at = l.bytes;
    l.bytes += (bytes + 63) / 64 * 64;
    return at;
  };
  place(sizeof(SchedHead));
  l.at_append = place(l.cap_append * sizeof(AppendItem));
  l.at_units = place(l.cap_units * sizeof(NarrowUnit));
  l.at_tiles = place((l.cap_units + 1) * 4);
  for (int k = 0; k < 2; ++k) {
    l.at_run_units[k] = place(l.cap_units ? l.runs[k] * 4 : 0);
  }
  l.at_scan = place(l.wide_tokens ? (reqs + 1) * 4 : 0);
  l.at_wide = place(l.cap_wide * sizeof(WideUnit));
  l.at_items = place(l.cap_items * sizeof(WideItem));
  l.at_joins = place(l.cap_joins * sizeof(WideJoin));
  *out = l;
  return 0;
}

// ------------------------------------------------------------------- plan
//
// One launch.  Blocks 1.. each fill kPlanTokens rows of the slot map; every
// one of them repeats the scan over the lengths (8 bytes a request, from
// L2), which is cheaper than a second launch.  Block 0 writes the prefix
// sums, the new head of the free list and the attention schedule.  A new
// block begins at exactly one new token (its place is 0), so that token's
// thread enters it in the table: nothing is written twice, and no atomics.

constexpr int kPlanThreads = 1024;
constexpr int kPlanTokens = 4096;
constexpr int kPerThread = 4;
constexpr int kPlanChunk = kPlanThreads * kPerThread;  // requests to a scan step

struct PlanArgs {
  const int32_t* ctx_lens;
  const int32_t* new_lens;
  int32_t* table;
  const int32_t* free_list;
  const int32_t* free_head;
  int32_t* free_head_out;
  int32_t* cu_new;
  int64_t* slots;
  int32_t* positions;
  char* work;
  int32_t requests, width, tokens, window, reach;
  int32_t free_count, group, wide_tokens, kv_heads;
  int32_t wide_blocks, block_log2;
  int32_t cap_append, cap_units, cap_wide, cap_items, cap_joins, cap_parts;
  int32_t runs[2];
  uint64_t at_append, at_units, at_tiles, at_run_units[2], at_scan, at_wide, at_items, at_joins;
};

// Sums of rows and wide units stop at the largest int: lengths of more tokens
// than the batch has rows leave what follows past its end.  The other sums are
// looked at only before that.
__device__ inline int add(int a, int b) { return __builtin_elementwise_add_sat(a, b); }

// Exclusive sums over the block of N values per thread (0 or more); totals to
// `sum`.  Bits of STOPS: those that stop.  `scratch` holds N * 16 ints.  Two
// barriers.
template <int N, unsigned STOPS>
__device__ void block_scan(int (&v)[N], int (&sum)[N], int* scratch) {
  const int lane = __lane_id(), wave = threadIdx.x / kWave;
  constexpr int kWaves = kPlanThreads / kWave;
  int own[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    own[k] = v[k];
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const int o = __shfl_up(v[k], d);
      if (lane >= d) v[k] = STOPS >> k & 1 ? add(v[k], o) : v[k] + o;
    }
    if (lane == kWave - 1) scratch[k * kWaves + wave] = v[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) {
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const int t = scratch[k * kWaves + w];
      const int mine = w < wave ? t : 0;
      before = STOPS >> k & 1 ? add(before, mine) : before + mine;
      all = STOPS >> k & 1 ? add(all, t) : all + t;
    }
    v[k] = STOPS >> k & 1 ? add(v[k] - own[k], before) : v[k] - own[k] + before;
    sum[k] = all;
  }
  __syncthreads();
}

__device__ inline int wave_sum(int v) {
#pragma unroll
  for (int d = kWave / 2; d > 0; d >>= 1) v += __shfl_xor(v, d);
  return v;
}

struct Lens {
  int ctx, fresh, held, need, touched;
};

__device__ inline Lens lens_of(const PlanArgs& a, int r) {
  Lens l{0, 0, 0, 0, 0};
  if (r >= a.requests) return l;
  l.ctx = clamp_len(a.ctx_lens[r]);
  l.fresh = clamp_len(a.new_lens[r]);
  const int bs = 1 << a.block_log2;
  l.held = (l.ctx + bs - 1) >> a.block_log2;
  if (l.fresh > 0) {
    const int last = (l.ctx + l.fresh + bs - 1) >> a.block_log2;
    l.need = max(0, min(last, a.width) - l.held);
    l.touched = last - (l.ctx >> a.block_log2);
  }
  return l;
}

// Largest i in [0, n) with pre[i] <= x (pre ascending, pre[0] <= x).
__device__ inline int upper(const int* pre, int n, int x) {
  int lo = 0, len = n;
  while (len > 1) {
    const int half = len >> 1;
    if (pre[lo + half] <= x) lo += half;
    len -= half;
  }
  return lo;
}

// Key tiles [lo, hi) of `tile` tokens that query tokens [t0, t0 + n) of a
// request see, as far as the table has blocks; one at least.
__device__ inline void tiles_of(const PlanArgs& a, int tile, int ctx, int t0, int n, int* lo,
                                int* hi) {
  const int last = ctx + t0 + n;  // keys before this are seen by the last token
  const int first = a.window > 0 ? max(0, ctx + t0 + 1 - a.window) : 0;
  *lo = first / tile;
  *hi = max(*lo + 1, (min(last, a.reach) + tile - 1) / tile);
}

__device__ void plan_slots(const PlanArgs& a, int t0, int* lds) {
  int* s_cu = lds;                     // [kPlanChunk + 1]
  int* s_ctx = s_cu + kPlanChunk + 1;  // [kPlanChunk]
  int* s_need = s_ctx + kPlanChunk;
  int* s_touch = s_need + kPlanChunk;
  int* scratch = s_touch + kPlanChunk;  // [3 * 16]
  const int bs = 1 << a.block_log2;
  const int t1 = min(t0 + kPlanTokens, a.tokens);
  const int head = a.free_head ? max(0, *a.free_head) : 0;
  AppendItem* appends = reinterpret_cast<AppendItem*>(a.work + a.at_append);
  int done_new = 0, done_need = 0, done_touch = 0;
  int filled = t0;  // rows before this have their request
  for (int base = 0; base < a.requests && done_new < t1; base += kPlanChunk) {
    const int r0 = base + static_cast<int>(threadIdx.x) * kPerThread;
    Lens l[kPerThread];
    int v[3] = {0, 0, 0}, sum[3];
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
      l[j] = lens_of(a, r0 + j);
      v[0] = add(v[0], l[j].fresh);
      v[1] += l[j].need;
      v[2] += l[j].touched;
    }
    block_scan<3, 1u>(v, sum, scratch);
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
      const int i = threadIdx.x * kPerThread + j;
      s_cu[i] = add(done_new, v[0]);
      s_ctx[i] = l[j].ctx;
      s_need[i] = done_need + v[1];
      s_touch[i] = done_touch + v[2];
      v[0] = add(v[0], l[j].fresh);
      v[1] += l[j].need;
      v[2] += l[j].touched;
    }
    __syncthreads();
    const int here = min(kPlanChunk, a.requests - base);
    const int end = min(t1, add(done_new, sum[0]));
    for (int i = max(t0, done_new) + static_cast<int>(threadIdx.x); i < end; i += kPlanThreads) {
      // the last request whose first row is not past i: it has a token there
      const int k = upper(s_cu, here, i);
      const int r = base + k, ctx = s_ctx[k], t = i - s_cu[k];
      const int pos = ctx + t, j = pos >> a.block_log2, place = pos & (bs - 1);
      const int held = (ctx + bs - 1) >> a.block_log2;
      int block = -1;
      if (j < a.width) {
        if (a.free_head && j >= held) {
          const int at = head + s_need[k] + j - held;
          block = at >= 0 && at < a.free_count ? a.free_list[at] : -1;
          if (place == 0) a.table[static_cast<size_t>(r) * a.width + j] = block;
        } else {
          block = a.table[static_cast<size_t>(r) * a.width + j];
        }
      }
      if (a.slots) a.slots[i] = block < 0 ? -1 : static_cast<int64_t>(block) * bs + place;
      if (a.positions) a.positions[i] = pos;
      if (i == a.tokens - 1) {
        // The last row: blocks past it, of lengths longer than the batch has
        // rows, are in no entry of the list.
        reinterpret_cast<SchedHead*>(a.work)->appends =
            min(s_touch[k] + j - (ctx >> a.block_log2) + 1, a.cap_append);
      }
      if (place == 0 || t == 0) {
        const int at = s_touch[k] + j - (ctx >> a.block_log2);
        const int next = k + 1 < here ? s_cu[k + 1] : add(done_new, sum[0]);
        if (static_cast<unsigned>(at) < static_cast<unsigned>(a.cap_append)) {
          AppendItem it;
          it.block = block;
          it.row = i;
          it.place = place;
          it.count = min(min(bs - place, next - i), a.tokens - i);
          appends[at] = it;
        }
      }
    }
    filled = max(filled, end);
    done_new = add(done_new, sum[0]);
    done_need += sum[1];
    done_touch += sum[2];
    __syncthreads();
  }
  for (int i = max(t0, filled) + static_cast<int>(threadIdx.x); i < t1; i += kPlanThreads) {
    if (a.slots) a.slots[i] = -1;
    if (a.positions) a.positions[i] = -1;
  }
}

constexpr int kScanInts = 6 * 16 + 32;  // scan sums, and the candidates' counts
constexpr int kPlanInts = 4 * kPlanChunk + 256;

// The schedule, by one block, beside the blocks that write slots and positions:
// one scan over the requests for all sums, four requests to a thread, then the
// units.  Latency: 256 requests of one token take 10.4 us, 4001 of 1 to 300
// tokens 27.4, four prompts whose units are cut 12.
__device__ void plan_schedule(const PlanArgs& a, int* lds) {
  if (a.requests == 0) {
    // no schedule, which nobody reads; the lists that others go on from
    if (threadIdx.x == 0) {
      if (a.cu_new) a.cu_new[0] = 0;
      if (a.free_head && a.free_head_out) *a.free_head_out = max(0, *a.free_head);
    }
    return;
  }
  int* scratch = lds;                                     // [kScanInts]
  int* tiles_lds = lds + kScanInts;                       // [kPlanChunk]
  int* wide_lds = tiles_lds + kPlanChunk;                 // the rest
  constexpr int kWideInts = kPlanInts - kScanInts - kPlanChunk;
  SchedHead* head = reinterpret_cast<SchedHead*>(a.work);
  NarrowUnit* units = reinterpret_cast<NarrowUnit*>(a.work + a.at_units);
  int* tiles = reinterpret_cast<int*>(a.work + a.at_tiles);
  int* wide_at = reinterpret_cast<int*>(a.work + a.at_scan);
  const bool wide_fits = a.requests < kWideInts;
  // new tokens, blocks needed, touched blocks, narrow tiles, wide units,
  // narrow units
  int done[6] = {0, 0, 0, 0, 0, 0};
  for (int base = 0; base < a.requests; base += kPlanChunk) {
    const int r0 = base + static_cast<int>(threadIdx.x) * kPerThread;
    Lens l[kPerThread];
    int lo[kPerThread], hi[kPerThread], wide[kPerThread];
    bool narrow[kPerThread];
    int v[6] = {0, 0, 0, 0, 0, 0}, sum[6];
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
      l[j] = lens_of(a, r0 + j);
      narrow[j] = l[j].fresh > 0 && a.cap_units > 0 &&
                  static_cast<int64_t>(l[j].fresh) * a.group <= kNarrowCols;
      lo[j] = hi[j] = 0;
      if (narrow[j]) {
        tiles_of(a, narrow_tile(1 << a.block_log2), l[j].ctx, 0, l[j].fresh, &lo[j], &hi[j]);
      }
      wide[j] = a.wide_tokens && l[j].fresh > 0 && !narrow[j]
                    ? (l[j].fresh + a.wide_tokens - 1) / a.wide_tokens : 0;
      v[0] = add(v[0], l[j].fresh);
      v[1] += l[j].need;
      v[2] += l[j].touched;
      v[3] += hi[j] - lo[j];
      v[4] = add(v[4], wide[j]);
      v[5] += narrow[j];
    }
    block_scan<6, 0x11u>(v, sum, scratch);
#pragma unroll
    for (int k = 0; k < 6; ++k) v[k] = k % 4 == 0 ? add(v[k], done[k]) : v[k] + done[k];
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
      const int r = r0 + j;
      if (r < a.requests) {
        a.cu_new[r] = v[0];
        if (a.wide_tokens) {
          wide_at[r] = v[4];
          if (wide_fits) wide_lds[r] = v[4];
        }
        if (narrow[j] && static_cast<unsigned>(v[5]) < static_cast<unsigned>(a.cap_units)) {
          NarrowUnit n;
          n.request = r;
          n.row = v[0];
          n.tokens = max(0, min(l[j].fresh, a.tokens - n.row));
          n.tile_lo = lo[j];
          n.ctx = l[j].ctx;
          n.pad[0] = n.pad[1] = n.pad[2] = 0;
          units[v[5]] = n;
          tiles[v[5]] = v[3];
          if (v[5] < kPlanChunk) tiles_lds[v[5]] = v[3];
        }
      }
      v[0] = add(v[0], l[j].fresh);
      v[2] += l[j].touched;
      v[3] += hi[j] - lo[j];
      v[4] = add(v[4], wide[j]);
      v[5] += narrow[j];
    }
#pragma unroll
    for (int k = 0; k < 6; ++k) done[k] = k % 4 == 0 ? add(done[k], sum[k]) : done[k] + sum[k];
  }
  const int done_units = max(0, min(done[5], a.cap_units));
  const int wide_units = done[4];
  const bool tiles_fit = done_units < kPlanChunk;
  if (threadIdx.x == 0) {
    a.cu_new[a.requests] = done[0];
    tiles[done_units] = done[3];
    if (tiles_fit) tiles_lds[done_units] = done[3];
    if (a.wide_tokens) {
      wide_at[a.requests] = wide_units;
      if (wide_fits) wide_lds[a.requests] = wide_units;
    }
    if (a.free_head) {
      const int at = max(0, *a.free_head);
      const int left = max(0, a.free_count - at);
      *a.free_head_out = at + min(left, max(0, done[1]));
    }
    if (done[0] < a.tokens || a.tokens == 0) head->appends = min(done[2], a.cap_append);
    head->units = done_units;
    head->narrow_tiles = done[3];
    head->items = 0;
    head->joins = 0;
  }
  __syncthreads();  // the lists are read back by other threads of this block

  // The unit that each run of the narrow kernel begins in; 0 where it is empty.
  if (a.cap_units > 0) {
    const int* from = tiles_fit ? tiles_lds : tiles;
    for (int k = 0; k < 2; ++k) {
      const Deal deal(done[3], a.runs[k]);
      int* run_units = reinterpret_cast<int*>(a.work + a.at_run_units[k]);
      for (int r = threadIdx.x; r < a.runs[k]; r += kPlanThreads) {
        const int begin = deal.begin(r);
        run_units[r] = begin < deal.begin(r + 1) ? upper(from, done_units, begin) : 0;
      }
    }
  }
  if (wide_units == 0) return;

  // Longest share C of a wide item, from kCands parts of the even share.
  // Blocks take items longest first, so that a candidate's time is estimated
  // as its mean load and, where the last round is not full, its shortest
  // item; no less than its longest.  Four tiles are added to each item for its
  // start and end.
  constexpr int kCands = 8;
  const float kOf[kCands] = {1.25f, 1.125f, 1.0f, 0.625f, 0.5f, 0.4f, 1.0f / 3.0f, 0.25f};
  // Of each candidate: items, longest, shortest; then all tiles and the longest
  // unit.
  int* count = lds + 6 * 16;
  int* longest_of = count + kCands;
  int* shortest_of = longest_of + kCands;
  auto* total_at = reinterpret_cast<unsigned long long*>(shortest_of + kCands);
  int* longest_at = shortest_of + kCands + 2;
  if (threadIdx.x < 3 * kCands + 3) {
    const int k = static_cast<int>(threadIdx.x) - 2 * kCands;
    count[threadIdx.x] = k >= 0 && k < kCands ? kMaxLen : 0;
  }
  __syncthreads();
  // Each unit's request is searched for once, in LDS where the sums fit.
  const int* wide_from = wide_fits ? wide_lds : wide_at;
  WideUnit* wide = reinterpret_cast<WideUnit*>(a.work + a.at_wide);
  const int stored = min(wide_units, a.cap_wide);
  unsigned long long mine = 0;  // long prompts of many: past 32 bits
  int longest = 0;
  for (int u = threadIdx.x; u < stored; u += kPlanThreads) {
    WideUnit w;
    w.request = upper(wide_from, a.requests, u);
    w.t0 = (u - wide_from[w.request]) * a.wide_tokens;
    const int ctx = clamp_len(a.ctx_lens[w.request]);
    const int n = min(a.wide_tokens, clamp_len(a.new_lens[w.request]) - w.t0);
    tiles_of(a, kTile, ctx, w.t0, n, &w.lo, &w.hi);
    wide[u] = w;
    mine += w.hi - w.lo;
    longest = max(longest, w.hi - w.lo);
  }
#pragma unroll
  for (int d = kWave / 2; d > 0; d >>= 1) {
    mine += __shfl_xor(mine, d);
    longest = max(longest, __shfl_xor(longest, d));
  }
  if (__lane_id() == 0) {
    atomicAdd(total_at, mine);
    atomicMax(longest_at, longest);
  }
  __syncthreads();
  longest = *longest_at;
  const unsigned long long total = *total_at;
  const int even = static_cast<int>(
      min(max(1ull, (total + a.wide_blocks - 1) / a.wide_blocks),
          static_cast<unsigned long long>(kMaxLen)));
  int share = longest;
  if (even < longest) {  // else none is cut
    auto candidate = [&](float of) {
      return max(kLeastShare, static_cast<int>(ceilf(static_cast<float>(even) * of)));
    };
    // A candidate to a wavefront, or to several that share the units.
    constexpr int kShare = kPlanThreads / kWave / kCands;
    static_assert(kShare >= 1, "a wavefront to each candidate");
    const int wave = static_cast<int>(threadIdx.x) / kWave, mine_k = wave % kCands;
    if (wave < kShare * kCands) {
      const float part = 1.0f / static_cast<float>(candidate(kOf[mine_k]));
      int items = 0, high = 0, low = kMaxLen;
      for (int u = wave / kCands * kWave + __lane_id(); u < stored; u += kShare * kWave) {
        const int tiles_here = wide[u].hi - wide[u].lo;
        // in fp32: an estimate
        const float cut = fmaxf(1.0f, ceilf(static_cast<float>(tiles_here) * part));
        const int each =
            static_cast<int>(ceilf(static_cast<float>(tiles_here) * __builtin_amdgcn_rcpf(cut)));
        items += static_cast<int>(cut);
        high = max(high, each);
        low = min(low, each);
      }
#pragma unroll
      for (int d = kWave / 2; d > 0; d >>= 1) {
        items += __shfl_xor(items, d);
        high = max(high, __shfl_xor(high, d));
        low = min(low, __shfl_xor(low, d));
      }
      if (__lane_id() == 0) {
        atomicAdd(&count[mine_k], items);
        atomicMax(&longest_of[mine_k], high);
        atomicMin(&shortest_of[mine_k], low);
      }
    }
    __syncthreads();
    share = candidate(kOf[0]);
    float best = INFINITY;
#pragma unroll
    for (int k = 0; k < kCands; ++k) {
      constexpr float kEnds = 4.0f;
      const float blocks = static_cast<float>(a.wide_blocks);
      const float items = static_cast<float>(max(1, count[k]));
      const float rounds = items / blocks;
      const float open = ceilf(rounds) - rounds;  // of the last round
      const float est = fmaxf((static_cast<float>(total) + kEnds * items) / blocks +
                                  open * (static_cast<float>(shortest_of[k]) + kEnds),
                              static_cast<float>(longest_of[k]) + kEnds);
      if (est < best) {
        best = est;
        share = candidate(kOf[k]);
      }
    }
  }

  WideItem* items = reinterpret_cast<WideItem*>(a.work + a.at_items);
  WideJoin* joins = reinterpret_cast<WideJoin*>(a.work + a.at_joins);
  int done_items = 0, done_joins = 0, done_parts = 0;
  for (int base = 0; base < stored; base += kPlanThreads) {
    // The last units of a causal request are its longest: they go first.
    const int u = stored - 1 - (base + static_cast<int>(threadIdx.x));
    int r = 0, t0 = 0, n = 0, lo = 0, hi = 0;
    if (u >= 0) {
      const WideUnit w = wide[u];
      r = w.request;
      t0 = w.t0;
      n = min(a.wide_tokens, clamp_len(a.new_lens[r]) - t0);
      lo = w.lo;
      hi = w.hi;
    }
    int cut = u >= 0 ? max(1, (hi - lo + share - 1) / share) : 0;
    int v[3] = {cut, cut > 1 ? 1 : 0, cut > 1 ? cut : 0}, sum[3];
    block_scan<3, 0u>(v, sum, scratch);
    if (u >= 0) {
      const int ctx_row = a.cu_new[r];
      const int part = done_parts + v[2];
      const int each = (hi - lo + cut - 1) / cut;
      for (int i = 0; i < cut; ++i) {
        const int at = done_items + v[0] + i;
        if (static_cast<unsigned>(at) >= static_cast<unsigned>(a.cap_items)) break;
        WideItem it;
        it.request = r;
        it.row = ctx_row + t0;
        it.tokens = max(0, min(n, a.tokens - it.row));
        it.pos = clamp_len(a.ctx_lens[r]) + t0;
        it.tile_lo = min(hi, lo + i * each);
        it.tile_hi = min(hi, lo + (i + 1) * each);
        it.part = cut > 1 ? part + i : -1;
        it.pad = 0;
        items[at] = it;
      }
      if (cut > 1 && static_cast<unsigned>(done_joins + v[1]) < static_cast<unsigned>(a.cap_joins)) {
        WideJoin j;
        j.row = ctx_row + t0;
        j.tokens = max(0, min(n, a.tokens - j.row));
        j.part = part;
        j.parts = cut;
        joins[done_joins + v[1]] = j;
      }
    }
    done_items += sum[0];
    done_joins += sum[1];
    done_parts += sum[2];
  }
  if (threadIdx.x == 0) {
    head->items = min(done_items, a.cap_items);
    head->joins = min(done_joins, a.cap_joins);
  }
}

__global__ __launch_bounds__(kPlanThreads) void plan_kernel(PlanArgs a) {
  __shared__ __align__(16) int lds[kPlanInts];
  if (blockIdx.x == 0) plan_schedule(a, lds);
  else plan_slots(a, static_cast<int>(blockIdx.x - 1) * kPlanTokens, lds);
}

// ----------------------------------------------------------------- append

struct AppendArgs {
  const char* work;
  uint64_t at_append;
  int8_t* codes[2];
  float* scales[2];
  const void* x[2];
  int64_t token_stride[2], head_stride[2];
  int32_t kv_heads, head_dim, block_log2, rows;
  uint64_t blocks;
};

constexpr int kAppendThreads = 256;

__device__ inline float wave_max(float v) {
#pragma unroll
  for (int d = kWave / 2; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
  return v;
}

// The step of a (block, head) whose new values reach `top` in magnitude.
__device__ inline float step_of(float top, float before, bool odd) {
  const float scale = fmaxf(before, top * (1.0f / 127.0f));
  return odd || !(before <= 3.4028235e38f) ? NAN : scale;
}

// rint(v / step) in [-127, 127], the quotient rounded to fp32 first.  QUICK:
// the correctly rounded quotient from the correctly rounded reciprocal, by
// Markstein's theorem (q' = q + (v - q s) / s in two fused steps, exact where
// nothing under- or overflows); elsewhere the division itself.  A step of 0 or
// NaN gives 0.
constexpr float kQuickFrom = 0x1p-90f, kQuickTo = 0x1p100f;

template <bool QUICK>
__device__ inline int quantise(float v, float scale, float inv) {
  float q;
  if constexpr (QUICK) {
    const float q0 = v * inv;
    q = fmaf(fmaf(-q0, scale, v), inv, q0);
  } else {
    q = scale > 0.0f ? v / scale : 0.0f;
  }
  return static_cast<int>(fminf(fmaxf(rintf(q), -127.0f), 127.0f));
}

__device__ inline int follow(int code, float ratio) {
  return static_cast<int>(rintf(static_cast<float>(code) * ratio));
}

// Four codes of a word after a change of step.
__device__ inline uint32_t follow4(uint32_t w, float ratio) {
  uint32_t r = 0;
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    r |= (static_cast<uint32_t>(follow(code_at(w, b), ratio)) & 0xffu) << (8 * b);
  }
  return r;
}

// Bytes [lo, hi) of a word, as a mask (any lo and hi).
__device__ inline uint32_t bytes_in(int lo, int hi) {
  lo = max(lo, 0);
  hi = min(hi, 4);
  if (lo >= hi) return 0u;
  return (hi == 4 ? 0xffffffffu : (1u << (8 * hi)) - 1u) & ~((1u << (8 * lo)) - 1u);
}

// What one block of an append works on.
template <class T>
struct AppendWork {
  AppendItem it;
  const typename T::store* x;  // the item's first row, this head
  int64_t token_stride;
  int8_t* codes;
  float* scale;
};

template <class T>
__device__ inline bool append_work(const AppendArgs& a, AppendWork<T>* w) {
  const auto* head = reinterpret_cast<ConstHead>(reinterpret_cast<uintptr_t>(a.work));
  const int item = blockIdx.x, g = blockIdx.y, kv = blockIdx.z;
  const auto* list =
      reinterpret_cast<ConstAppend>(reinterpret_cast<uintptr_t>(a.work) + a.at_append);
  // the list has a place for every block of the grid
  w->it = {list[item].block, list[item].row, list[item].place, list[item].count};
  if (item >= head->appends) return false;
  if (w->it.count <= 0 || w->it.row < 0 || w->it.row > a.rows - w->it.count) return false;
  if (w->it.block < 0 || static_cast<uint64_t>(w->it.block) >= a.blocks) return false;
  w->token_stride = a.token_stride[kv];
  w->x = static_cast<const typename T::store*>(a.x[kv]) +
         static_cast<int64_t>(w->it.row) * a.token_stride[kv] +
         static_cast<int64_t>(g) * a.head_stride[kv];
  const size_t cell = static_cast<size_t>(w->it.block) * a.kv_heads + g;
  w->codes = a.codes[kv] + (cell * a.head_dim << a.block_log2);
  w->scale = a.scales[kv] + cell;
  return true;
}

// The new step from the threads' largest values.
__device__ inline float block_step(float top, bool odd, float before) {
  __shared__ float s_top[kAppendThreads / kWave];
  __shared__ int s_odd[kAppendThreads / kWave];
  top = wave_max(top);
  const bool wave_odd = __any(odd);
  if (__lane_id() == 0) {
    s_top[threadIdx.x / kWave] = top;
    s_odd[threadIdx.x / kWave] = wave_odd;
  }
  __syncthreads();
  top = fmaxf(fmaxf(s_top[0], s_top[1]), fmaxf(s_top[2], s_top[3]));
  return step_of(top, before, s_odd[0] | s_odd[1] | s_odd[2] | s_odd[3]);
}

// Value by value: any strides; also the faster way for a token or two (4.4
// against 7.4 us for 64 requests of one token).
template <class T>
__device__ inline void append_values(const AppendArgs& a, const AppendWork<T>& w) {
  const int kv = blockIdx.z, bs = 1 << a.block_log2, hd = a.head_dim;
  const int n = w.it.count * hd, place = w.it.place;
  const float before = place > 0 ? *w.scale : 0.0f;
  float top = 0.0f;
  bool odd = false;  // something not finite
  for (int i = threadIdx.x; i < n; i += kAppendThreads) {
    const float v = fabsf(T::get(w.x[static_cast<int64_t>(i / hd) * w.token_stride + i % hd]));
    odd |= !(v <= 3.4028235e38f);
    top = fmaxf(top, v);
  }
  const float scale = block_step(top, odd, before);
  // V is transposed in its block: element (place p, column d) at d * bs + p.
  const int step_p = kv ? 1 : hd, step_d = kv ? bs : 1;
  if (place > 0 && !(scale == before)) {  // the held codes follow
    const float ratio = scale > 0.0f ? before / scale : 0.0f;
    if (kv == 0) {
      uint32_t* held = reinterpret_cast<uint32_t*>(w.codes);
      for (int i = threadIdx.x; i < place * hd / 4; i += kAppendThreads) {
        held[i] = follow4(held[i], ratio);
      }
    } else {
      const int words = (place + 3) / 4;
      for (int i = threadIdx.x; i < words * hd; i += kAppendThreads) {
        const int p = i % words * 4;
        uint32_t* at = reinterpret_cast<uint32_t*>(w.codes + i / words * bs + p);
        const uint32_t held = bytes_in(0, place - p);
        *at = (follow4(*at, ratio) & held) | (*at & ~held);
      }
      __syncthreads();  // a word may hold new places too
    }
  }
  for (int i = threadIdx.x; i < n; i += kAppendThreads) {
    const int t = i / hd, d = i % hd;
    const float v = T::get(w.x[static_cast<int64_t>(t) * w.token_stride + d]);
    w.codes[(place + t) * step_p + d * step_d] = static_cast<int8_t>(quantise<false>(v, scale, 0.0f));
  }
  if (threadIdx.x == 0) *w.scale = scale;
}

// One block per (touched block, kv head, keys or values).  A thread takes 4
// neighbouring places x 8 columns (up to UNITS such), loads them once in
// 16-byte pieces and keeps them while the block's largest is found.  Keys go
// out as 8 bytes a place.  Values are transposed in their block: 4 places of
// a column are one word, gathered in LDS, and leave as 16 bytes; where a
// group of 16 places holds tokens that were there, its old codes are merged.
// A new value is read once and its code written once: 15235 fp16 tokens of 4
// heads x 256, keys and values, take 28 us (94 MB, 3.3 TB/s; 34.7 us with the
// divisions themselves, so the vector unit still has its part in it).
template <class T, int UNITS>
__device__ inline void append_block(const AppendArgs& a, const AppendWork<T>& work) {
  constexpr int kWords = 8 * sizeof(typename T::store) / 16;  // 16-byte pieces of 8 values
  const AppendItem it = work.it;
  const int kv = blockIdx.z, bs = 1 << a.block_log2, hd = a.head_dim;
  const typename T::store* x = work.x;
  int8_t* codes = work.codes;
  const int end = it.place + it.count;       // places [it.place, end) are new
  const int p0 = it.place & ~3;              // units begin at whole words
  const int vecs = hd / 8, units = ((end - p0 + 3) / 4) * vecs;

  u32x4 raw[UNITS][4][kWords];
  float top = 0.0f;
  bool odd = false;  // something not finite
#pragma unroll
  for (int k = 0; k < UNITS; ++k) {
    const int u = k * kAppendThreads + static_cast<int>(threadIdx.x);
    if (u < units) {
      const int p = p0 + u / vecs * 4, d = u % vecs * 8;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        if (p + t >= it.place && p + t < end) {
          const u32x4* from = reinterpret_cast<const u32x4*>(
              x + static_cast<int64_t>(p + t - it.place) * work.token_stride + d);
#pragma unroll
          for (int w = 0; w < kWords; ++w) raw[k][t][w] = from[w];
        } else {
#pragma unroll
          for (int w = 0; w < kWords; ++w) raw[k][t][w] = u32x4{0u, 0u, 0u, 0u};
        }
      }
    }
  }
  auto value = [&](int k, int t, int e) {
    if constexpr (T::code == kF32) {
      return __uint_as_float(raw[k][t][e / 4][e % 4]);
    } else {
      return T::get(static_cast<uint16_t>((raw[k][t][0][e / 2] >> (16 * (e & 1))) & 0xffffu));
    }
  };
#pragma unroll
  for (int k = 0; k < UNITS; ++k) {
    if (k * kAppendThreads + static_cast<int>(threadIdx.x) < units) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float v = fabsf(value(k, t, e));
          odd |= !(v <= 3.4028235e38f);
          top = fmaxf(top, v);
        }
      }
    }
  }
  __shared__ __align__(16) uint32_t s_v[UNITS * kAppendThreads * 8];  // [column][places / 4]
  const float before = it.place > 0 ? *work.scale : 0.0f;
  const float scale = block_step(top, odd, before);
  const bool moved = it.place > 0 && !(scale == before);
  const float ratio = scale > 0.0f ? before / scale : 0.0f;

  const int words = bs / 4;  // of a value column
  const float inv = 1.0f / scale;
  auto write_codes = [&](auto quick) {
    constexpr bool kQuick = decltype(quick)::value;
#pragma unroll
    for (int k = 0; k < UNITS; ++k) {
      const int u = k * kAppendThreads + static_cast<int>(threadIdx.x);
      if (u < units) {
        const int p = p0 + u / vecs * 4, d = u % vecs * 8;
        uint32_t q[4][2];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            q[t][w] = 0u;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              q[t][w] |= (static_cast<uint32_t>(quantise<kQuick>(value(k, t, 4 * w + e), scale, inv)) & 0xffu)
                         << (8 * e);
            }
          }
          if (kv == 0 && p + t >= it.place && p + t < end) {
            *reinterpret_cast<u32x2*>(codes + (p + t) * hd + d) = u32x2{q[t][0], q[t][1]};
          }
        }
        if (kv == 1) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            uint32_t w = 0u;
#pragma unroll
            for (int t = 0; t < 4; ++t) w |= (q[t][e / 4] >> (8 * (e % 4)) & 0xffu) << (8 * t);
            s_v[(d + e) * words + (p >> 2)] = w;
          }
        }
      }
    }
  };
  if (scale >= kQuickFrom && scale <= kQuickTo) write_codes(std::true_type{});
  else write_codes(std::false_type{});
  if (kv == 0) {
    if (moved) {  // the held codes follow
      uint32_t* held = reinterpret_cast<uint32_t*>(codes);
      for (int i = threadIdx.x; i < it.place * hd / 4; i += kAppendThreads) {
        held[i] = follow4(held[i], ratio);
      }
    }
  } else {
    __syncthreads();
    const int first_group = moved ? 0 : it.place >> 4, groups = (end + 15) >> 4;
    for (int i = threadIdx.x; i < (groups - first_group) * hd; i += kAppendThreads) {
      const int d = i % hd, grp = first_group + i / hd;
      u32x4* at = reinterpret_cast<u32x4*>(codes + d * bs + 16 * grp);
      u32x4 v;
      if (16 * grp >= it.place && 16 * grp + 16 <= end) {
        v = *reinterpret_cast<const u32x4*>(&s_v[d * words + 4 * grp]);
      } else if (!moved) {
        // what is there stays: only the new bytes are written
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int p = 16 * grp + 4 * w;
          const uint32_t fresh = s_v[d * words + 4 * grp + w];
          if (p >= it.place && p + 4 <= end) {
            reinterpret_cast<uint32_t*>(at)[w] = fresh;
          } else {
            for (int b = max(0, it.place - p); b < min(4, end - p); ++b) {
              reinterpret_cast<int8_t*>(at)[4 * w + b] = static_cast<int8_t>(code_at(fresh, b));
            }
          }
        }
        continue;
      } else {
        v = *at;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int p = 16 * grp + 4 * w;  // the word's first place
          const uint32_t fresh = bytes_in(it.place - p, end - p), held = bytes_in(0, it.place - p);
          uint32_t x2 = v[w];
          if (held) x2 = (follow4(x2, ratio) & held) | (x2 & ~held);
          if (fresh) x2 = (s_v[d * words + 4 * grp + w] & fresh) | (x2 & ~fresh);
          v[w] = x2;
        }
      }
      *at = v;
    }
  }
  if (threadIdx.x == 0) *work.scale = scale;
}

template <class T, int UNITS>
__global__ __launch_bounds__(kAppendThreads) void append_kernel(AppendArgs a) {
  AppendWork<T> work;
  if (!append_work(a, &work)) return;
  if (work.it.count <= 2) append_values(a, work);
  else append_block<T, UNITS>(a, work);
}

// Inputs whose rows are not 16-byte aligned.
template <class T>
__global__ __launch_bounds__(kAppendThreads) void append_any_kernel(AppendArgs a) {
  AppendWork<T> work;
  if (append_work(a, &work)) append_values(a, work);
}

// ----------------------------------------------------------- turned append

// A block's keys, turned to their positions in fp32 and quantised from there:
// a thread takes up to UNITS times eight pairs of a place (or sixteen channels
// that are not turned), and keeps the turned values while the block's largest
// is found.  Bound by vector instructions on long appends (14151 tokens of 4 heads x 256,
// 128 of them turned: 31 us, 26 without a turn), by a chain of loads on short ones (64
// tokens 6 us).
template <class T, int UNITS, bool ALIGNED>
__device__ inline void append_turned(const AppendArgs& a, const Rotary& r,
                                     const AppendWork<T>& work, int position) {
  const AppendItem it = work.it;
  const int hd = a.head_dim, units = hd / 16, turned = r.dim / 16, half = r.dim / 2;
  const float before = it.place > 0 ? *work.scale : 0.0f;
  float v[UNITS][2][8];
  auto channels = [&](int u, int* first, int* second) {
    if (u < turned) {
      unit_channels(r.layout, half, u, first, second);
    } else {
      *first = 16 * u;
      *second = 16 * u + 8;
    }
  };
#pragma unroll
  for (int k = 0; k < UNITS; ++k) {
    const int i = k * kAppendThreads + static_cast<int>(threadIdx.x);
    if (i < it.count * units) {
      const int t = i / units;
      int first, second;
      channels(i - t * units, &first, &second);
      const typename T::store* x = work.x + static_cast<int64_t>(t) * work.token_stride;
      get8<T, ALIGNED>(x + first, v[k][0]);
      get8<T, ALIGNED>(x + second, v[k][1]);
    }
  }
  float top = 0.0f;
  bool odd = false;  // something not finite
#pragma unroll
  for (int k = 0; k < UNITS; ++k) {
    const int i = k * kAppendThreads + static_cast<int>(threadIdx.x);
    if (i < it.count * units) {
      const int t = i / units, u = i - t * units;
      if (u < turned) {
        turn_unit(r.layout, v[k], [&](int e) { return angle(r, 8 * u + e, position + t); });
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float m = fabsf(v[k][e / 8][e % 8]);
        odd |= !(m <= 3.4028235e38f);
        top = fmaxf(top, m);
      }
    }
  }
  const float scale = block_step(top, odd, before);
  if (it.place > 0 && !(scale == before)) {  // the held codes follow
    const float ratio = scale > 0.0f ? before / scale : 0.0f;
    uint32_t* held = reinterpret_cast<uint32_t*>(work.codes);
    for (int i = threadIdx.x; i < it.place * hd / 4; i += kAppendThreads) {
      held[i] = follow4(held[i], ratio);
    }
  }
  const float inv = 1.0f / scale;
  auto write_codes = [&](auto quick) {
    constexpr bool kQuick = decltype(quick)::value;
#pragma unroll
    for (int k = 0; k < UNITS; ++k) {
      const int i = k * kAppendThreads + static_cast<int>(threadIdx.x);
      if (i < it.count * units) {
        const int t = i / units;
        int at[2];
        channels(i - t * units, &at[0], &at[1]);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          u32x2 q = {0u, 0u};
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            q[e / 4] |= (static_cast<uint32_t>(quantise<kQuick>(v[k][s][e], scale, inv)) & 0xffu)
                        << (8 * (e % 4));
          }
          *reinterpret_cast<u32x2*>(work.codes + (it.place + t) * hd + at[s]) = q;
        }
      }
    }
  };
  if (scale >= kQuickFrom && scale <= kQuickTo) write_codes(std::true_type{});
  else write_codes(std::false_type{});
  if (threadIdx.x == 0) *work.scale = scale;
}

// Any even number of turned channels: value by value, its angle made for both
// passes.
template <class T>
__device__ inline void append_turned_any(const AppendArgs& a, const Rotary& r,
                                         const AppendWork<T>& work, int position) {
  const AppendItem it = work.it;
  const int hd = a.head_dim, n = it.count * hd;
  const float before = it.place > 0 ? *work.scale : 0.0f;
  auto value = [&](int t, int d) {
    const typename T::store* x = work.x + static_cast<int64_t>(t) * work.token_stride;
    float v = T::get(x[d]);
    if (d >= r.dim) return v;
    int other;
    const int p = pair_of(r.layout, r.dim / 2, d, &other);
    float w = T::get(x[other]);
    const CosSin c = angle(r, p, position + t);
    if (d < other) turn(c, v, w);
    else turn(c, w, v);
    return v;
  };
  float top = 0.0f;
  bool odd = false;
  for (int i = threadIdx.x; i < n; i += kAppendThreads) {
    const float m = fabsf(value(i / hd, i % hd));
    odd |= !(m <= 3.4028235e38f);
    top = fmaxf(top, m);
  }
  const float scale = block_step(top, odd, before);
  if (it.place > 0 && !(scale == before)) {
    const float ratio = scale > 0.0f ? before / scale : 0.0f;
    uint32_t* held = reinterpret_cast<uint32_t*>(work.codes);
    for (int i = threadIdx.x; i < it.place * hd / 4; i += kAppendThreads) {
      held[i] = follow4(held[i], ratio);
    }
  }
  for (int i = threadIdx.x; i < n; i += kAppendThreads) {
    work.codes[it.place * hd + i] =
        static_cast<int8_t>(quantise<false>(value(i / hd, i % hd), scale, 0.0f));
  }
  if (threadIdx.x == 0) *work.scale = scale;
}

// UNITS of the values' blocks; a key thread's sixteen channels are half as many.
// 0: any dims and alignment.
template <class T, int UNITS>
__global__ __launch_bounds__(kAppendThreads) void append_turned_kernel(AppendArgs a, Rotary r,
                                                                       const int32_t* positions) {
  AppendWork<T> work;
  if (!append_work(a, &work)) return;
  if (blockIdx.z == 0) {
    const int position = positions[work.it.row];
    if constexpr (UNITS == 0) append_turned_any(a, r, work, position);
    else if (work.it.count * a.head_dim <= 16 * kAppendThreads) append_turned<T, 1, true>(a, r, work, position);
    else append_turned<T, 2 * UNITS, true>(a, r, work, position);
  } else if constexpr (UNITS == 0) {
    append_values(a, work);
  } else {
    if (work.it.count <= 2) append_values(a, work);
    else append_block<T, UNITS>(a, work);
  }
}

// ------------------------------------------------------------------- read

struct ReadArgs {
  const int8_t* codes[2];
  const float* scales[2];
  void* out[2];
  const int32_t* table;
  const int32_t* starts;
  const int32_t* cu;
  int32_t width, requests, kv_heads, head_dim, block_log2;
  uint64_t rows, blocks;
};

// A run of rows inside one group of 16 places: `rows` from output row `row`
// on, the first at place `place` (of the group) of `cell` (-1: no block).
struct ReadJob {
  int32_t row, rows, block, place;
};

constexpr int kReadRows = 64, kReadBatch = 8;

// Values of codes w, as many as fill 16 bytes of T.
template <class T>
__device__ inline void put(typename T::store* out, u32x2 w, float scale) {
  if constexpr (T::code == kF32) {
    f32x4 v;
#pragma unroll
    for (int b = 0; b < 4; ++b) v[b] = static_cast<float>(code_at(w[0], b)) * scale;
    __builtin_nontemporal_store(v, reinterpret_cast<f32x4*>(out));
  } else {
    u32x4 v;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const uint32_t word = w[b / 2];
      const uint32_t lo = T::put(static_cast<float>(code_at(word, 2 * (b & 1))) * scale);
      const uint32_t hi = T::put(static_cast<float>(code_at(word, 2 * (b & 1) + 1)) * scale);
      v[b] = lo | (hi << 16);
    }
    __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(out));
  }
}

template <class T>
__device__ inline u32x2 codes_for(const int8_t* p) {
  if constexpr (T::code == kF32) return u32x2{*reinterpret_cast<const uint32_t*>(p), 0u};
  else return *reinterpret_cast<const u32x2*>(p);
}

// One block per 64 output rows and kv head: the rows that begin a group of 16
// places become jobs (a request's rows follow each other, so there are 4 or
// 5 of them unless requests are tiny).  A thread writes 16 bytes, its wave 1 KiB.
// A value column's 16 places are one 16-byte load; they turn through LDS.
// Bound by bytes: 15521 rows of 4 heads x 256 to fp32, keys and values, take
// 34 us (159 MB, 4.7 TB/s; a large copy reaches 4.8).  Few rows are latency:
// 2078 rows of 8 heads x 128 take 11 us, a chain of four loads that miss.
template <class T>
__global__ __launch_bounds__(256) void read_kernel(ReadArgs a) {
  const int bs = 1 << a.block_log2, hd = a.head_dim, g = blockIdx.y;
  const uint64_t row0 = static_cast<uint64_t>(blockIdx.x) * kReadRows;
  __shared__ ReadJob s_job[kReadRows];
  __shared__ int s_jobs;
  __shared__ __align__(16) int8_t s_v[kReadBatch * 16 * 256];
  __shared__ float s_scale[2][kReadBatch];
  __shared__ int s_cu[kWave], s_start[kWave];
  if (threadIdx.x < kWave) {
    const int lane = threadIdx.x, row = static_cast<int>(row0) + lane;
    // The requests of the block's rows follow each other: 64 are looked at in
    // LDS, and all of them only where more end here.
    const int r0 = a.requests <= kWave ? 0 : find_unit(a.cu, a.requests, static_cast<int>(row0));
    s_cu[lane] = r0 + 1 + lane <= a.requests ? a.cu[r0 + 1 + lane] : 0x7fffffff;
    s_start[lane] = a.starts[min(r0 + lane, a.requests - 1)];
    const int cu0 = a.cu[r0];
    __builtin_amdgcn_wave_barrier();
    bool begins = false;
    ReadJob job{row, 0, -1, 0};
    if (static_cast<uint64_t>(row) < a.rows) {
      const int ended = s_cu[0] <= row ? 1 + upper(s_cu, kWave, row) : 0;
      int r = min(r0 + ended, a.requests - 1), from, to, start;
      if (r < r0 + kWave) {
        from = r > r0 ? s_cu[r - r0 - 1] : cu0;
        to = s_cu[r - r0];
        start = s_start[r - r0];
      } else {
        r = r0 + kWave + upper(a.cu + r0 + kWave, a.requests - r0 - kWave, row);
        from = a.cu[r];
        to = a.cu[r + 1];
        start = a.starts[r];
      }
      to = min(to, static_cast<int>(a.rows));
      const int pos = start + row - from, j = pos >> a.block_log2;
      begins = row == from || (pos & 15) == 0;
      job.place = pos & (bs - 1);
      job.rows = min(16 - (pos & 15), to - row);
      if (pos >= 0 && j < a.width) {
        const int block = a.table[static_cast<size_t>(r) * a.width + j];
        if (static_cast<uint64_t>(static_cast<int64_t>(block)) < a.blocks) job.block = block;
      }
    }
    const uint64_t all = __ballot(begins);
    if (begins) s_job[__popcll(all & ((1ull << lane) - 1ull))] = job;
    if (lane == 0) s_jobs = __popcll(all);
  }
  __syncthreads();
  constexpr int kPer = 16 / sizeof(typename T::store);  // values a thread writes
  const int jobs = s_jobs, chunks = hd / kPer;
  auto out_at = [&](int kv, int row, int d) {
    return static_cast<typename T::store*>(a.out[kv]) +
           (static_cast<size_t>(row) * a.kv_heads + g) * hd + d;
  };
  for (int first = 0; first < jobs; first += kReadBatch) {
    const int n = min(kReadBatch, jobs - first);
    // Four pieces at a time, so that their loads do not wait for each other.
    const int keys = a.out[0] ? n * 16 * chunks : 0, columns = a.out[1] ? n * hd : 0;
    u32x2 kw[4];
    auto load_keys = [&](int i0) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + u * 256;
        const int d = i % chunks * kPer, b = i / chunks % 16, k = i / chunks / 16;
        kw[u] = u32x2{0u, 0u};
        if (i < keys && b < s_job[first + k].rows && s_job[first + k].block >= 0) {
          const ReadJob& job = s_job[first + k];
          const size_t cell = static_cast<size_t>(job.block) * a.kv_heads + g;
          kw[u] = codes_for<T>(a.codes[0] + (cell * bs + job.place + b) * hd + d);
        }
      }
    };
    float scale = 0.0f;
    if (threadIdx.x < 2 * kReadBatch) {
      const int k = threadIdx.x % kReadBatch;
      if (k < n && s_job[first + k].block >= 0) {
        scale = a.scales[threadIdx.x / kReadBatch]
                        [static_cast<size_t>(s_job[first + k].block) * a.kv_heads + g];
      }
    }
    load_keys(threadIdx.x);
    for (int i0 = threadIdx.x; i0 < columns; i0 += 4 * 256) {
      u32x4 w[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + u * 256, d = i % hd, k = i / hd;
        w[u] = u32x4{0u, 0u, 0u, 0u};
        if (i < columns && s_job[first + k].block >= 0) {
          const ReadJob& job = s_job[first + k];
          const size_t cell = static_cast<size_t>(job.block) * a.kv_heads + g;
          w[u] = *reinterpret_cast<const u32x4*>(a.codes[1] + cell * bs * hd +
                                                 static_cast<size_t>(d) * bs + (job.place & ~15));
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + u * 256, d = i % hd, k = i / hd;
        if (i < columns) {
#pragma unroll
          for (int b = 0; b < 16; ++b) {
            s_v[(k * 16 + b) * hd + d] = static_cast<int8_t>(code_at(w[u][b / 4], b % 4));
          }
        }
      }
    }
    if (threadIdx.x < 2 * kReadBatch) {
      s_scale[threadIdx.x / kReadBatch][threadIdx.x % kReadBatch] = scale;
    }
    __syncthreads();
    for (int i0 = threadIdx.x; i0 < keys; i0 += 4 * 256) {
      if (i0 >= 4 * 256) load_keys(i0);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + u * 256;
        const int d = i % chunks * kPer, b = i / chunks % 16, k = i / chunks / 16;
        if (i < keys && b < s_job[first + k].rows) {
          put<T>(out_at(0, s_job[first + k].row + b, d), kw[u], s_scale[0][k]);
        }
      }
    }
    const int values = a.out[1] ? n * 16 * chunks : 0;
    for (int i = threadIdx.x; i < values; i += 256) {
      const int d = i % chunks * kPer, b = i / chunks % 16, k = i / chunks / 16;
      const ReadJob& job = s_job[first + k];
      if (b >= job.rows) continue;
      put<T>(out_at(1, job.row + b, d),
             codes_for<T>(&s_v[(k * 16 + (job.place & 15) + b) * hd + d]), s_scale[1][k]);
    }
    __syncthreads();
  }
}

template <class T>
static void launch_append(const AppendArgs& a, unsigned items, bool aligned, hipStream_t s) {
  const dim3 grid(items, static_cast<unsigned>(a.kv_heads), 2);
  const int values = a.head_dim << a.block_log2;  // of a block
  if (!aligned) append_any_kernel<T><<<grid, kAppendThreads, 0, s>>>(a);
  else if (values <= 32 * kAppendThreads) append_kernel<T, 1><<<grid, kAppendThreads, 0, s>>>(a);
  else if (values <= 64 * kAppendThreads) append_kernel<T, 2><<<grid, kAppendThreads, 0, s>>>(a);
  else append_kernel<T, 4><<<grid, kAppendThreads, 0, s>>>(a);
}

template <class T>
static void launch_append_turned(const AppendArgs& a, const Rotary& r, const int32_t* positions,
                                 unsigned items, bool aligned, hipStream_t s) {
  const dim3 grid(items, static_cast<unsigned>(a.kv_heads), 2);
  const int values = a.head_dim << a.block_log2;
  if (!aligned || !whole_units(r)) {
    append_turned_kernel<T, 0><<<grid, kAppendThreads, 0, s>>>(a, r, positions);
  } else if (values <= 32 * kAppendThreads) {
    append_turned_kernel<T, 1><<<grid, kAppendThreads, 0, s>>>(a, r, positions);
  } else if (values <= 64 * kAppendThreads) {
    append_turned_kernel<T, 2><<<grid, kAppendThreads, 0, s>>>(a, r, positions);
  } else {
    append_turned_kernel<T, 4><<<grid, kAppendThreads, 0, s>>>(a, r, positions);
  }
}

static int log2_of(int n) { return n == 16 ? 4 : n == 32 ? 5 : n == 64 ? 6 : 7; }

}  // namespace kv
}  // namespace grm

using namespace grm::kv;

extern "C" int grm_hip_kv_work_bytes(const grm_kv_batch_desc* batch, uint64_t* out_bytes) {
  if (!out_bytes) return grm::fail(-1, "null output pointer");
  GRM_CHECK_RC(check_batch(batch, false));
  Layout l;
  GRM_CHECK_RC(layout_of(batch, &l));
  *out_bytes = l.bytes;
  grm::clear_error();
  return 0;
}

extern "C" int grm_hip_kv_plan(const grm_kv_batch_desc* b, void* stream) {
  GRM_CHECK_RC(check_batch(b, true));
  Layout l;
  GRM_CHECK_RC(layout_of(b, &l));
  if (b->requests && b->work_bytes < l.bytes) return grm::fail(-1, "work is smaller than grm_hip_kv_work_bytes");
  PlanArgs a{};
  a.ctx_lens = b->ctx_lens;
  a.new_lens = b->new_lens;
  a.table = b->block_table;
  a.free_list = b->free_list;
  a.free_head = b->free_head;
  a.free_head_out = b->free_head_out;
  a.cu_new = b->cu_new;
  a.slots = b->slot_map;
  a.positions = b->positions;
  a.work = static_cast<char*>(b->work);
  a.requests = b->requests;
  a.width = b->table_width;
  a.tokens = b->tokens;
  a.window = b->window;
  a.reach = l.reach;
  a.free_count = static_cast<int32_t>(b->free_count);
  a.group = l.group;
  a.wide_tokens = l.wide_tokens;
  a.kv_heads = b->kv_heads;
  a.wide_blocks = l.wide_blocks;
  a.block_log2 = log2_of(b->block_tokens);
  a.cap_append = static_cast<int32_t>(l.cap_append);
  a.cap_units = static_cast<int32_t>(l.cap_units);
  a.cap_wide = static_cast<int32_t>(l.cap_wide);
  a.cap_items = static_cast<int32_t>(l.cap_items);
  a.cap_joins = static_cast<int32_t>(l.cap_joins);
  a.cap_parts = static_cast<int32_t>(l.cap_parts);
  a.at_append = l.at_append;
  a.at_units = l.at_units;
  a.at_tiles = l.at_tiles;
  for (int k = 0; k < 2; ++k) {
    a.runs[k] = l.runs[k];
    a.at_run_units[k] = l.at_run_units[k];
  }
  a.at_scan = l.at_scan;
  a.at_wide = l.at_wide;
  a.at_items = l.at_items;
  a.at_joins = l.at_joins;
  const unsigned blocks = 1u + static_cast<unsigned>((b->tokens + kPlanTokens - 1) / kPlanTokens);
  plan_kernel<<<blocks, kPlanThreads, 0, static_cast<hipStream_t>(stream)>>>(a);
  GRM_HIP_CHECK(hipGetLastError());
  grm::clear_error();
  return 0;
}

// Appends, with keys turned where there is a rotary.
static int append_call(const grm_kv_cache_desc* c, const grm_kv_batch_desc* b, bool turned,
                       const grm_rotary_desc* rotary, const void* k, const void* v, int dtype,
                       int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride,
                       int64_t v_head_stride, void* stream) {
  GRM_CHECK_RC(check_pair(c, b, true));
  Rotary r;
  if (turned) GRM_CHECK_RC(rotary_of(rotary, c->head_dim, &r));
  if (dtype != grm::kF32 && dtype != grm::kBF16 && dtype != grm::kF16) {
    return grm::fail(-1, "keys and values are F32, BF16 or F16");
  }
  if (b->requests == 0 || b->tokens == 0) {
    grm::clear_error();
    return 0;
  }
  if (!k || !v) return grm::fail(-1, "null keys or values");
  if (turned && !b->positions) return grm::fail(-1, "turned keys need the batch's positions");
  Layout l;
  GRM_CHECK_RC(layout_of(b, &l));
  if (b->work_bytes < l.bytes) return grm::fail(-1, "work is smaller than grm_hip_kv_work_bytes");
  AppendArgs a{};
  a.work = static_cast<const char*>(b->work);
  a.at_append = l.at_append;
  a.codes[0] = static_cast<int8_t*>(c->k_codes);
  a.codes[1] = static_cast<int8_t*>(c->v_codes);
  a.scales[0] = c->k_scales;
  a.scales[1] = c->v_scales;
  a.x[0] = k;
  a.x[1] = v;
  a.token_stride[0] = k_token_stride;
  a.token_stride[1] = v_token_stride;
  a.head_stride[0] = k_head_stride;
  a.head_stride[1] = v_head_stride;
  a.kv_heads = c->kv_heads;
  a.head_dim = c->head_dim;
  a.block_log2 = log2_of(c->block_tokens);
  a.rows = b->tokens;
  a.blocks = c->blocks;
  const int64_t unit = dtype == grm::kF32 ? 4 : 8;
  const bool aligned = aligned16(k) && aligned16(v) && k_token_stride % unit == 0 &&
                       k_head_stride % unit == 0 && v_token_stride % unit == 0 &&
                       v_head_stride % unit == 0;
  const auto items = static_cast<unsigned>(l.cap_append);
  const auto s = static_cast<hipStream_t>(stream);
  if (turned) {
    if (dtype == grm::kF32) launch_append_turned<F32>(a, r, b->positions, items, aligned, s);
    else if (dtype == grm::kBF16) launch_append_turned<BF16>(a, r, b->positions, items, aligned, s);
    else launch_append_turned<F16>(a, r, b->positions, items, aligned, s);
  } else if (dtype == grm::kF32) {
    launch_append<F32>(a, items, aligned, s);
  } else if (dtype == grm::kBF16) {
    launch_append<BF16>(a, items, aligned, s);
  } else {
    launch_append<F16>(a, items, aligned, s);
  }
  GRM_HIP_CHECK(hipGetLastError());
  grm::clear_error();
  return 0;
}

extern "C" int grm_hip_kv_append(const grm_kv_cache_desc* c, const grm_kv_batch_desc* b,
                                 const void* k, const void* v, int dtype, int64_t k_token_stride,
                                 int64_t k_head_stride, int64_t v_token_stride,
                                 int64_t v_head_stride, void* stream) {
  return append_call(c, b, false, nullptr, k, v, dtype, k_token_stride, k_head_stride,
                     v_token_stride, v_head_stride, stream);
}

extern "C" int grm_hip_kv_append_turned(const grm_kv_cache_desc* c, const grm_kv_batch_desc* b,
                                        const grm_rotary_desc* rotary, const void* k,
                                        const void* v, int dtype, int64_t k_token_stride,
                                        int64_t k_head_stride, int64_t v_token_stride,
                                        int64_t v_head_stride, void* stream) {
  return append_call(c, b, true, rotary, k, v, dtype, k_token_stride, k_head_stride,
                     v_token_stride, v_head_stride, stream);
}

extern "C" int grm_hip_kv_read(const grm_kv_cache_desc* c, const int32_t* block_table,
                               int table_width, int requests, const int32_t* starts,
                               const int32_t* cu_rows, uint64_t rows, int dtype, void* k_out,
                               void* v_out, void* stream) {
  GRM_CHECK_RC(check_cache(c));
  if (dtype != grm::kF32 && dtype != grm::kBF16 && dtype != grm::kF16) {
    return grm::fail(-1, "values are read as F32, BF16 or F16");
  }
  if (requests < 0 || table_width < 0) return grm::fail(-1, "negative size");
  if (rows > static_cast<uint64_t>(kMaxLen)) return grm::fail(-1, "too many rows");
  if (rows == 0 || (!k_out && !v_out)) {
    grm::clear_error();
    return 0;
  }
  if (requests == 0) return grm::fail(-1, "rows of no request");
  if (!starts || !cu_rows || (table_width > 0 && !block_table)) return grm::fail(-1, "null array");
  if (!aligned16(k_out) || !aligned16(v_out)) {
    return grm::fail(-1, "outputs must be 16-byte aligned");
  }
  ReadArgs a{};
  a.codes[0] = static_cast<const int8_t*>(c->k_codes);
  a.codes[1] = static_cast<const int8_t*>(c->v_codes);
  a.scales[0] = c->k_scales;
  a.scales[1] = c->v_scales;
  a.out[0] = k_out;
  a.out[1] = v_out;
  a.table = block_table;
  a.starts = starts;
  a.cu = cu_rows;
  a.width = table_width;
  a.requests = requests;
  a.kv_heads = c->kv_heads;
  a.head_dim = c->head_dim;
  a.block_log2 = log2_of(c->block_tokens);
  a.rows = rows;
  a.blocks = c->blocks;
  const dim3 grid(static_cast<unsigned>((rows + kReadRows - 1) / kReadRows),
                  static_cast<unsigned>(c->kv_heads));
  const auto s = static_cast<hipStream_t>(stream);
  if (dtype == grm::kF32) read_kernel<F32><<<grid, 256, 0, s>>>(a);
  else if (dtype == grm::kBF16) read_kernel<BF16><<<grid, 256, 0, s>>>(a);
  else read_kernel<F16><<<grid, 256, 0, s>>>(a);
  GRM_HIP_CHECK(hipGetLastError());
  grm::clear_error();
  return 0;
}
