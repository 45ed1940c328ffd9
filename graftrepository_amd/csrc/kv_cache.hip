// kv_cache.hip -- the 8-bit key/value cache: a step's plan (block tables,
// slot map, schedule), the quantising append, and the dense read back.
//
// The cache's law is the header's (include/grm_hip_router.h).  The plan is
// latency, the append and the read are bytes: append reads the new values
// once, and writes a byte for each; read loads a byte per value and writes
// two or four.

#include "kv_common.hpp"

#include <mutex>

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

int check_pair(const grm_kv_cache_desc* c, const grm_kv_batch_desc* b) {
  GRM_CHECK_RC(check_cache(c));
  GRM_CHECK_RC(check_batch(b, true));
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
    const uint64_t units = rows / l.wide_tokens + busy;
    // Only units longer than the share C = all / (4 x blocks) are cut, into
    // at most 2 x length / C parts.
    l.cap_parts = 8 * static_cast<uint64_t>(l.wide_blocks) + 8;
    l.cap_joins = l.cap_parts / 2;
    l.cap_items = units + l.cap_parts;
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
    l.at_runs[k] = place(l.cap_units ? l.runs[k] * sizeof(NarrowRun) : 0);
  }
  l.at_scan = place(l.wide_tokens ? (reqs + 1) * 4 : 0);
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
  int32_t requests, width, tokens, window;
  int32_t free_count, group, wide_tokens, kv_heads;
  int32_t wide_blocks, block_log2;
  int32_t cap_append, cap_units, cap_items, cap_joins, cap_parts;
  int32_t runs[2];
  uint64_t at_append, at_units, at_tiles, at_runs[2], at_scan, at_items, at_joins;
};

// Exclusive sums over the block of N values per thread; totals to `sum`.
// `scratch` holds N * 16 ints.  Two barriers.
template <int N>
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
      if (lane >= d) v[k] += o;
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
      before += w < wave ? t : 0;
      all += t;
    }
    v[k] = v[k] - own[k] + before;
    sum[k] = all;
  }
  __syncthreads();
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
// request see.
__device__ inline void tiles_of(const PlanArgs& a, int tile, int ctx, int t0, int n, int* lo,
                                int* hi) {
  const int last = ctx + t0 + n;  // keys before this are seen by the last token
  const int first = a.window > 0 ? max(0, ctx + t0 + 1 - a.window) : 0;
  *lo = first / tile;
  *hi = (last + tile - 1) / tile;
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
      v[0] += l[j].fresh;
      v[1] += l[j].need;
      v[2] += l[j].touched;
    }
    block_scan(v, sum, scratch);
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
      const int i = threadIdx.x * kPerThread + j;
      s_cu[i] = done_new + v[0];
      s_ctx[i] = l[j].ctx;
      s_need[i] = done_need + v[1];
      s_touch[i] = done_touch + v[2];
      v[0] += l[j].fresh;
      v[1] += l[j].need;
      v[2] += l[j].touched;
    }
    __syncthreads();
    const int here = min(kPlanChunk, a.requests - base);
    const int end = min(t1, done_new + sum[0]);
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
      if (place == 0 || t == 0) {
        const int at = s_touch[k] + j - (ctx >> a.block_log2);
        const int next = k + 1 < here ? s_cu[k + 1] : done_new + sum[0];
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
    done_new += sum[0];
    done_need += sum[1];
    done_touch += sum[2];
    __syncthreads();
  }
  for (int i = max(t0, filled) + static_cast<int>(threadIdx.x); i < t1; i += kPlanThreads) {
    if (a.slots) a.slots[i] = -1;
    if (a.positions) a.positions[i] = -1;
  }
}

constexpr int kScanInts = 5 * 16 + 16;

__device__ void plan_schedule(const PlanArgs& a, int* lds) {
  int* scratch = lds;  // [5 * 16] and, after it, the candidates' counts: kScanInts
  SchedHead* head = reinterpret_cast<SchedHead*>(a.work);
  NarrowUnit* units = reinterpret_cast<NarrowUnit*>(a.work + a.at_units);
  int* tiles = reinterpret_cast<int*>(a.work + a.at_tiles);
  int* wide_at = reinterpret_cast<int*>(a.work + a.at_scan);
  int done[5] = {0, 0, 0, 0, 0};  // new, need, touched, narrow tiles, wide units
  int done_units = 0;
  for (int base = 0; base < a.requests; base += kPlanThreads) {
    const int r = base + static_cast<int>(threadIdx.x);
    const Lens l = lens_of(a, r);
    const bool narrow =
        l.fresh > 0 && static_cast<int64_t>(l.fresh) * a.group <= kNarrowCols && a.cap_units > 0;
    int lo = 0, hi = 0;
    if (narrow) tiles_of(a, narrow_tile(1 << a.block_log2), l.ctx, 0, l.fresh, &lo, &hi);
    const int wide = a.wide_tokens && l.fresh > 0 && !narrow
                         ? (l.fresh + a.wide_tokens - 1) / a.wide_tokens : 0;
    int v[5] = {l.fresh, l.need, l.touched, hi - lo, wide}, sum[5];
    block_scan(v, sum, scratch);
    int u[1] = {narrow ? 1 : 0}, usum[1];
    block_scan(u, usum, scratch);
    if (r < a.requests) {
      a.cu_new[r] = done[0] + v[0];
      if (a.wide_tokens) wide_at[r] = done[4] + v[4];
      const int at = done_units + u[0];
      if (narrow && static_cast<unsigned>(at) < static_cast<unsigned>(a.cap_units)) {
        NarrowUnit n;
        n.request = r;
        n.row = done[0] + v[0];
        n.tokens = max(0, min(l.fresh, a.tokens - n.row));
        n.tile_lo = lo;
        n.ctx = l.ctx;
        units[at] = n;
        tiles[at] = done[3] + v[3];
      }
    }
#pragma unroll
    for (int k = 0; k < 5; ++k) done[k] += sum[k];
    done_units += usum[0];
  }
  done_units = min(done_units, a.cap_units);
  const int wide_units = done[4];
  if (threadIdx.x == 0) {
    a.cu_new[a.requests] = done[0];
    tiles[done_units] = done[3];
    if (a.wide_tokens) wide_at[a.requests] = wide_units;
    if (a.free_head) {
      const int at = max(0, *a.free_head);
      const int left = max(0, a.free_count - at);
      *a.free_head_out = at + min(left, done[1]);
    }
    head->appends = min(done[2], a.cap_append);
    head->units = done_units;
    head->narrow_tiles = done[3];
    head->items = 0;
    head->joins = 0;
  }
  __syncthreads();  // the lists are read back by other threads of this block

  // Where the narrow kernel's wavefronts begin; without units every run is
  // empty.
  if (a.cap_units > 0) {
    int* cached = lds + kScanInts;
    const bool fits = done_units < kPlanChunk;
    if (fits) {
      for (int u = threadIdx.x; u <= done_units; u += kPlanThreads) cached[u] = tiles[u];
      __syncthreads();
    }
    const int* from = fits ? cached : tiles;
    for (int k = 0; k < 2; ++k) {
      NarrowRun* runs = reinterpret_cast<NarrowRun*>(a.work + a.at_runs[k]);
      for (int r = threadIdx.x; r < a.runs[k]; r += kPlanThreads) {
        NarrowRun n;
        n.begin = run_begin(done[3], a.runs[k], r);
        n.stop = run_begin(done[3], a.runs[k], r + 1);
        n.block_begin = run_begin(done[3], a.runs[k], r / 4 * 4);
        n.block_stop = run_begin(done[3], a.runs[k], r / 4 * 4 + 4);
        NarrowUnit u{};
        n.at = n.first = n.end = 0;
        if (n.begin < n.stop) {
          n.at = upper(from, done_units, n.begin);
          n.first = from[n.at];
          n.end = from[n.at + 1];
          u = units[n.at];
        }
        n.request = u.request;
        n.row = u.row;
        n.tokens = u.tokens;
        n.tile_lo = u.tile_lo;
        n.ctx = u.ctx;
#pragma unroll
        for (int e = 0; e < 4; ++e) n.pad[e] = 0;
        runs[r] = n;
      }
    }
  }
  if (wide_units == 0) return;
  __syncthreads();

  // Longest share C of a wide item.  More blocks than units: units are cut.
  // Candidates are the even share over k = 1..4; the estimate of each is
  // (rounds of blocks) x (mean item + 2 tiles for its prologue), no less
  // than its longest item.
  constexpr int kCands = 4;
  int* count = lds + 5 * 16;  // [kCands], then total and longest
  int* total_at = count + kCands;
  if (threadIdx.x < kCands + 2) count[threadIdx.x] = 0;
  __syncthreads();
  auto unit_tiles = [&](int u, int* r, int* t0, int* n, int* lo, int* hi) {
    *r = upper(wide_at, a.requests, u);
    *t0 = (u - wide_at[*r]) * a.wide_tokens;
    const int ctx = clamp_len(a.ctx_lens[*r]);
    *n = min(a.wide_tokens, clamp_len(a.new_lens[*r]) - *t0);
    tiles_of(a, kTile, ctx, *t0, *n, lo, hi);
  };
  int mine = 0, longest = 0;
  for (int u = threadIdx.x; u < wide_units; u += kPlanThreads) {
    int r, t0, n, lo, hi;
    unit_tiles(u, &r, &t0, &n, &lo, &hi);
    mine += hi - lo;
    longest = max(longest, hi - lo);
  }
  atomicAdd(&total_at[0], mine);
  atomicMax(&total_at[1], longest);
  __syncthreads();
  const int total = total_at[0];
  longest = total_at[1];
  const int even = max(1, (total + a.wide_blocks - 1) / a.wide_blocks);
  int cand[kCands], items_of[kCands];
#pragma unroll
  for (int k = 0; k < kCands; ++k) {
    cand[k] = max(8, (even + k) / (k + 1));
    items_of[k] = 0;
  }
  for (int u = threadIdx.x; u < wide_units; u += kPlanThreads) {
    int r, t0, n, lo, hi;
    unit_tiles(u, &r, &t0, &n, &lo, &hi);
#pragma unroll
    for (int k = 0; k < kCands; ++k) items_of[k] += (hi - lo + cand[k] - 1) / cand[k];
  }
#pragma unroll
  for (int k = 0; k < kCands; ++k) atomicAdd(&count[k], items_of[k]);
  __syncthreads();
  int share = cand[0];
  float best = INFINITY;
#pragma unroll
  for (int k = 0; k < kCands; ++k) {
    const int items = max(1, count[k]);
    const float rounds = static_cast<float>((items + a.wide_blocks - 1) / a.wide_blocks);
    const float mean = static_cast<float>(total) / static_cast<float>(items) + 2.0f;
    const float est = fmaxf(rounds * mean, static_cast<float>(min(longest, cand[k])) + 2.0f);
    if (est < best) {
      best = est;
      share = cand[k];
    }
  }

  WideItem* items = reinterpret_cast<WideItem*>(a.work + a.at_items);
  WideJoin* joins = reinterpret_cast<WideJoin*>(a.work + a.at_joins);
  int done_items = 0, done_joins = 0, done_parts = 0;
  for (int base = 0; base < wide_units; base += kPlanThreads) {
    // The last units of a causal request are its longest: they go first.
    const int u = wide_units - 1 - (base + static_cast<int>(threadIdx.x));
    int r = 0, t0 = 0, n = 0, lo = 0, hi = 0;
    if (u >= 0) unit_tiles(u, &r, &t0, &n, &lo, &hi);
    int cut = u >= 0 ? max(1, (hi - lo + share - 1) / share) : 0;
    int v[3] = {cut, cut > 1 ? 1 : 0, cut > 1 ? cut : 0}, sum[3];
    block_scan(v, sum, scratch);
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
  __shared__ int lds[4 * kPlanChunk + 1 + 3 * 16];
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

// One block per (touched block, kv head, keys or values).
template <class T>
__global__ __launch_bounds__(kAppendThreads) void append_kernel(AppendArgs a) {
  const SchedHead* head = reinterpret_cast<const SchedHead*>(a.work);
  const int item = blockIdx.x, g = blockIdx.y, kv = blockIdx.z;
  if (item >= head->appends) return;
  const AppendItem it = reinterpret_cast<const AppendItem*>(a.work + a.at_append)[item];
  if (it.block < 0 || static_cast<uint64_t>(it.block) >= a.blocks) return;
  const int bs = 1 << a.block_log2, hd = a.head_dim;
  const typename T::store* x = static_cast<const typename T::store*>(a.x[kv]) +
                               static_cast<int64_t>(it.row) * a.token_stride[kv] +
                               static_cast<int64_t>(g) * a.head_stride[kv];
  const size_t cell = static_cast<size_t>(it.block) * a.kv_heads + g;
  int8_t* codes = a.codes[kv] + cell * bs * hd;
  float* scale_at = a.scales[kv] + cell;
  const int n = it.count * hd;

  float top = 0.0f;
  bool odd = false;  // something not finite
  for (int i = threadIdx.x; i < n; i += kAppendThreads) {
    const float v = fabsf(T::get(x[static_cast<int64_t>(i / hd) * a.token_stride[kv] + i % hd]));
    odd |= !(v <= 3.4028235e38f);
    top = fmaxf(top, v);
  }
  __shared__ float s_top[kAppendThreads / kWave];
  __shared__ int s_odd;
  if (threadIdx.x == 0) s_odd = 0;
  __syncthreads();
  top = wave_max(top);
  if (__lane_id() == 0) s_top[threadIdx.x / kWave] = top;
  if (odd) s_odd = 1;
  const float before = it.place > 0 ? *scale_at : 0.0f;
  __syncthreads();
  top = fmaxf(fmaxf(s_top[0], s_top[1]), fmaxf(s_top[2], s_top[3]));
  float scale = fmaxf(before, top * (1.0f / 127.0f));
  if (s_odd || !(before <= 3.4028235e38f)) scale = NAN;

  // V is transposed in its block: element (place p, column d) at d * bs + p.
  const int step_p = kv ? 1 : hd, step_d = kv ? bs : 1;
  if (it.place > 0 && !(scale == before)) {
    const float ratio = scale > 0.0f ? before / scale : 0.0f;
    for (int i = threadIdx.x; i < it.place * hd; i += kAppendThreads) {
      const int p = kv ? i % it.place : i / hd, d = kv ? i / it.place : i % hd;
      int8_t* c = codes + p * step_p + d * step_d;
      *c = static_cast<int8_t>(rintf(static_cast<float>(*c) * ratio));
    }
  }
  for (int i = threadIdx.x; i < n; i += kAppendThreads) {
    const int t = i / hd, d = i % hd;
    const float v = T::get(x[static_cast<int64_t>(t) * a.token_stride[kv] + d]);
    const float q = scale > 0.0f ? fminf(fmaxf(rintf(v / scale), -127.0f), 127.0f) : 0.0f;
    codes[(it.place + t) * step_p + d * step_d] = static_cast<int8_t>(q);
  }
  if (threadIdx.x == 0) *scale_at = scale;
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

template <class T>
__global__ __launch_bounds__(256) void read_kernel(ReadArgs a) {
  const uint64_t row = blockIdx.x;
  const int kv = blockIdx.y;
  if (!a.out[kv]) return;
  const int bs = 1 << a.block_log2, hd = a.head_dim;
  const int r = upper(a.cu, a.requests, static_cast<int>(row));
  const int pos = a.starts[r] + static_cast<int>(row) - a.cu[r];
  const int j = pos >> a.block_log2, p = pos & (bs - 1);
  const int block = pos >= 0 && j < a.width ? a.table[static_cast<size_t>(r) * a.width + j] : -1;
  const bool there = block >= 0 && static_cast<uint64_t>(block) < a.blocks;
  typename T::store* out = static_cast<typename T::store*>(a.out[kv]) + row * a.kv_heads * hd;
  for (int i = threadIdx.x; i < a.kv_heads * hd; i += 256) {
    const int g = i / hd, d = i % hd;
    float v = 0.0f;
    if (there) {
      const size_t cell = static_cast<size_t>(block) * a.kv_heads + g;
      v = static_cast<float>(a.codes[kv][cell * bs * hd + (kv ? d * bs + p : p * hd + d)]) *
          a.scales[kv][cell];
    }
    out[i] = T::put(v);
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
  if (b->requests == 0) {
    grm::clear_error();
    return 0;
  }
  Layout l;
  GRM_CHECK_RC(layout_of(b, &l));
  if (b->work_bytes < l.bytes) return grm::fail(-1, "work is smaller than grm_hip_kv_work_bytes");
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
  a.free_count = static_cast<int32_t>(b->free_count);
  a.group = l.group;
  a.wide_tokens = l.wide_tokens;
  a.kv_heads = b->kv_heads;
  a.wide_blocks = l.wide_blocks;
  a.block_log2 = log2_of(b->block_tokens);
  a.cap_append = static_cast<int32_t>(l.cap_append);
  a.cap_units = static_cast<int32_t>(l.cap_units);
  a.cap_items = static_cast<int32_t>(l.cap_items);
  a.cap_joins = static_cast<int32_t>(l.cap_joins);
  a.cap_parts = static_cast<int32_t>(l.cap_parts);
  a.at_append = l.at_append;
  a.at_units = l.at_units;
  a.at_tiles = l.at_tiles;
  for (int k = 0; k < 2; ++k) {
    a.runs[k] = l.runs[k];
    a.at_runs[k] = l.at_runs[k];
  }
  a.at_scan = l.at_scan;
  a.at_items = l.at_items;
  a.at_joins = l.at_joins;
  const unsigned blocks = 1u + static_cast<unsigned>((b->tokens + kPlanTokens - 1) / kPlanTokens);
  plan_kernel<<<blocks, kPlanThreads, 0, static_cast<hipStream_t>(stream)>>>(a);
  GRM_HIP_CHECK(hipGetLastError());
  grm::clear_error();
  return 0;
}

extern "C" int grm_hip_kv_append(const grm_kv_cache_desc* c, const grm_kv_batch_desc* b,
                                 const void* k, const void* v, int dtype, int64_t k_token_stride,
                                 int64_t k_head_stride, int64_t v_token_stride,
                                 int64_t v_head_stride, void* stream) {
  GRM_CHECK_RC(check_pair(c, b));
  if (dtype != grm::kF32 && dtype != grm::kBF16 && dtype != grm::kF16) {
    return grm::fail(-1, "keys and values are F32, BF16 or F16");
  }
  if (b->requests == 0 || b->tokens == 0) {
    grm::clear_error();
    return 0;
  }
  if (!k || !v) return grm::fail(-1, "null keys or values");
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
  const dim3 grid(static_cast<unsigned>(l.cap_append), static_cast<unsigned>(c->kv_heads), 2);
  const auto s = static_cast<hipStream_t>(stream);
  if (dtype == grm::kF32) append_kernel<F32><<<grid, kAppendThreads, 0, s>>>(a);
  else if (dtype == grm::kBF16) append_kernel<BF16><<<grid, kAppendThreads, 0, s>>>(a);
  else append_kernel<F16><<<grid, kAppendThreads, 0, s>>>(a);
  GRM_HIP_CHECK(hipGetLastError());
  grm::clear_error();
  return 0;
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
  const dim3 grid(static_cast<unsigned>(rows), 2);
  const auto s = static_cast<hipStream_t>(stream);
  if (dtype == grm::kF32) read_kernel<F32><<<grid, 256, 0, s>>>(a);
  else if (dtype == grm::kBF16) read_kernel<BF16><<<grid, 256, 0, s>>>(a);
  else read_kernel<F16><<<grid, 256, 0, s>>>(a);
  GRM_HIP_CHECK(hipGetLastError());
  grm::clear_error();
  return 0;
}
