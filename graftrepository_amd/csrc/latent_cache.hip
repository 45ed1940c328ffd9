// latent_cache.hip -- rows of the latent cache: a step's latents and key parts
// into their places, and rows read back dense.  Both are bytes: a value is read
// and written once.  20 thousand rows of 576 values from fp32 to bf16 take 14 us (69 MB,
// 4.8 TB/s).
#include "latent_common.hpp"

namespace grm {
namespace kv {

static bool is_16bit(int dtype) { return dtype == kBF16 || dtype == kF16; }
static bool is_float(int dtype) { return dtype == kF32 || is_16bit(dtype); }

int check_latent(const grm_latent_desc* c) {
  if (!c) return fail(-1, "null cache");
  if (c->block_tokens != 16 && c->block_tokens != 32 && c->block_tokens != 64 &&
      c->block_tokens != 128) {
    return fail(-1, "block_tokens must be 16, 32, 64 or 128");
  }
  if (c->rank <= 0 || c->rank > 512 || c->rank % 16 != 0) {
    return fail(-1, "rank must be a multiple of 16, at most 512");
  }
  if (c->rope < 0 || c->rope > 128 || c->rope % 16 != 0) {
    return fail(-1, "rope must be a multiple of 16, at most 128");
  }
  if (!is_16bit(c->dtype)) return fail(-1, "latent rows are BF16 or F16");
  if (c->blocks == 0 || c->blocks > 0x7fffffffull) return fail(-1, "bad block count");
  if (!c->rows) return fail(-1, "null rows");
  if (!aligned16(c->rows)) return fail(-1, "rows must be 16-byte aligned");
  return 0;
}

int check_latent_pair(const grm_latent_desc* c, const grm_kv_batch_desc* b, bool with_arrays) {
  GRM_CHECK_RC(check_latent(c));
  GRM_CHECK_RC(check_batch(b, with_arrays));
  if (c->block_tokens != b->block_tokens) return fail(-1, "cache and batch differ in block_tokens");
  if (b->kv_heads != 1) return fail(-1, "a latent cache's batch has one kv head");
  return 0;
}

int check_ranges(const int32_t* block_table, int table_width, int requests, const int32_t* starts,
                 const int32_t* cu_rows, uint64_t rows) {
  if (requests < 0 || table_width < 0) return fail(-1, "negative size");
  if (rows > static_cast<uint64_t>(kMaxLen)) return fail(-1, "too many rows");
  if (rows == 0) return 0;
  if (requests == 0) return fail(-1, "rows of no request");
  if (!starts || !cu_rows || (table_width > 0 && !block_table)) return fail(-1, "null array");
  return 0;
}

// ----------------------------------------------------------------- append

struct LatentAppendArgs {
  uint16_t* rows;
  const void* latents;
  const void* keys;
  const int64_t* slots;
  const int32_t* positions;
  int64_t latent_stride, key_stride;
  uint64_t cache_rows;
  int32_t tokens, rank, rope, turned;
};

constexpr int kRowThreads = 256;

// A thread brings 16 values of a token: of its latent, or eight pairs of its key
// part (whose angles no other thread needs).
template <class S, class D, bool ALIGNED>
__global__ __launch_bounds__(kRowThreads) void latent_append_kernel(LatentAppendArgs a, Rotary r) {
  const int each = (a.rank + a.rope) / 16;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kRowThreads + threadIdx.x;
  if (i >= static_cast<int64_t>(a.tokens) * each) return;
  // the key parts first: their angles take longest
  const int t = static_cast<int>(i / each), u = static_cast<int>(i - static_cast<int64_t>(t) * each);
  const int64_t slot = a.slots[t];
  if (slot < 0 || static_cast<uint64_t>(slot) >= a.cache_rows) return;
  uint16_t* to = a.rows + slot * (a.rank + a.rope);
  const int key_units = a.rope / 16;
  float v[2][8];
  int first, second;
  if (u < key_units) {
    const typename S::store* x = static_cast<const typename S::store*>(a.keys) + t * a.key_stride;
    if (u < a.turned) {
      unit_channels(r.layout, r.dim / 2, u, &first, &second);
    } else {
      first = 16 * u;
      second = first + 8;
    }
    get8<S, ALIGNED>(x + first, v[0]);
    get8<S, ALIGNED>(x + second, v[1]);
    if (u < a.turned) {
      const int position = a.positions[t];
      turn_unit(r.layout, v, [&](int e) { return angle(r, 8 * u + e, position); });
    }
    first += a.rank;
    second += a.rank;
  } else {
    const typename S::store* x =
        static_cast<const typename S::store*>(a.latents) + t * a.latent_stride;
    first = 16 * (u - key_units);
    second = first + 8;
    get8<S, ALIGNED>(x + first, v[0]);
    get8<S, ALIGNED>(x + second, v[1]);
  }
  put8<D, true>(to + first, v[0]);
  put8<D, true>(to + second, v[1]);
}

template <class S>
static void launch_latent_append(const LatentAppendArgs& a, const Rotary& r, int dtype, bool aligned,
                                 hipStream_t s) {
  const int64_t items = static_cast<int64_t>(a.tokens) * ((a.rank + a.rope) / 16);
  const auto grid = static_cast<unsigned>((items + kRowThreads - 1) / kRowThreads);
  if (dtype == kBF16) {
    if (aligned) latent_append_kernel<S, BF16, true><<<grid, kRowThreads, 0, s>>>(a, r);
    else latent_append_kernel<S, BF16, false><<<grid, kRowThreads, 0, s>>>(a, r);
  } else {
    if (aligned) latent_append_kernel<S, F16, true><<<grid, kRowThreads, 0, s>>>(a, r);
    else latent_append_kernel<S, F16, false><<<grid, kRowThreads, 0, s>>>(a, r);
  }
}

// ------------------------------------------------------------------- read

struct LatentReadArgs {
  const uint16_t* rows;
  void* out;
  RowRanges of;
  int32_t values;  // of a row
};

constexpr int kReadRowsEach = 16;

// A block finds the places of 16 rows (one chain of loads for all), and copies
// them 8 values to a thread.
template <class S, class D>
__global__ __launch_bounds__(kRowThreads) void latent_read_kernel(LatentReadArgs a) {
  __shared__ int64_t s_row[kReadRowsEach];
  const uint64_t row0 = static_cast<uint64_t>(blockIdx.x) * kReadRowsEach;
  if (threadIdx.x < kReadRowsEach) {
    s_row[threadIdx.x] = cache_row(a.of, static_cast<int>(row0) + static_cast<int>(threadIdx.x));
  }
  __syncthreads();
  const int each = a.values / 8;
  const int n = static_cast<int>(min(static_cast<uint64_t>(kReadRowsEach), a.of.rows - row0));
  for (int i = threadIdx.x; i < n * each; i += kRowThreads) {
    const int t = i / each, d = 8 * (i - t * each);
    float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (s_row[t] >= 0) get8<S, true>(a.rows + s_row[t] * a.values + d, v);
    put8<D, true>(static_cast<typename D::store*>(a.out) + (row0 + t) * a.values + d, v);
  }
}

template <class S>
static void launch_latent_read(const LatentReadArgs& a, int dtype, hipStream_t s) {
  const auto grid = static_cast<unsigned>((a.of.rows + kReadRowsEach - 1) / kReadRowsEach);
  if (dtype == kF32) latent_read_kernel<S, F32><<<grid, kRowThreads, 0, s>>>(a);
  else if (dtype == kBF16) latent_read_kernel<S, BF16><<<grid, kRowThreads, 0, s>>>(a);
  else latent_read_kernel<S, F16><<<grid, kRowThreads, 0, s>>>(a);
}

}  // namespace kv
}  // namespace grm

using namespace grm::kv;

extern "C" int grm_hip_latent_append(const grm_latent_desc* c, const grm_kv_batch_desc* b,
                                     const grm_rotary_desc* rotary, const void* latents,
                                     const void* keys, int dtype, int64_t latent_token_stride,
                                     int64_t key_token_stride, void* stream) {
  GRM_CHECK_RC(check_latent_pair(c, b, true));
  if (!is_float(dtype)) return grm::fail(-1, "latents and key parts are F32, BF16 or F16");
  Rotary r{};
  if (rotary) {
    GRM_CHECK_RC(rotary_of(rotary, c->rope, &r));
    if (!whole_units(r)) return grm::fail(-1, "a latent cache's rotary turns a multiple of 16 channels");
  }
  if (b->requests == 0 || b->tokens == 0) {
    grm::clear_error();
    return 0;
  }
  if (!latents || (c->rope && !keys)) return grm::fail(-1, "null latents or key parts");
  if (!b->slot_map || (rotary && !b->positions)) {
    return grm::fail(-1, "the batch has no slot map or no positions");
  }
  LatentAppendArgs a{};
  a.rows = static_cast<uint16_t*>(c->rows);
  a.latents = latents;
  a.keys = keys;
  a.slots = b->slot_map;
  a.positions = b->positions;
  a.latent_stride = latent_token_stride;
  a.key_stride = key_token_stride;
  a.cache_rows = c->blocks * static_cast<uint64_t>(c->block_tokens);
  a.tokens = b->tokens;
  a.rank = c->rank;
  a.rope = c->rope;
  a.turned = r.dim / 16;
  const int64_t items = static_cast<int64_t>(a.tokens) * ((a.rank + a.rope) / 16);
  GRM_CHECK_RC(check_blocks((items + kRowThreads - 1) / kRowThreads));
  const int64_t unit = dtype == grm::kF32 ? 4 : 8;
  const bool aligned = aligned16(latents) && aligned16(keys) &&
                       (latent_token_stride | (c->rope ? key_token_stride : 0)) % unit == 0;
  const auto s = static_cast<hipStream_t>(stream);
  if (dtype == grm::kF32) launch_latent_append<F32>(a, r, c->dtype, aligned, s);
  else if (dtype == grm::kBF16) launch_latent_append<BF16>(a, r, c->dtype, aligned, s);
  else launch_latent_append<F16>(a, r, c->dtype, aligned, s);
  GRM_HIP_CHECK(hipGetLastError());
  grm::clear_error();
  return 0;
}

extern "C" int grm_hip_latent_read(const grm_latent_desc* c, const int32_t* block_table,
                                   int table_width, int requests, const int32_t* starts,
                                   const int32_t* cu_rows, uint64_t rows, int dtype, void* out,
                                   void* stream) {
  GRM_CHECK_RC(check_latent(c));
  if (!is_float(dtype)) return grm::fail(-1, "rows are read as F32, BF16 or F16");
  GRM_CHECK_RC(check_ranges(block_table, table_width, requests, starts, cu_rows, rows));
  if (rows == 0) {
    grm::clear_error();
    return 0;
  }
  if (!out || !aligned16(out)) return grm::fail(-1, "output must be 16-byte aligned");
  GRM_CHECK_RC(check_blocks((rows + kReadRowsEach - 1) / kReadRowsEach));
  LatentReadArgs a{};
  a.rows = static_cast<const uint16_t*>(c->rows);
  a.out = out;
  a.of = {block_table, starts, cu_rows, table_width, requests, block_log2(c->block_tokens), rows,
          c->blocks};
  a.values = c->rank + c->rope;
  const auto s = static_cast<hipStream_t>(stream);
  if (c->dtype == grm::kBF16) launch_latent_read<BF16>(a, dtype, s);
  else launch_latent_read<F16>(a, dtype, s);
  GRM_HIP_CHECK(hipGetLastError());
  grm::clear_error();
  return 0;
}
