// kv_common.hpp -- what the 8-bit key/value cache's entry points share: the
// checked descriptors, the schedule a step's plan leaves for append and
// attend, and conversions of the storage types.
#pragma once

#include "grm_common.hpp"
#include "grm_hip_router.h"

#include <algorithm>

namespace grm {
namespace kv {

constexpr int kTile = 64;         // key tokens to a tile of the wide kernel
constexpr int kNarrowCols = 16;   // (token, head) columns of a narrow unit
constexpr int kWideCols = 128;    // and of a wide one
constexpr int kLeastShare = 8;    // key tiles that a wide unit is cut by, at least
// A length read from the device is cut to this: two of them and a block fit
// an int.
constexpr int kMaxLen = (1 << 30) - 256;

// Head of the schedule in device memory (written by the plan).
struct SchedHead {
  int32_t appends;       // (request, block) pairs that take new tokens
  int32_t units;         // narrow units: a request whose columns fit kNarrowCols
  int32_t narrow_tiles;  // their key tiles in all
  int32_t items;         // wide items
  int32_t joins;         // wide units cut into several items
  int32_t pad[11];
};
static_assert(sizeof(SchedHead) == 64, "the lists behind it stay aligned");

// One touched block: `count` new rows from `row` on go to places
// [place, place + count) of physical block `block`.
struct AppendItem {
  int32_t block, row, place, count;
};

// One narrow unit: all of a request's new tokens, for every kv head.
struct NarrowUnit {
  int32_t request, row, tokens, tile_lo;
  int32_t ctx, pad[3];
};

// Key tokens to a tile of the narrow kernel: both halves of a 128-token
// block's value lines, else the least that fills its loads.
__host__ __device__ constexpr int narrow_tile(int block_tokens) {
  return block_tokens == 128 ? 128 : 64;
}

// Runs of the narrow kernel to a kv head, with `per_cu` blocks of four to a CU.
inline int narrow_runs(int cus, int kv_heads, int per_cu) {
  return 4 * std::max(1, per_cu * cus / kv_heads);
}

// Tiles dealt to runs, equal to within one: the first `rem` of the `used`
// runs have `each` + 1 tiles.
struct Deal {
  int tiles, used, each, rem;
  __host__ __device__ Deal(int tiles_, int runs)
      : tiles(tiles_), used(runs < tiles_ ? runs : tiles_),
        each(used ? tiles_ / used : 0), rem(used ? tiles_ % used : 0) {}
  // First tile of run r.
  __host__ __device__ int begin(int r) const {
    return r >= used ? tiles : r * each + (r < rem ? r : rem);
  }
  // The run that tile t lies in.
  __host__ __device__ int run(int t) const {
    const int more = rem * (each + 1);
    return t < more ? t / (each + 1) : rem + (t - more) / each;
  }
};

// A wide unit while the plan cuts it: tokens from t0 on of a request, key
// tiles [lo, hi).
struct WideUnit {
  int32_t request, t0, lo, hi;
};

// One wide item: query rows [row, row + tokens) of a request against key
// tiles [tile_lo, tile_hi); the first of them has position `pos`.  part:
// where the partial result goes, -1 where the item is the whole unit.
struct WideItem {
  int32_t request, row, tokens, pos;
  int32_t tile_lo, tile_hi, part, pad;
};

// One cut wide unit: its parts are consecutive.
struct WideJoin {
  int32_t row, tokens, part, parts;
};

// What the plan wrote, as memory that no kernel running beside this one
// changes: scalar loads where the address is uniform.
typedef const __attribute__((address_space(4))) SchedHead* ConstHead;
typedef const __attribute__((address_space(4))) AppendItem* ConstAppend;
typedef const __attribute__((address_space(4))) NarrowUnit* ConstUnit;
typedef const __attribute__((address_space(4))) WideItem* ConstItem;
typedef const __attribute__((address_space(4))) int32_t* ConstInt;

// Sizes and places of the schedule, from host-known fields alone.
struct Layout {
  int group;          // query heads to a kv head
  int wide_tokens;    // tokens to a wide unit (0: no wide units)
  int wide_blocks;    // wide blocks that run at once, per kv head
  uint64_t cap_append, cap_units, cap_wide, cap_items, cap_joins, cap_parts;
  int32_t reach;      // tokens of a request that the table has blocks for
  int runs[2];        // of the narrow kernel, with one and two blocks to a CU
  uint64_t at_append, at_units, at_tiles, at_run_units[2], at_scan, at_wide, at_items, at_joins, bytes;
};

int device_cus(int* out);
int layout_of(const grm_kv_batch_desc* b, Layout* out);
int check_batch(const grm_kv_batch_desc* b, bool with_arrays);
int check_cache(const grm_kv_cache_desc* c);
int check_pair(const grm_kv_cache_desc* c, const grm_kv_batch_desc* b, bool with_arrays);

// A launch's first dimension holds fewer than 2^32 threads: so many blocks of 256.
constexpr uint64_t kMaxBlocks = 0xffffffffull / 256;
inline int check_blocks(uint64_t blocks) {
  return blocks > kMaxBlocks ? fail(-1, "too many rows for one call") : 0;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// ---------------------------------------------------------- storage types

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

struct F32 {
  typedef float store;
  static constexpr int code = kF32;
  static __device__ float get(float v) { return v; }
  static __device__ float put(float v) { return v; }
};
struct BF16 {
  typedef uint16_t store;
  static constexpr int code = kBF16;
  static __device__ float get(uint16_t v) { return __uint_as_float(static_cast<uint32_t>(v) << 16); }
  static __device__ uint16_t put(float v) {
    const __bf16 h = static_cast<__bf16>(v);
    return __builtin_bit_cast(uint16_t, h);
  }
};
struct F16 {
  typedef uint16_t store;
  static constexpr int code = kF16;
  static __device__ float get(uint16_t v) {
    return static_cast<float>(__builtin_bit_cast(_Float16, v));
  }
  // the empty asm keeps the fp32 value a value of its own: fused into one
  // instruction with the product before it, it would be rounded once only
  static __device__ uint16_t put(float v) {
    asm volatile("" : "+v"(v));
    const _Float16 h = static_cast<_Float16>(v);
    return __builtin_bit_cast(uint16_t, h);
  }
};

__device__ inline int clamp_len(int v) { return v < 0 ? 0 : (v > kMaxLen ? kMaxLen : v); }

__device__ inline int code_at(uint32_t word, int byte) {
  return static_cast<int>(static_cast<int8_t>((word >> (8 * byte)) & 0xffu));
}

// The last unit whose first tile is not past t (wave-uniform; first tiles
// ascend).  64 entries a step.
template <class P>
__device__ inline int find_unit(P first, int n, int t) {
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

}  // namespace kv
}  // namespace grm
