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

// Where a wavefront of the narrow kernel begins: its run [begin, stop) of all
// narrow tiles in order, its block's [block_begin, block_stop), and the unit
// of the first tile (index, its tiles [first, end), the unit itself).
struct NarrowRun {
  int32_t begin, stop, block_begin, block_stop;
  int32_t at, first, end, request;
  int32_t row, tokens, tile_lo, ctx;
  int32_t pad[4];
};
static_assert(sizeof(NarrowRun) == 64, "one line");

// Key tokens to a tile of the narrow kernel: both halves of a 128-token
// block's value lines, else the least that fills its loads.
__host__ __device__ constexpr int narrow_tile(int block_tokens) {
  return block_tokens == 128 ? 128 : 64;
}

// Runs of the narrow kernel to a kv head, with `per_cu` blocks of four to a CU.
inline int narrow_runs(int cus, int kv_heads, int per_cu) {
  return 4 * std::max(1, per_cu * cus / kv_heads);
}

// First tile of run r of `runs`, `tiles` in all; equal to within one.
__host__ __device__ inline int run_begin(int tiles, int runs, int r) {
  const int used = runs < tiles ? runs : tiles;
  if (r >= used) return tiles;
  return static_cast<int>(static_cast<uint64_t>(tiles) * static_cast<uint32_t>(r) /
                          static_cast<uint32_t>(used));
}

// The run that tile t lies in.
__device__ inline int run_of(int tiles, int runs, int t) {
  const int used = runs < tiles ? runs : tiles;
  return static_cast<int>((static_cast<uint64_t>(t + 1) * static_cast<uint32_t>(used) - 1) /
                          static_cast<uint32_t>(tiles));
}

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

// Sizes and places of the schedule, from host-known fields alone.
struct Layout {
  int group;          // query heads to a kv head
  int wide_tokens;    // tokens to a wide unit (0: no wide units)
  int wide_blocks;    // wide blocks that run at once, per kv head
  uint64_t cap_append, cap_units, cap_items, cap_joins, cap_parts;
  int runs[2];        // of the narrow kernel, with one and two blocks to a CU
  uint64_t at_append, at_units, at_tiles, at_runs[2], at_scan, at_items, at_joins, bytes;
};

int device_cus(int* out);
int layout_of(const grm_kv_batch_desc* b, Layout* out);
int check_batch(const grm_kv_batch_desc* b, bool with_arrays);
int check_cache(const grm_kv_cache_desc* c);
int check_pair(const grm_kv_cache_desc* c, const grm_kv_batch_desc* b);

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// ---------------------------------------------------------- storage types

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
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

}  // namespace kv
}  // namespace grm
