// latent_expand.hip -- the expanded form of latent attention: a head's own keys and
// values from cached latents, and causal attention over such dense rows.
//
//   k[row, head] = [W_k[head] c | key part],  v[row, head] = W_v[head] c
//
// An expansion is a matrix product whose left operand is gathered through the
// block table; a prompt of n tokens needs 2 n (dk + dv) operations a key after it,
// where the absorbed form needs 2 n (2 rank + rope).
#include "latent_attend.hpp"

namespace grm {
namespace kv {

// ----------------------------------------------------------------- expand

struct ExpandArgs {
  const uint16_t* rows;
  const uint16_t* weight;  // [heads][key_dim + value_dim][rank]
  uint16_t* k;             // [rows][heads][key_dim + rope]
  uint16_t* v;             // [rows][heads][value_dim]
  RowRanges of;
  int32_t rank, rope, heads, key_dim, value_dim;
};

// 128 rows x 256 columns to a block, 64 x 128 to a wavefront, 32 of the rank a
// stage; three stages of direct loads in LDS, two blocks to a CU, so that one's
// stores run beside the other's products.  Bound by the rounds of so few steps (16 at
// rank 512) and their ends: 4096 rows of 32 heads x 256 columns take 50 us (688
// TFLOP/s), 4137 rows 57; torch's product of the same sizes without the gather, in
// one plane, 47 and 73.  Chunks of 16 bytes are stored at c ^ (row >> 3
// & 3) of their 64: the 16 rows that are read at once lie in all banks.  Results
// leave through LDS, 16 bytes to a lane.
constexpr int kExpandRows = 128, kExpandCols = 256, kExpandStep = 32, kExpandStages = 3;
constexpr int kExpandStage = (kExpandRows + kExpandCols) * kExpandStep * 2;  // bytes
constexpr int kExpandOut = kExpandCols * 2 + 16;                             // of a row on its way out

template <class T>
__global__ __launch_bounds__(256, 2) void latent_expand_kernel(ExpandArgs a) {
  __shared__ __align__(1024) char lds[kExpandStages * kExpandStage];
  __shared__ int64_t s_row[kExpandRows];
  static_assert(kExpandRows * kExpandOut <= kExpandStages * kExpandStage, "results fit the ring");
  const int lane = __lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int c = lane % 32, h = lane / 32;
  const int width = a.key_dim + a.value_dim, columns = a.heads * width;
  // Blocks go to the XCDs in turn: with whole eighths of the columns each has its
  // own of the weights, which stay in its L2.
  const int wide = (columns + kExpandCols - 1) / kExpandCols;
  const int col0 = static_cast<int>(blockIdx.x % wide) * kExpandCols;
  const int row0 = static_cast<int>(blockIdx.x / wide) * kExpandRows;
  const int values = a.rank + a.rope;
  if (threadIdx.x < kExpandRows) {
    s_row[threadIdx.x] = cache_row(a.of, row0 + static_cast<int>(threadIdx.x));
  }
  __syncthreads();
  // loads of 16 rows by four chunks: two of cache rows, four of weights
  const int r16 = lane / 4, chunk = (lane % 4) ^ (r16 >> 3);  // of an even load
  const uint16_t* from[6];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t row = s_row[(2 * wave + i) * 16 + r16];
    from[i] = (row >= 0 ? a.rows + row * values : reinterpret_cast<const uint16_t*>(latent_zeros)) + 8 * (chunk ^ 2 * i);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = min(col0 + (4 * wave + i) * 16 + r16, columns - 1);
    from[2 + i] = a.weight + static_cast<int64_t>(n) * a.rank + 8 * (chunk ^ 2 * (i & 1));
  }
  auto issue = [&](int step) {
    const uint32_t to = lds_address(lds) + (step % kExpandStages) * kExpandStage;
#pragma unroll
    for (int i = 0; i < 6; ++i) {
      load_direct(from[i] + step * kExpandStep,
                  i < 2 ? to + (2 * wave + i) * 1024
                        : to + kExpandRows * kExpandStep * 2 + (4 * wave + i - 2) * 1024);
    }
  };
  const int steps = a.rank / kExpandStep;
  issue(0);
  if (steps > 1) issue(1);

  const int wave_row = 64 * (wave & 1), wave_col = 128 * (wave >> 1);
  f32x16 acc[2][4];  // [rows][columns]: a lane's column of 32 is a row, its results columns
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
    }
  }
  const int at = c * 64 + 16 * (h ^ (c >> 3 & 3));
  for (int s = 0; s < steps; ++s) {
    if (s + 1 < steps) wait_loads<6>();
    else wait_loads<0>();
    block_barrier();
    if (s + 2 < steps) issue(s + 2);
    const char* rows = lds + (s % kExpandStages) * kExpandStage + wave_row * 64;
    const char* cols = lds + (s % kExpandStages) * kExpandStage + kExpandRows * 64 + wave_col * 64;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      u32x4 x[2], w[4];
#pragma unroll
      for (int i = 0; i < 2; ++i) x[i] = *reinterpret_cast<const u32x4*>(rows + i * 32 * 64 + (at ^ 32 * k));
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = *reinterpret_cast<const u32x4*>(cols + j * 32 * 64 + (at ^ 32 * k));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int i = 0; i < 2; ++i) acc[i][j] = mfma<T::code == kBF16>(w[j], x[i], acc[i][j]);
      }
    }
  }
  wait_loads<0>();
  block_barrier();  // the ring is read
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        u32x2 v;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t lo = T::put(acc[i][j][4 * q + 2 * e]), hi = T::put(acc[i][j][4 * q + 2 * e + 1]);
          v[e] = lo | (hi << 16);
        }
        *reinterpret_cast<u32x2*>(lds + (wave_row + 32 * i + c) * kExpandOut +
                                  2 * (wave_col + 32 * j + 8 * q + 4 * h)) = v;
      }
    }
  }
  __syncthreads();
  const int rows_here = static_cast<int>(min(static_cast<uint64_t>(kExpandRows), a.of.rows - row0));
  {
    // a thread's eight columns stay, its row goes on by eight
    const int n = col0 + 8 * (static_cast<int>(threadIdx.x) % 32);
    if (n < columns) {
      const int head = n / width, d = n - head * width;
      const bool key = d < a.key_dim;
      const int64_t stride = static_cast<int64_t>(a.heads) * (key ? a.key_dim + a.rope : a.value_dim);
      uint16_t* to = key ? a.k + static_cast<int64_t>(head) * (a.key_dim + a.rope) + d
                         : a.v + static_cast<int64_t>(head) * a.value_dim + d - a.key_dim;
      for (int r = threadIdx.x / 32; r < rows_here; r += 8) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(lds + r * kExpandOut + 2 * (n - col0));
        *reinterpret_cast<u32x4*>(to + (row0 + r) * stride) = x;
      }
    }
  }
  // the key parts of the heads that begin in this block's columns
  const int first = (col0 + width - 1) / width, last = min(a.heads, (col0 + kExpandCols + width - 1) / width);
  const int chunks = a.rope / 8, each = chunks * (last - first);
  for (int i = threadIdx.x; i < each * rows_here; i += 256) {
    const int r = i / each, j = i - r * each, head = first + j / chunks, d = 8 * (j % chunks);
    const int64_t row = s_row[r];
    u32x4 x = {0u, 0u, 0u, 0u};
    if (row >= 0) x = *reinterpret_cast<const u32x4*>(a.rows + row * values + a.rank + d);
    *reinterpret_cast<u32x4*>(a.k + (static_cast<int64_t>(row0 + r) * a.heads + head) * (a.key_dim + a.rope) +
                              a.key_dim + d) = x;
  }
}

// Ranks that are no whole stages: a row to a block, its latent in LDS.
template <class T>
__global__ __launch_bounds__(256) void latent_expand_any_kernel(ExpandArgs a) {
  __shared__ float s_c[512];
  const int row = blockIdx.x, values = a.rank + a.rope, width = a.key_dim + a.value_dim;
  const int64_t at = cache_row(a.of, row);
  for (int d = threadIdx.x; d < a.rank; d += 256) s_c[d] = at >= 0 ? T::get(a.rows[at * values + d]) : 0.0f;
  __syncthreads();
  for (int n = threadIdx.x; n < a.heads * width; n += 256) {
    float sum = 0.0f;
    for (int d = 0; d < a.rank; d += 8) {
      float w[8];
      get8<T, true>(a.weight + static_cast<int64_t>(n) * a.rank + d, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = fmaf(w[e], s_c[d + e], sum);
    }
    const int head = n / width, d = n - head * width;
    if (d < a.key_dim) a.k[(static_cast<int64_t>(row) * a.heads + head) * (a.key_dim + a.rope) + d] = T::put(sum);
    else a.v[(static_cast<int64_t>(row) * a.heads + head) * a.value_dim + d - a.key_dim] = T::put(sum);
  }
  for (int i = threadIdx.x; i < a.heads * a.rope; i += 256) {
    const int head = i / a.rope, d = i - head * a.rope;
    a.k[(static_cast<int64_t>(row) * a.heads + head) * (a.key_dim + a.rope) + a.key_dim + d] =
        at >= 0 ? a.rows[at * values + a.rank + d] : uint16_t{0};
  }
}

// ------------------------------------------------- attention over dense rows

struct RowsArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* out;
  float* lse;
  const int32_t* cu_new;
  const int32_t* ctx_lens;
  const int32_t* cu_rows;
  const int32_t* starts;  // NULL: 0
  const char* work;
  int64_t q_token, q_head, k_row, k_head, v_row, v_head, out_token, out_head;
  float* parts;
  uint64_t at_items, at_row_joins;
  SumUnit unit;
  float scale;
  int32_t requests, tokens, window, heads, key_dim, value_dim, rows;
};

// A unit's rows: where its request's begin, how many there are, the first's
// position.
struct KeyRows {
  int first, count, start;
};
__device__ inline KeyRows key_rows(const RowsArgs& a, int request) {
  KeyRows k;
  k.first = a.cu_rows[request];
  const int end = min(a.cu_rows[request + 1], a.rows);
  k.first = max(0, min(k.first, a.rows));
  k.count = max(0, end - k.first);
  k.start = a.starts ? max(-kMaxLen, min(a.starts[request], kMaxLen)) : 0;
  return k;
}

// 128 tokens of a head to a block, 32 to a wavefront, against tiles of 32 rows that
// all four read from LDS: the layout and the softmax of latent_attend.hpp, with a
// head's own keys and values.
//
// In a wavefront, vector work stands beside matrix work: a tile's weights are made
// between the instructions of the next tile's first product (each of which takes the
// matrix cores eight times as long as its issue).  So a tile's keys are read one tile
// before its values: three tiles of keys in LDS and four of values, two blocks to a
// CU.  The rest is one stream of tiles: those that all columns see are asked nothing.
//
// Bound by the matrix cores on long rows: a prompt of 16384 tokens, 32 heads of 192 and
// 128, 1083 TFLOP/s in bf16 (a large matrix product here has 1221); 40 heads of 96
// and 64 in fp16 845, where a tile's vector instructions take as long as its
// products.  Short ones by a unit's ends, about ten tiles' time each, and the
// slots that stay empty at the end: 4096 tokens 899, 1024 tokens 346.
//
// A unit of 128 tokens is cut where there are fewer than the blocks that fit: by the
// plan, at the share of eight for which the longest-first order ends first.
template <class T, int DK, int DV>
struct RowsShape {
  static constexpr int kKeyBytes = (2 * DK + 127) / 128 * 128;  // of a row in LDS
  static constexpr int kValueBytes = 2 * DV;
  static constexpr int kKeyTile = kLatentTile * kKeyBytes, kValueTile = kLatentTile * kValueBytes;
  static constexpr int kKeyStages = 3, kValueStages = 4;
  static constexpr int kValuesAt = kKeyStages * kKeyTile;
  static constexpr int kLds = kValuesAt + kValueStages * kValueTile;
  // direct loads of a wavefront
  static constexpr int kKeyLoads = kKeyTile / 4096, kValueLoads = kValueTile / 4096;
  static constexpr int kLoads = kKeyLoads + kValueLoads;
  static constexpr int kSteps = DK / 16, kTilesD = DV / 32;
  static constexpr bool kBf = T::code == kBF16;
  static constexpr float kSlack = slack_of(T::code), kBias = kBf ? 0.0f : 13.0f;
  // Where a row's chunks of 16 bytes go: chunk c to c ^ turn.  A 16-byte read is served
  // 16 lanes at a time (0-3, 12-15, 20-23, 24-27; 4-11, 16-19, 28-31; and so on), whose
  // rows are then in all 64 banks.
  static __device__ __forceinline__ int key_turn(int row) {
    return (row >> 2 & 3) + (kKeyBytes % 256 == 0 ? 4 * (row & 3) : 4 * (row >> 1 & 1));
  }
  // A transposed read takes 64 bytes of each of four rows, which then lie in all
  // banks.  The same for every fourth row, so that these are a constant apart.
  static __device__ __forceinline__ int value_turn(int row) {
    return kValueBytes % 256 == 0 ? 4 * (row & 3) : 4 * (row >> 1 & 1);
  }
};

// Floats of a part: its sums as the wavefronts have them, maxima, sums of weights.
__host__ __device__ constexpr size_t rows_part_floats(int value_dim) {
  return static_cast<size_t>(kRowUnit) * (value_dim + 2);
}

// A unit's piece.  Values that are no finite numbers (in a row that no column sees, with
// a weight of 0; a score of -inf, which would hide its row) take questions at every tile
// that is seen in part.  Without CAREFUL there are none: at its end such a thing shows
// in the sums or in the least score, nothing is written then, and the answer is
// false.  (With the questions three prompts took 117 us in place of 112, a chunk of 1021
// tokens 119 in place of 110.)
template <class T, int DK, int DV, bool CAREFUL>
__device__ __forceinline__ bool attend_piece(const RowsArgs& a, int head, const RowItem& u, char* ring,
                                             uint32_t* s_bad) {
  typedef RowsShape<T, DK, DV> S;
  const int lane = __lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int c = lane % 32, h = lane / 32;
  const int tokens = u.tokens, first_pos = u.pos, unit_row = u.row, part = u.part;
  const KeyRows keys = key_rows(a, u.request);
  const int last_pos = first_pos + tokens - 1;
  // columns: tokens; positions are counted from the rows' first
  const bool mine = 32 * wave + c < tokens;
  const int token = min(32 * wave + c, tokens - 1);
  const int wave_last = first_pos + min(32 * wave + 31, tokens - 1) - keys.start;
  const int wave_first = first_pos + min(32 * wave, tokens - 1) - keys.start;
  const int wave_from = a.window > 0 ? max(0, wave_first + 1 - a.window) : 0;
  const int wave_all_from = a.window > 0 ? max(0, wave_last + 1 - a.window) : 0;
  const bool busy = 32 * wave < tokens;
  const int block_first = first_pos - keys.start;
  const int all_from = a.window > 0 ? max(0, last_pos - keys.start + 1 - a.window) : 0;
  const int block_from = a.window > 0 ? max(0, block_first + 1 - a.window) : 0;
  const int seen_lo = block_from / kLatentTile;
  const int seen_hi = max(seen_lo, (min(last_pos - keys.start + 1, keys.count) + kLatentTile - 1) / kLatentTile);
  const int tile_lo = seen_lo + static_cast<int>(static_cast<int64_t>(seen_hi - seen_lo) * u.piece / u.pieces);
  const int tile_hi = seen_lo + static_cast<int>(static_cast<int64_t>(seen_hi - seen_lo) * (u.piece + 1) / u.pieces);
  const int n = tile_hi - tile_lo;

  // Offsets of this lane's rows in a tile, which stay; a tile past the rows' end has
  // its last row again.
  uint32_t offsets[S::kLoads];
  auto offset_of = [&](int j, int last) {
    const bool key = j < S::kKeyLoads;
    constexpr int kKeyChunks = S::kKeyBytes / 16, kValueChunks = S::kValueBytes / 16;
    const int at = (key ? wave * S::kKeyLoads + j : wave * S::kValueLoads + j - S::kKeyLoads) * kWave + lane;
    const int r = at / (key ? kKeyChunks : kValueChunks), place = at - r * (key ? kKeyChunks : kValueChunks);
    const int chunk = place ^ (key ? S::key_turn(r) : S::value_turn(r));
    // (a row's last places in LDS may be nobody's)
    const int64_t row = static_cast<int64_t>(min(r, last)) * (key ? a.k_row : a.v_row);
    return static_cast<uint32_t>(2 * (row + 8 * (!key || chunk < DK / 8 ? chunk : 0)));
  };
#pragma unroll
  for (int j = 0; j < S::kLoads; ++j) offsets[j] = offset_of(j, kLatentTile);
  // Loads are issued tile after tile: where the next one's rows are, and its places.
  const int64_t row0 = keys.first + static_cast<int64_t>(tile_lo) * kLatentTile;
  const char* next_k = reinterpret_cast<const char*>(a.k + row0 * a.k_row + head * a.k_head);
  const char* next_v = reinterpret_cast<const char*>(a.v + row0 * a.v_row + head * a.v_head);
  const int64_t k_step = 2 * kLatentTile * a.k_row, v_step = 2 * kLatentTile * a.v_row;
  uint32_t to_k = lds_address(ring) + wave * S::kKeyLoads * 1024;
  uint32_t to_v = lds_address(ring) + S::kValuesAt + wave * S::kValueLoads * 1024;
  const uint32_t end_k = to_k + S::kKeyStages * S::kKeyTile, end_v = to_v + S::kValueStages * S::kValueTile;
  int rows_left = keys.count - tile_lo * kLatentTile;
  auto issue = [&]() {
    if (rows_left >= kLatentTile) {
#pragma unroll
      for (int j = 0; j < S::kLoads; ++j) {
        const bool key = j < S::kKeyLoads;
        load_direct(key ? next_k : next_v, offsets[j], key ? to_k + j * 1024 : to_v + (j - S::kKeyLoads) * 1024);
      }
    } else {
#pragma unroll
      for (int j = 0; j < S::kLoads; ++j) {
        const bool key = j < S::kKeyLoads;
        load_direct(key ? next_k : next_v, offset_of(j, rows_left - 1),
                    key ? to_k + j * 1024 : to_v + (j - S::kKeyLoads) * 1024);
      }
    }
    next_k += k_step;
    next_v += v_step;
    rows_left -= kLatentTile;
    to_k += S::kKeyTile;
    if (to_k == end_k) to_k -= S::kKeyStages * S::kKeyTile;
    to_v += S::kValueTile;
    if (to_v == end_v) to_v -= S::kValueStages * S::kValueTile;
  };

  u32x4 q[S::kSteps];
  {
    const uint16_t* from = a.q + static_cast<int64_t>(unit_row + token) * a.q_token + head * a.q_head + 8 * h;
#pragma unroll
    for (int s = 0; s < S::kSteps; ++s) q[s] = *reinterpret_cast<const u32x4*>(from + 16 * s);
  }
  if (n > 0) issue();
  if (n > 1) issue();
  // In registers before the loop, so that a stage waits for rows only.
#pragma unroll
  for (int s = 0; s < S::kSteps; ++s) asm volatile("" : "+v"(q[s]));
  asm volatile("" ::: "memory");
  const int key_row = 16 * (c >> 2 & 1) + 4 * (c >> 3) + (c & 3);
  int k_at = key_row * S::kKeyBytes + 16 * (h ^ S::key_turn(key_row));
  const int i16 = lane % 16, v_row = 16 * h + i16 / 4;
  int v_at = S::kValuesAt + v_row * S::kValueBytes + 8 * (i16 & 1) +
                   16 * ((2 * (lane >> 4 & 1) + (i16 % 4 >> 1)) ^ S::value_turn(v_row));
  // (a register each; parts of them, spilled, were read back before every loop, and
  // waited for every direct load)
  asm volatile("" : "+v"(k_at), "+v"(v_at));
  f32x16 o[S::kTilesD];
#pragma unroll
  for (int d = 0; d < S::kTilesD; ++d) {
#pragma unroll
    for (int e = 0; e < 16; ++e) o[d][e] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f, poison = 0.0f, lowest = 0.0f;
  const float mul = a.scale * kLog2e;
  // Exponents' arguments of the tile whose scores were made last: score * scale_by +
  // shift.
  f32x16 scores;
  float scale_by = 1.0f, shift = 0.0f;
#pragma unroll
  for (int e = 0; e < 16; ++e) scores[e] = -INFINITY;
  int k_slot = 0, v_slot = 0;  // of tile i + 1

  // Both products: the scores of the tile in k_stage, left in `then` (not `now`) with
  // their extremes, and where `weigh` says so the values in v_stage by the weights of
  // `now`.  A value's first half needs eight weights, its second the others, so that
  // weights are made beside all instructions but the last half's, and the extremes
  // beside those.
  auto products = [&](auto weigh, const char* k_stage, const char* v_stage, const f32x16& now, f32x16& then,
                      float& top, float& low) {
    constexpr int kScores = S::kSteps, kEarly = kScores + S::kTilesD, kAll = kEarly + S::kTilesD;
    u32x4 w[2];
#pragma unroll
    for (int e = 0; e < 16; ++e) then[e] = 0.0f;
    in_order<decltype(weigh)::value ? kAll : kScores, 4>(
        [&](int k) {
          if (k < kScores) {
            constexpr int kIn = S::kKeyBytes % 256 == 0 ? 8 : 4;  // steps to whole turns
            return *reinterpret_cast<const u32x4*>(k_stage + ((k_at ^ 32 * (k % kIn)) + 32 * (k / kIn * kIn)));
          }
          const int d = (k - kScores) % S::kTilesD, x0 = 2 * ((k - kScores) / S::kTilesD);
          constexpr int kIn = S::kValueBytes % 256 == 0 ? 4 : 2;
          auto four = [&](int x) {  // keys 4 x on of the lane's sixteen
            return read_transposed(v_stage + ((v_at ^ 64 * (d % kIn)) + 64 * (d / kIn * kIn) +
                                              4 * x * S::kValueBytes));
          };
          const u32x2 lo = four(x0), hi = four(x0 + 1);
          return u32x4{lo[0], lo[1], hi[0], hi[1]};
        },
        [&](int k, u32x4 f) {
          if (k < kScores) {
            then = mfma<S::kBf>(f, q[k], then);
          } else {
            const int d = (k - kScores) % S::kTilesD;
            o[d] = mfma<S::kBf>(f, w[k < kEarly ? 0 : 1], o[d]);
          }
          if constexpr (decltype(weigh)::value) {
            if (k < kEarly) {
#pragma unroll
              for (int e = 16 * k / kEarly / 2 * 2; e < 16 * (k + 1) / kEarly / 2 * 2; e += 2) {
                const float x = __builtin_amdgcn_exp2f(fmaf(now[e], scale_by, shift));
                const float y = __builtin_amdgcn_exp2f(fmaf(now[e + 1], scale_by, shift));
                l += x;
                l += y;
                w[e / 8][e % 8 / 2] = two_weights<S::kBf>(x, y, a.unit);
              }
            } else {
              const int d = k - kEarly;
              if (d == 0) top = low = then[0];
#pragma unroll
              for (int e = 16 * d / S::kTilesD; e < 16 * (d + 1) / S::kTilesD; ++e) {
                top = fmaxf(top, then[e]);
                low = fminf(low, then[e]);
              }
            }
          }
        });
    if constexpr (!decltype(weigh)::value) {
      top = low = then[0];
#pragma unroll
      for (int e = 1; e < 16; ++e) {
        top = fmaxf(top, then[e]);
        low = fminf(low, then[e]);
      }
    }
  };
  // Scores of a tile from key0 on as arguments: what no column sees out of them, and
  // the reference moved where one passes it.  `whole`: all columns see all rows.
  auto settle = [&](f32x16& s, float top, float low, int key0, bool whole, uint32_t bad) {
    scale_by = mul;
    // NaN and +inf make their column's sums so by themselves; a weight of 0 would hide
    // -inf (with a negative scale +inf).
    if (!CAREFUL) lowest = fminf(lowest, mul < 0.0f ? -top : low);
    if (whole && !(CAREFUL && __any(low < -3.4028235e38f))) {
      top *= mul;
    } else {
      const int pos = first_pos + token - keys.start;
      // of the lane's sixteen keys it sees from `from` to `to`
      const int at = key0 + 16 * h;
      const int from = a.window > 0 ? max(0, pos + 1 - a.window) - at : 0;
      const int to = min(pos, keys.count - 1) - at;
      scale_by = 1.0f;
      if constexpr (CAREFUL) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const bool see = e <= to && e >= from;
          const bool fine = fabsf(s[e]) <= 3.4028235e38f;
          poison += see && (!fine || (bad >> (16 * h + e) & 1u)) ? NAN : 0.0f;
          s[e] = see && fine ? s[e] * mul : -INFINITY;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = e <= to ? s[e] * mul : -INFINITY;
        if (__any(from > 0)) {
#pragma unroll
          for (int e = 0; e < 16; ++e) s[e] = e >= from ? s[e] : -INFINITY;
        }
      }
      top = s[0];
#pragma unroll
      for (int e = 1; e < 16; ++e) top = fmaxf(top, s[e]);
    }
    if (__any(top > m + S::kSlack)) {
      float m2 = fmaxf(m, top);
      m2 = fmaxf(m2, __shfl_xor(m2, 32));
      const float keep = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - m2);
      if (__any(m != -INFINITY)) {
#pragma unroll
        for (int d = 0; d < S::kTilesD; ++d) o[d] *= keep;
      }
      l *= keep;
      m = m2;
      shift = S::kBias - (m == -INFINITY ? 0.0f : m);
    }
  };
  shift = S::kBias;
  auto turn_slots = [&]() {
    k_slot = k_slot == (S::kKeyStages - 1) * S::kKeyTile ? 0 : k_slot + S::kKeyTile;
    v_slot = v_slot == (S::kValueStages - 1) * S::kValueTile ? 0 : v_slot + S::kValueTile;
  };
  auto values_before = [&]() {  // of tile i
    return ring + (v_slot ? v_slot : S::kValueStages * S::kValueTile) - S::kValueTile;
  };

  // Step i: scores of tile i + 1 beside the weights of tile i, then tile i's values.
  auto step = [&](int i) {
    uint32_t bad = 0;
    const int key0 = (tile_lo + i + 1) * kLatentTile;
    if (i + 1 < n) {
      if (i + 2 < n) wait_loads<S::kLoads>();
      else wait_loads<0>();
      block_barrier();
      if (i + 3 < n) issue();
      // Where some column does not see all rows, values that are no finite numbers
      // (which a weight of 0 would not keep out) are taken from LDS, and the rows
      // that had them noted.
      const bool partly =
          CAREFUL && (key0 < all_from || key0 + kLatentTile - 1 > min(block_first, keys.count - 1));
      if (CAREFUL && threadIdx.x == 0) s_bad[i & 1] = 0;  // all have read it before this step
      if (partly) {
        constexpr uint32_t kLo = S::kBf ? 0x7f80u : 0x7c00u, kHi = kLo << 16;
        char* values = ring + S::kValuesAt + v_slot;
#pragma unroll
        for (int at = 16 * static_cast<int>(threadIdx.x); at < S::kValueTile; at += 4096) {
          u32x4* p = reinterpret_cast<u32x4*>(values + at);
          u32x4 v = *p;
          bool odd = false;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if ((v[e] & kLo) == kLo) {
              v[e] &= 0xffff0000u;
              odd = true;
            }
            if ((v[e] & kHi) == kHi) {
              v[e] &= 0xffffu;
              odd = true;
            }
          }
          if (odd) {
            *p = v;
            atomicOr(&s_bad[(i + 1) & 1], 1u << (at / S::kValueBytes));
          }
        }
        __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
        block_barrier();
        bad = s_bad[(i + 1) & 1];
      }
    }
    // some column of this wavefront's sees a row of the tile
    const bool weigh = busy && i >= 0 && key0 - kLatentTile <= wave_last && key0 > wave_from;
    const bool next = busy && i + 1 < n && key0 <= wave_last && key0 + kLatentTile > wave_from;
    const char *k_stage = ring + k_slot, *v_stage = values_before();
    turn_slots();
    if (!weigh && !next) return;
    // (scores of a tile that is not looked at are of whatever is in LDS, and not used)
    f32x16 then;
    float top, low;
    if (weigh) products(std::true_type{}, k_stage, v_stage, scores, then, top, low);
    else products(std::false_type{}, k_stage, v_stage, scores, then, top, low);
    scores = then;
    if (next) {
      settle(scores, top, low, key0, key0 >= wave_all_from && mul >= 0.0f && bad == 0 &&
                               key0 + kLatentTile - 1 <= min(wave_first, keys.count - 1), bad);
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) scores[e] = -INFINITY;
      scale_by = 1.0f;
    }
  };
  // The same where all columns of the block see all rows of both tiles, and the tile
  // that is loaded is whole: without the questions, which took as long as the products.
  auto inner_step = [&](int i, f32x16& now, f32x16& then) {
    wait_loads<S::kLoads>();
    block_barrier();
    issue();
    const char *k_stage = ring + k_slot, *v_stage = values_before();
    turn_slots();
    float top, low;
    products(std::true_type{}, k_stage, v_stage, now, then, top, low);
    settle(then, top, low, (tile_lo + i + 1) * kLatentTile, true, 0);
  };
  const int whole_lo = max(0, (all_from + kLatentTile - 1) / kLatentTile - tile_lo);
  const int whole_hi = (min(block_first, keys.count - 1) + 1) / kLatentTile - tile_lo;  // tiles [lo, hi)
  const int inner_lo = whole_lo, inner_hi = !CAREFUL && busy && mul >= 0.0f ? min(whole_hi - 1, n - 4) : 0;
  int i = -1;
  for (; i < min(inner_lo, n); ++i) step(i);
  if (i + 2 <= inner_hi) {
    f32x16 other;
    for (; i + 2 <= inner_hi; i += 2) {
      inner_step(i, scores, other);
      inner_step(i + 1, other, scores);
    }
  }
  for (; i < n; ++i) step(i);
  if constexpr (!CAREFUL) {
    // (columns past the tokens have the last one's sums; a wavefront without columns
    // has seen nothing)
    float odd = l * 0.0f;
#pragma unroll
    for (int d = 0; d < S::kTilesD; ++d) {
#pragma unroll
      for (int e = 0; e < 16; ++e) odd = fmaf(o[d][e], 0.0f, odd);
    }
    if (__any(odd != 0.0f || lowest < -3.4028235e38f) && lane == 0) s_bad[0] = 1;
    __syncthreads();
    if (s_bad[0]) return false;
  }
  l += __shfl_xor(l, 32);
  poison += __shfl_xor(poison, 32);
  l += poison;
  if (part >= 0) {
    float* to = a.parts + (static_cast<int64_t>(part) * a.heads + head) * rows_part_floats(DV);
#pragma unroll
    for (int d = 0; d < S::kTilesD; ++d) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = o[d][4 * k + e];
        *reinterpret_cast<f32x4*>(to + (((wave * S::kTilesD + d) * 4 + k) * kWave + lane) * 4) = v;
      }
    }
    if (h == 0) {
      to[kRowUnit * DV + 32 * wave + c] = m;
      to[kRowUnit * (DV + 1) + 32 * wave + c] = l;
    }
    return true;
  }
  if (!mine) return true;
  const float inv = 1.0f / l;
  const bool empty = m == -INFINITY && l == 0.0f;
  uint16_t* to = a.out + static_cast<int64_t>(unit_row + token) * a.out_token + head * a.out_head + 4 * h;
#pragma unroll
  for (int d = 0; d < S::kTilesD; ++d) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = o[d][4 * k + e];
      latent_put<T>(to + 32 * d + 8 * k, v, inv, empty, a.unit.up);
    }
  }
  if (a.lse && h == 0) {
    a.lse[static_cast<int64_t>(unit_row + token) * a.heads + head] = latent_lse<T>(m, l, S::kBias);
  }
  return true;
}

template <class T, int DK, int DV>
__global__ __launch_bounds__(256, 2) void rows_attend_kernel(RowsArgs a) {
  typedef RowsShape<T, DK, DV> S;
  static_assert(S::kKeyLoads * 4096 == S::kKeyTile && S::kValueLoads * 4096 == S::kValueTile,
                "whole loads to a wavefront");
  __shared__ __align__(1024) char ring[S::kLds];
  __shared__ uint32_t s_bad[2];
  const auto* plan = reinterpret_cast<ConstLatentHead>(reinterpret_cast<uintptr_t>(a.work));
  // (heads go to the XCDs in turn with their blocks)
  const int head = static_cast<int>(blockIdx.x % a.heads), nth = static_cast<int>(blockIdx.x / a.heads);
  const auto* at = reinterpret_cast<ConstRowItem>(reinterpret_cast<uintptr_t>(a.work) + a.at_items) + nth;
  const RowItem u{at->request, at->row, at->tokens, at->pos, at->piece, at->pieces, at->part, at->tiles};
  if (nth >= plan->row_items || u.tokens <= 0) return;
  if (threadIdx.x < 2) s_bad[threadIdx.x] = 0;  // (the first stage's barrier is after)
  if (attend_piece<T, DK, DV, false>(a, head, u, ring, s_bad)) return;
  __syncthreads();
  if (threadIdx.x < 2) s_bad[threadIdx.x] = 0;
  attend_piece<T, DK, DV, true>(a, head, u, ring, s_bad);
}

// Joins the parts of units in pieces: 1024 values to a step of a block, as they lie.
template <class T, int DV>
__global__ __launch_bounds__(256) void rows_join_kernel(RowsArgs a, float bias) {
  const auto* plan = reinterpret_cast<ConstLatentHead>(reinterpret_cast<uintptr_t>(a.work));
  const auto* joins = reinterpret_cast<ConstRowJoin>(reinterpret_cast<uintptr_t>(a.work) + a.at_row_joins);
  constexpr int kSteps = kRowUnit * DV / 1024;
  const int64_t all = static_cast<int64_t>(plan->row_joins) * a.heads * kSteps;
  for (int64_t step = blockIdx.x; step < all; step += gridDim.x) {
    const int piece = static_cast<int>(step % kSteps), head = static_cast<int>(step / kSteps % a.heads);
    const auto* j = joins + step / kSteps / a.heads;
    const int at = 256 * piece + static_cast<int>(threadIdx.x);  // of four values
    const int lane = at % kWave, k = at / kWave % 4, d = at / (4 * kWave) % (DV / 32), wave = at / (DV * 8);
    const int token = 32 * wave + lane % 32, x = 32 * d + 8 * k + 4 * (lane / 32);
    if (token >= j->tokens) continue;
    auto part = [&](int p) {
      return a.parts + (static_cast<int64_t>(j->part + p) * a.heads + head) * rows_part_floats(DV);
    };
    float m = -INFINITY, l = 0.0f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int kBatch = 4;  // parts whose loads go out together
    for (int p0 = 0; p0 < j->parts; p0 += kBatch) {
      float pm[kBatch], pl[kBatch];
      f32x4 po[kBatch];
#pragma unroll
      for (int e = 0; e < kBatch; ++e) {
        const float* p = part(min(p0 + e, j->parts - 1));
        pm[e] = p[kRowUnit * DV + token];
        pl[e] = p[kRowUnit * (DV + 1) + token];
        po[e] = *reinterpret_cast<const f32x4*>(p + 4 * at);
      }
      float m2 = m;
#pragma unroll
      for (int e = 0; e < kBatch; ++e) m2 = p0 + e < j->parts ? fmaxf(m2, pm[e]) : m2;
      const float keep = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - m2);
      o *= keep;
      l = l == l ? l * keep : l;
#pragma unroll
      for (int e = 0; e < kBatch; ++e) {
        if (p0 + e < j->parts) {
          // nothing seen: sums of 0 (or NaN, which stays)
          const float f = pm[e] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(pm[e] - m2);
          o += po[e] * f;
          l += pl[e] == pl[e] ? pl[e] * f : NAN;
        }
      }
      m = m2;
    }
    const bool empty = m == -INFINITY && l == 0.0f;
    latent_put<T>(a.out + static_cast<int64_t>(j->row + token) * a.out_token + head * a.out_head + x, o,
                  1.0f / l, empty, a.unit.up);
    if (a.lse && x == 0) {
      a.lse[static_cast<int64_t>(j->row + token) * a.heads + head] = latent_lse<T>(m, l, bias);
    }
  }
}

// Any dims: one block to a (token, head); each of its wavefronts takes 64 rows in
// turn, a row to a lane for the scores and eight columns to a lane for the values.
template <class T>
__global__ __launch_bounds__(256) void rows_any_kernel(RowsArgs a) {
  const int row = blockIdx.x, head = blockIdx.y;
  const int lane = __lane_id(), wave = threadIdx.x / kWave;
  __shared__ float s_q[512];
  __shared__ float s_p[4][kWave];
  __shared__ float s_o[4][512];
  __shared__ float s_m[4], s_l[4];
  if (row >= a.cu_new[a.requests]) return;
  const int r = last_not_past(a.cu_new, a.requests, row);
  const KeyRows keys = key_rows(a, r);
  const int pos = clamp_len(a.ctx_lens[r]) + row - a.cu_new[r] - keys.start;
  const int first = a.window > 0 ? max(0, pos + 1 - a.window) : 0;
  const int last = min(pos, keys.count - 1);
  const uint16_t* q = a.q + static_cast<int64_t>(row) * a.q_token + head * a.q_head;
  for (int d = threadIdx.x; d < a.key_dim; d += 256) s_q[d] = T::get(q[d]);
  __syncthreads();
  const uint16_t* k = a.k + keys.first * a.k_row + head * a.k_head;
  const uint16_t* v = a.v + keys.first * a.v_row + head * a.v_head;
  float m = -INFINITY, l = 0.0f, o[8] = {};
  for (int t0 = first / kWave * kWave + wave * kWave; t0 <= last; t0 += 4 * kWave) {
    const int key = t0 + lane;
    float s = -INFINITY;
    if (key >= first && key <= last) {
      float dot = 0.0f;
      for (int d = 0; d < a.key_dim; d += 8) {
        float x[8];
        get8<T, true>(k + key * a.k_row + d, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) dot = fmaf(s_q[d + e], x[e], dot);
      }
      s = fabsf(dot) <= 3.4028235e38f ? dot * a.scale * kLog2e : NAN;
    }
    float top = s;
    if (__any(s != s)) l = NAN;
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
    const float m2 = fmaxf(m, top);
    if (m2 == -INFINITY) continue;
    const float keep = __builtin_amdgcn_exp2f(m - m2);
    m = m2;
    const float p = s > -INFINITY ? __builtin_amdgcn_exp2f(s - m2) : 0.0f;
    float sum = p;
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
    l = l * keep + sum;
    s_p[wave][lane] = p * a.unit.down;
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] *= keep;
    if (8 * lane < a.value_dim) {
      const int lo = max(0, first - t0), hi = min(kWave, last + 1 - t0);
      for (int j = lo; j < hi; ++j) {
        const float w = s_p[wave][j];
        float x[8];
        get8<T, true>(v + (t0 + j) * a.v_row + 8 * lane, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = fmaf(w, x[e], o[e]);
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
  if (8 * lane < a.value_dim) {
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
  uint16_t* out = a.out + static_cast<int64_t>(row) * a.out_token + head * a.out_head;
  for (int d = threadIdx.x; d < a.value_dim; d += 256) {
    const float x = f[0] * s_o[0][d] + f[1] * s_o[1][d] + f[2] * s_o[2][d] + f[3] * s_o[3][d];
    out[d] = T::put(total == 0.0f ? 0.0f : x / total * a.unit.up);
  }
  if (a.lse && threadIdx.x == 0) {
    a.lse[static_cast<int64_t>(row) * a.heads + head] =
        total == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(total)) * kLn2;
  }
}

// The matrix cores' dims of keys and values.
static bool rows_cores(int key_dim, int value_dim) {
  return (key_dim == 192 && value_dim == 128) || (key_dim == 96 && value_dim == 64) ||
         (key_dim == 128 && value_dim == 128);
}

template <class T, int DK, int DV>
static void launch_rows_cores(const RowsArgs& a, const LatentLayout& l, hipStream_t s) {
  rows_attend_kernel<T, DK, DV><<<static_cast<unsigned>(l.cap_items * a.heads), 256, 0, s>>>(a);
  if (l.cap_row_joins == 0) return;
  const uint64_t steps = l.cap_row_joins * a.heads * (kRowUnit * DV / 1024);
  rows_join_kernel<T, DV><<<static_cast<unsigned>(std::min<uint64_t>(steps, 4 * l.runs[1])), 256, 0, s>>>(
      a, RowsShape<T, DK, DV>::kBias);
}

template <class T>
static void launch_rows(const RowsArgs& a, const LatentLayout& l, bool cores, hipStream_t s) {
  if (!cores) {
    rows_any_kernel<T><<<dim3(static_cast<unsigned>(a.tokens), static_cast<unsigned>(a.heads)), 256, 0, s>>>(a);
  } else if (a.key_dim == 192) {
    launch_rows_cores<T, 192, 128>(a, l, s);
  } else if (a.key_dim == 96) {
    launch_rows_cores<T, 96, 64>(a, l, s);
  } else {
    launch_rows_cores<T, 128, 128>(a, l, s);
  }
}

}  // namespace kv
}  // namespace grm

using namespace grm::kv;

extern "C" int grm_hip_latent_expand(const grm_latent_desc* c, const void* weight, int heads,
                                     int key_dim, int value_dim, const int32_t* block_table,
                                     int table_width, int requests, const int32_t* starts,
                                     const int32_t* cu_rows, uint64_t rows, void* k_out, void* v_out,
                                     void* stream) {
  GRM_CHECK_RC(check_latent(c));
  GRM_CHECK_RC(check_ranges(block_table, table_width, requests, starts, cu_rows, rows));
  if (heads <= 0 || heads > 65535) return grm::fail(-1, "bad heads");
  if (key_dim <= 0 || key_dim > 512 || key_dim % 8 != 0 || value_dim <= 0 || value_dim > 512 ||
      value_dim % 8 != 0) {
    return grm::fail(-1, "key_dim and value_dim must be multiples of 8, at most 512");
  }
  if (rows == 0) {
    grm::clear_error();
    return 0;
  }
  if (!weight || !k_out || !v_out) return grm::fail(-1, "null weight or output");
  if (!aligned16(weight) || !aligned16(k_out) || !aligned16(v_out)) {
    return grm::fail(-1, "weight and outputs must be 16-byte aligned");
  }
  ExpandArgs a{};
  a.rows = static_cast<const uint16_t*>(c->rows);
  a.weight = static_cast<const uint16_t*>(weight);
  a.k = static_cast<uint16_t*>(k_out);
  a.v = static_cast<uint16_t*>(v_out);
  a.of = {block_table, starts, cu_rows, table_width, requests, block_log2(c->block_tokens), rows,
          c->blocks};
  a.rank = c->rank;
  a.rope = c->rope;
  a.heads = heads;
  a.key_dim = key_dim;
  a.value_dim = value_dim;
  const auto s = static_cast<hipStream_t>(stream);
  const bool bf = c->dtype == grm::kBF16;
  const uint64_t columns = static_cast<uint64_t>(heads) * (key_dim + value_dim);
  const uint64_t blocks = (rows + kExpandRows - 1) / kExpandRows * ((columns + kExpandCols - 1) / kExpandCols);
  GRM_CHECK_RC(check_blocks(c->rank % kExpandStep == 0 ? blocks : rows));
  if (c->rank % kExpandStep == 0) {
    const auto grid = static_cast<unsigned>(blocks);
    if (bf) latent_expand_kernel<BF16><<<grid, 256, 0, s>>>(a);
    else latent_expand_kernel<F16><<<grid, 256, 0, s>>>(a);
  } else {
    const auto grid = static_cast<unsigned>(rows);
    if (bf) latent_expand_any_kernel<BF16><<<grid, 256, 0, s>>>(a);
    else latent_expand_any_kernel<F16><<<grid, 256, 0, s>>>(a);
  }
  GRM_HIP_CHECK(hipGetLastError());
  grm::clear_error();
  return 0;
}

extern "C" int grm_hip_rows_attend_bytes(const grm_kv_batch_desc* b, int key_dim, int value_dim,
                                         uint64_t* out_bytes) {
  if (!out_bytes) return grm::fail(-1, "null output pointer");
  GRM_CHECK_RC(check_batch(b, false));
  LatentLayout l;
  GRM_CHECK_RC(latent_layout_of(b, &l));
  *out_bytes = rows_cores(key_dim, value_dim) && l.cap_row_joins
                   ? l.cap_parts * b->heads * rows_part_floats(value_dim) * 4
                   : 0;
  grm::clear_error();
  return 0;
}

extern "C" int grm_hip_rows_attend(const grm_kv_batch_desc* b, const void* work, uint64_t work_bytes,
                                   int dtype, int key_dim, int value_dim, const void* q,
                                   int64_t q_token_stride, int64_t q_head_stride, const void* k,
                                   int64_t k_row_stride, int64_t k_head_stride, const void* v,
                                   int64_t v_row_stride, int64_t v_head_stride, uint64_t rows,
                                   const int32_t* cu_rows, const int32_t* starts, void* out,
                                   int64_t out_token_stride, int64_t out_head_stride, float* lse,
                                   float softmax_scale, void* scratch, uint64_t scratch_bytes,
                                   void* stream) {
  GRM_CHECK_RC(check_batch(b, true));
  if (b->kv_heads != 1) return grm::fail(-1, "a latent cache's batch has one kv head");
  if (dtype != grm::kBF16 && dtype != grm::kF16) return grm::fail(-1, "dense rows are BF16 or F16");
  if (key_dim <= 0 || key_dim > 512 || key_dim % 8 != 0 || value_dim <= 0 || value_dim > 512 ||
      value_dim % 8 != 0) {
    return grm::fail(-1, "key_dim and value_dim must be multiples of 8, at most 512");
  }
  if (rows > static_cast<uint64_t>(kMaxLen)) return grm::fail(-1, "too many rows");
  if (!(softmax_scale - softmax_scale == 0.0f)) return grm::fail(-1, "softmax_scale must be finite");
  if (b->requests == 0 || b->tokens == 0) {
    grm::clear_error();
    return 0;
  }
  if (!q || !out || !cu_rows || (rows && (!k || !v))) return grm::fail(-1, "null array");
  if (!aligned16(q) || !aligned16(out) || !aligned16(k) || !aligned16(v) ||
      (q_token_stride | q_head_stride | out_token_stride | out_head_stride | k_row_stride |
       k_head_stride | v_row_stride | v_head_stride) % 8 != 0) {
    return grm::fail(-1, "queries, rows and output: 16-byte aligned rows");
  }
  if (!work || !aligned16(work)) return grm::fail(-1, "latent work must be 16-byte aligned");
  // the matrix cores' kernel takes a tile's rows by 32-bit offsets
  const auto near = [](int64_t stride) { return stride >= 0 && stride < (1ll << 25); };
  const bool shape = rows_cores(key_dim, value_dim) && near(k_row_stride) && near(v_row_stride);
  if (!shape) GRM_CHECK_RC(check_blocks(static_cast<uint64_t>(b->tokens)));
  LatentLayout l;
  GRM_CHECK_RC(latent_layout_of(b, &l));
  if (work_bytes < l.bytes) return grm::fail(-1, "work is smaller than grm_hip_latent_work_bytes");
  RowsArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.out = static_cast<uint16_t*>(out);
  a.lse = lse;
  a.cu_new = b->cu_new;
  a.ctx_lens = b->ctx_lens;
  a.cu_rows = cu_rows;
  a.starts = starts;
  a.work = static_cast<const char*>(work);
  a.q_token = q_token_stride;
  a.q_head = q_head_stride;
  a.k_row = k_row_stride;
  a.k_head = k_head_stride;
  a.v_row = v_row_stride;
  a.v_head = v_head_stride;
  a.out_token = out_token_stride;
  a.out_head = out_head_stride;
  a.parts = static_cast<float*>(scratch);
  a.at_items = l.at_items;
  a.at_row_joins = l.at_row_joins;
  a.unit = sum_unit(dtype, static_cast<int64_t>(rows));
  a.scale = softmax_scale;
  a.requests = b->requests;
  a.tokens = b->tokens;
  a.window = b->window;
  a.heads = b->heads;
  a.key_dim = key_dim;
  a.value_dim = value_dim;
  a.rows = static_cast<int32_t>(rows);
  const bool cores = shape && l.cap_items * static_cast<uint64_t>(b->heads) <= kMaxBlocks;
  if (!cores) GRM_CHECK_RC(check_blocks(static_cast<uint64_t>(b->tokens)));
  if (cores && l.cap_row_joins) {
    const uint64_t need = l.cap_parts * b->heads * rows_part_floats(value_dim) * 4;
    if (!scratch || !aligned16(scratch) || scratch_bytes < need) {
      return grm::fail(-1, "scratch is smaller than grm_hip_rows_attend_bytes, or not 16-byte aligned");
    }
  }
  const auto s = static_cast<hipStream_t>(stream);
  if (dtype == grm::kBF16) launch_rows<BF16>(a, l, cores, s);
  else launch_rows<F16>(a, l, cores, s);
  GRM_HIP_CHECK(hipGetLastError());
  grm::clear_error();
  return 0;
}
