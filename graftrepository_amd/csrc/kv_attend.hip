// kv_attend.hip -- causal grouped-query attention over the 8-bit key/value
// cache.
//
//   s_j = scale * (q . kc_j) * ks(j),  o = sum_j p_j vs(j) vc_j / sum_j p_j
//
// with p_j = exp(s_j - max s), kc and vc the int8 codes and ks, vs the
// scales of the block that holds token j.  One pass over the cache with a
// running maximum and sum; all sums and statistics in fp32.

#include "kv_attend.hpp"
#include "kv_narrow.hpp"
#include "kv_wide.hpp"

namespace grm {
namespace kv {

// Any head_dim, any number of heads: one block per (token, query head), a
// tile of 64 keys to each of its waves in turn; a lane takes one key for
// the scores and columns lane, lane + 64.. for the values.  Every key byte
// is read once for each query head, so this serves what the matrix-core
// kernels do not take.
template <class T>
__global__ __launch_bounds__(256) void attend_any_kernel(AttendArgs a) {
  const int row = blockIdx.x, h = blockIdx.y, g = h / a.group;
  const int lane = __lane_id(), wave = threadIdx.x / kWave;
  const int hd = a.head_dim, bs = 1 << a.block_log2;
  __shared__ float s_q[256];
  __shared__ float s_p[4][kTile];
  __shared__ float s_o[4][256];
  __shared__ float s_m[4], s_l[4], s_ref[4];
  if (row >= a.cu_new[a.requests]) return;
  int lo = 0, len = a.requests;  // the last request whose first row is not past this one
  while (len > 1) {
    const int half = len >> 1;
    if (a.cu_new[lo + half] <= row) lo += half;
    len -= half;
  }
  const int r = lo;
  const int pos = clamp_len(a.ctx_lens[r]) + row - a.cu_new[r];
  const int first = a.window > 0 ? max(0, pos + 1 - a.window) : 0;
  const typename T::store* q = static_cast<const typename T::store*>(a.q) +
                               row * a.q_token_stride + h * a.q_head_stride;
  for (int d = threadIdx.x; d < hd; d += 256) s_q[d] = T::get(q[d]);
  __syncthreads();

  float m = -INFINITY, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  float ref = 0.0f;  // o is in units of this power of two, above all value scales
  bool odd = false;  // a score that is not a number
  for (int t0 = first / kTile * kTile + wave * kTile; t0 <= pos; t0 += 4 * kTile) {
    const int key = t0 + lane;
    const int j = key >> a.block_log2, p = key & (bs - 1);
    int block = -1;
    if (key >= first && key <= pos && j < a.width) {
      block = a.table[static_cast<size_t>(r) * a.width + j];
      if (static_cast<uint64_t>(static_cast<int64_t>(block)) >= a.blocks) block = -1;
    }
    float s = -INFINITY, vs = 0.0f;
    if (block >= 0) {
      const size_t cell = static_cast<size_t>(block) * a.kv_heads + g;
      const u32x4* k = reinterpret_cast<const u32x4*>(a.k_codes + (cell * bs + p) * hd);
      float dot = 0.0f;
      for (int c = 0; c < hd / 16; ++c) {
        const u32x4 w = k[c];
#pragma unroll
        for (int b = 0; b < 16; ++b) {
          dot = fmaf(s_q[16 * c + b], static_cast<float>(code_at(w[b / 4], b % 4)), dot);
        }
      }
      s = dot * a.k_scales[cell] * a.scale;
      vs = a.v_scales[cell];
    }
    odd |= s != s;
    float top = s, v_top = vs <= 3.0e38f ? vs : 0.0f;
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) {
      top = fmaxf(top, __shfl_xor(top, d));
      v_top = fmaxf(v_top, __shfl_xor(v_top, d));
    }
    const float m2 = fmaxf(m, top);
    if (m2 == -INFINITY) continue;  // no key of this tile is seen
    const float keep = __builtin_amdgcn_exp2f((m - m2) * kLog2e);
    const float ref2 = v_top > ref ? power_above(v_top) : ref;
    const float keep_o = keep * unit_change(ref, ref2);
    ref = ref2;
    const float pr = block >= 0 ? __builtin_amdgcn_exp2f((s - m2) * kLog2e) : 0.0f;
    m = m2;
    float sum = pr;
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
    l = l * keep + sum;
    s_p[wave][lane] = block >= 0 ? pr * (vs * (ref > 0.0f ? 1.0f / ref : 0.0f)) : 0.0f;
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int c = 0; c < 4; ++c) o[c] *= keep_o;
    for (int b0 = 0; b0 < kTile; b0 += 16) {
      // the 16 tokens lie in one block; the window may hide the first
      const uint64_t seen = (__ballot(block >= 0) >> b0) & 0xffffull;
      if (seen == 0) continue;
      const int any = __shfl(block, b0 + __ffsll(static_cast<long long>(seen)) - 1);
      const size_t cell = static_cast<size_t>(any) * a.kv_heads + g;
      const int8_t* v = a.v_codes + cell * bs * hd + ((t0 + b0) & (bs - 1));
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int d = c * kWave + lane;
        if (d < hd) {
          const u32x4 w = *reinterpret_cast<const u32x4*>(v + static_cast<size_t>(d) * bs);
#pragma unroll
          for (int b = 0; b < 16; ++b) {
            o[c] = fmaf(s_p[wave][b0 + b], static_cast<float>(code_at(w[b / 4], b % 4)), o[c]);
          }
        }
      }
    }
  }
  if (__any(odd)) l = NAN;
#pragma unroll
  for (int c = 0; c < 4; ++c) s_o[wave][c * kWave + lane] = o[c];
  if (lane == 0) {
    s_m[wave] = m;
    s_l[wave] = l;
    s_ref[wave] = ref;
  }
  __syncthreads();
  const float top = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  ref = fmaxf(fmaxf(s_ref[0], s_ref[1]), fmaxf(s_ref[2], s_ref[3]));
  float total = 0.0f, f[4];
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    f[w] = s_m[w] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((s_m[w] - top) * kLog2e);
    total += s_l[w] != s_l[w] ? NAN : f[w] * s_l[w];
    f[w] *= unit_change(s_ref[w], ref);
  }
  typename T::store* out = static_cast<typename T::store*>(a.out) + row * a.out_token_stride +
                           h * a.out_head_stride;
  for (int d = threadIdx.x; d < hd; d += 256) {
    const float v = f[0] * s_o[0][d] + f[1] * s_o[1][d] + f[2] * s_o[2][d] + f[3] * s_o[3][d];
    out[d] = T::put(total == 0.0f ? 0.0f : v / total * ref);
  }
  if (a.lse && threadIdx.x == 0) {
    a.lse[static_cast<size_t>(row) * a.heads + h] =
        total == 0.0f ? -INFINITY : top + __builtin_amdgcn_logf(total) * kLn2;
  }
}

// ------------------------------------------------------------- dispatch

struct Shape {
  bool cores;         // the matrix-core kernels take the batch
  uint64_t wide_bytes;  // of scratch that the wide kernel's parts take
  int cap_parts, cap_items, cap_joins;
  int cus;
  uint64_t units;     // at most so many narrow units
  int64_t reach;      // tokens that a request can see
  int runs[2];
  uint64_t at_run_units[2];
  uint64_t narrow_bytes, bytes;  // of scratch: the narrow parts, all
};

static int shape_of(const grm_kv_cache_desc* c, const Layout& l, Shape* out) {
  Shape s{};
  GRM_CHECK_RC(device_cus(&s.cus));
  const int hd = c->head_dim;
  s.cores = (hd == 64 || hd == 128 || hd == 256) && l.group <= kWideCols;
  s.cap_parts = static_cast<int>(l.cap_parts);
  s.cap_items = static_cast<int>(l.cap_items);
  s.cap_joins = static_cast<int>(l.cap_joins);
  s.units = l.cap_units;
  for (int k = 0; k < 2; ++k) {
    s.runs[k] = l.runs[k];
    s.at_run_units[k] = l.at_run_units[k];
  }
  if (s.cores && l.cap_units > 0) {
    s.bytes = static_cast<uint64_t>(c->kv_heads) * l.runs[hd == 256 ? 0 : 1] * 2 *
              narrow_part_floats(hd) * 4;
  }
  if (s.cores) {
    s.wide_bytes = static_cast<uint64_t>(c->kv_heads) * l.cap_parts * wide_part_floats(hd) * 4;
  }
  s.narrow_bytes = (s.bytes + 255) / 256 * 256;
  s.bytes = s.narrow_bytes + s.wide_bytes;
  *out = s;
  return 0;
}

// Measured with a block to a request and with runs and a join (us a call;
// sessions x tokens):          1 x 40       16 x 250     1 x 1000     16 x 1000    1 x 2000
//   bf16, 32 heads on 8 x 128  9.4, 12.0    9.5, 13.2    13.2, 12.1   14.5, 16.9   17.0, 12.2
//   fp32, the same             9.4, 11.2    9.5, 14.5    16.9, 13.4   18.0, 19.6   26.2, 14.0
//   bf16, 12 on 4 x 64         9.4, 11.2    9.3, 11.6    9.2, 11.5    10.2, 11.3   11.1, 11.6
//   fp32, the same             9.3, 11.3    9.4, 11.6    11.2, 11.4   11.4, 11.4   15.9, 11.3
//                                           1 x 500      16 x 500     1 x 1000
//   fp16, 16 on 4 x 256        9.4, 11.6    13.1, 14.8   16.2, 17.2   20.4, 15.2
//   fp32, 8 on 2 x 256         11.0, 13.0   16.9, 17.4   18.8, 19.8   27.4, 17.3
// The bound is where a step of many sessions still gains; a lone one near it
// loses 1 us in 16 bits and 3.5 in fp32.
constexpr int kWholeTokens = 1152;  // to a block, half of it at head_dim 256

template <class T, int D>
static void launch_cores(AttendArgs a, const Shape& s, hipStream_t stream) {
  const auto kv = static_cast<unsigned>(a.kv_heads);
  JoinShape join{a.parts + s.narrow_bytes / 4, 0, 0, 0, 1};
  int joins = 0;
  if (s.cap_items) {
    constexpr int kItems = wide_items(T::code, D);
    AttendArgs b = a;
    b.parts += s.narrow_bytes / 4;
    const unsigned grid = kv * static_cast<unsigned>((s.cap_items + kItems - 1) / kItems);
    attend_wide_kernel<T, D><<<grid, wide_threads(T::code, D), 0, stream>>>(b);
    // eight blocks to a CU, or one to each that there can be
    joins = std::min(s.cap_joins * (kWideCols / join_wide_cols<D>()),
                     std::max(1, 8 * s.cus / a.kv_heads));
  }
  if (s.units) {
    const int k = narrow_blocks_per_cu(T::code, D) - 1;
    a.at_run_units = s.at_run_units[k];
    join.runs = s.runs[k];
    // A block to a request, without a join, where the table (or the window)
    // bounds the requests to kWholeTokens and the blocks run all at once.
    a.whole = s.cap_items == 0 && s.reach <= kWholeTokens * 128 / std::max(128, D) &&
              s.units * kv <= static_cast<uint64_t>(s.cus) * (k + 1);
    const dim3 grid(kv, static_cast<unsigned>(a.whole ? s.units : join.runs / 4));
    if (a.block_log2 == 7) attend_narrow_kernel<T, D, 2><<<grid, 256, 0, stream>>>(a);
    else attend_narrow_kernel<T, D, 1><<<grid, 256, 0, stream>>>(a);
    if (a.whole) return;
    // Blocks to a unit or, where there are fewer, a boundary between two runs:
    // one to a column where eight to a CU are enough for that, else one to a
    // head of the group (three tokens of 7 sessions: 4.6 against 8.5 us; one
    // token of most of 16 sessions with 16 kv heads: 13.3 against 6.9).
    join.by_unit = s.units < static_cast<uint64_t>(join.runs - 1);
    const int places = join.by_unit ? static_cast<int>(s.units) : join.runs - 1;
    join.cols = static_cast<int64_t>(places) * a.cols * a.kv_heads <= 8 * s.cus ? a.cols : a.group;
    join.narrow = places * join.cols;
    joins += join.narrow;
  }
  // no units of either kind (a step that may bring no token): nothing to do
  if (joins) join_kernel<T, D><<<dim3(static_cast<unsigned>(joins), kv), 256, 0, stream>>>(a, join);
}

template <class T>
static void launch(const AttendArgs& a, const Shape& s, hipStream_t stream) {
  if (!s.cores) {
    const dim3 grid(static_cast<unsigned>(a.tokens), static_cast<unsigned>(a.heads));
    attend_any_kernel<T><<<grid, 256, 0, stream>>>(a);
  } else if (a.head_dim == 64) {
    launch_cores<T, 64>(a, s, stream);
  } else if (a.head_dim == 128) {
    launch_cores<T, 128>(a, s, stream);
  } else {
    launch_cores<T, 256>(a, s, stream);
  }
}

}  // namespace kv
}  // namespace grm

using namespace grm::kv;

extern "C" int grm_hip_kv_attend_bytes(const grm_kv_cache_desc* cache,
                                       const grm_kv_batch_desc* batch, uint64_t* out_bytes) {
  if (!out_bytes) return grm::fail(-1, "null output pointer");
  GRM_CHECK_RC(check_pair(cache, batch, false));
  Layout l;
  GRM_CHECK_RC(layout_of(batch, &l));
  Shape s;
  GRM_CHECK_RC(shape_of(cache, l, &s));
  *out_bytes = s.bytes;
  grm::clear_error();
  return 0;
}

extern "C" int grm_hip_kv_attend(const grm_kv_cache_desc* c, const grm_kv_batch_desc* b,
                                 const void* q, int dtype, int64_t q_token_stride,
                                 int64_t q_head_stride, void* out, int64_t out_token_stride,
                                 int64_t out_head_stride, float* lse, float softmax_scale,
                                 void* scratch, uint64_t scratch_bytes, void* stream) {
  GRM_CHECK_RC(check_pair(c, b, true));
  if (dtype != grm::kF32 && dtype != grm::kBF16 && dtype != grm::kF16) {
    return grm::fail(-1, "queries are F32, BF16 or F16");
  }
  if (b->requests == 0 || b->tokens == 0) {
    grm::clear_error();
    return 0;
  }
  if (!q || !out) return grm::fail(-1, "null queries or output");
  const int64_t unit = dtype == grm::kF32 ? 4 : 8;
  if (!aligned16(q) || !aligned16(out) || q_token_stride % unit || q_head_stride % unit ||
      out_token_stride % unit || out_head_stride % unit) {
    return grm::fail(-1, "queries and output: 16-byte aligned rows");
  }
  if (!(softmax_scale == softmax_scale) || softmax_scale - softmax_scale != 0.0f) {
    return grm::fail(-1, "softmax_scale must be finite");
  }
  Layout l;
  GRM_CHECK_RC(layout_of(b, &l));
  if (b->work_bytes < l.bytes) return grm::fail(-1, "work is smaller than grm_hip_kv_work_bytes");
  Shape sh;
  GRM_CHECK_RC(shape_of(c, l, &sh));
  if (scratch_bytes < sh.bytes || (sh.bytes && !scratch)) {
    return grm::fail(-1, "scratch is smaller than grm_hip_kv_attend_bytes");
  }
  if (sh.bytes && !aligned16(scratch)) return grm::fail(-1, "scratch must be 16-byte aligned");
  AttendArgs a{};
  a.k_codes = static_cast<const int8_t*>(c->k_codes);
  a.v_codes = static_cast<const int8_t*>(c->v_codes);
  a.k_scales = c->k_scales;
  a.v_scales = c->v_scales;
  a.q = q;
  a.out = out;
  a.lse = lse;
  a.ctx_lens = b->ctx_lens;
  a.cu_new = b->cu_new;
  // A table without columns may have no memory; entry 0, which the kernels ask
  // for all the same and do not use, is then the first sum's.
  a.table = b->table_width ? b->block_table : b->cu_new;
  a.work = static_cast<const char*>(b->work);
  a.q_token_stride = q_token_stride;
  a.q_head_stride = q_head_stride;
  a.out_token_stride = out_token_stride;
  a.out_head_stride = out_head_stride;
  a.blocks = c->blocks;
  a.scale = softmax_scale;
  a.requests = b->requests;
  a.width = b->table_width;
  a.tokens = b->tokens;
  a.window = b->window;
  a.heads = b->heads;
  a.kv_heads = b->kv_heads;
  a.group = l.group;
  a.head_dim = c->head_dim;
  a.block_log2 = c->block_tokens == 16 ? 4 : c->block_tokens == 32 ? 5 : c->block_tokens == 64 ? 6 : 7;
  a.parts = static_cast<float*>(scratch);
  a.at_units = l.at_units;
  a.at_tiles = l.at_tiles;
  a.at_items = l.at_items;
  a.at_joins = l.at_joins;
  a.cap_parts = sh.cap_parts;
  const int64_t reach = static_cast<int64_t>(b->table_width) * b->block_tokens;
  const int64_t seen = b->window ? static_cast<int64_t>(b->window) + b->max_new : reach;
  sh.reach = std::min(reach, seen);
  a.cols = static_cast<int32_t>(
      std::min<int64_t>(kNarrowCols, static_cast<int64_t>(std::max(1, b->max_new)) * l.group));
  const auto s = static_cast<hipStream_t>(stream);
  if (dtype == grm::kF32) launch<F32>(a, sh, s);
  else if (dtype == grm::kBF16) launch<BF16>(a, sh, s);
  else launch<F16>(a, sh, s);
  GRM_HIP_CHECK(hipGetLastError());
  grm::clear_error();
  return 0;
}
