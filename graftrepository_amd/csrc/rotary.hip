// rotary.hip -- rows of heads turned to their positions.
//
// A block takes some tokens and heads.  It makes the angles of its tokens once,
// in LDS, for all of its heads; then a thread turns eight pairs (two 16-byte
// loads and stores) or copies eight channels that are not turned.  Bound by
// bytes; few rows are one chain: position, angle, values.  8011 rows of 40 heads x 96
// in fp16 take 27 us (123 MB, 4.5 TB/s), 32 rows of 32 heads x 128 3.7.
#include "rotary.hpp"

namespace grm {
namespace kv {

int rotary_of(const grm_rotary_desc* d, int channels, Rotary* out) {
  if (!d) return fail(-1, "null rotary");
  if (d->dim <= 0 || d->dim % 2 != 0 || d->dim > 2 * kMaxPairs) {
    return fail(-1, "rotary: dim must be even, 2 to 256");
  }
  if (d->dim > channels) return fail(-1, "rotary: more channels than there are");
  if (d->layout != kHalf && d->layout != kNeighbours) return fail(-1, "rotary: unknown layout");
  if (!(d->magnitude > 0.0f) || d->magnitude - d->magnitude != 0.0f) {
    return fail(-1, "rotary: magnitude must be positive and finite");
  }
  for (int i = 0; i < d->dim / 2; ++i) {
    // a turn a position at most: the product with a position stays exact enough
    if (!(d->turns[i] >= -1.0 && d->turns[i] <= 1.0)) {
      return fail(-1, "rotary: a frequency past one turn a position");
    }
  }
  *out = Rotary{};
  const double sign = d->inverse ? -1.0 : 1.0;
  for (int i = 0; i < d->dim / 2; ++i) out->quarters[i] = 4.0 * sign * d->turns[i];
  out->magnitude = d->inverse ? 1.0f / d->magnitude : d->magnitude;
  if (out->magnitude - out->magnitude != 0.0f) return fail(-1, "rotary: magnitude too small to divide by");
  out->dim = d->dim;
  out->layout = d->layout;
  return 0;
}

struct RotateArgs {
  const void* x;
  void* out;
  const int32_t* positions;
  int64_t x_token, x_head, out_token, out_head;  // strides
  uint64_t tokens;
  int32_t heads, head_dim, start;
  int32_t tokens_each, heads_each;  // of a block
  int32_t units, copies;            // of a head: turned units, copied runs of eight
};

constexpr int kRotateThreads = 256;
constexpr int kRotateTokens = 8;  // to a block, at most

template <class T, bool ALIGNED>
__global__ __launch_bounds__(kRotateThreads) void rotate_kernel(RotateArgs a, Rotary r) {
  __shared__ CosSin s_angle[kRotateTokens * kMaxPairs];
  __shared__ int s_pos[kRotateTokens];
  const uint64_t t0 = static_cast<uint64_t>(blockIdx.x) * a.tokens_each;
  const int h0 = static_cast<int>(blockIdx.y) * a.heads_each;
  const int n = static_cast<int>(min(static_cast<uint64_t>(a.tokens_each), a.tokens - t0));
  const int heads = min(a.heads_each, a.heads - h0);
  const int pairs = r.dim / 2;
  for (int i = threadIdx.x; i < n * pairs; i += kRotateThreads) {
    const int t = i / pairs, p = i - t * pairs, at = a.positions[t0 + t];
    if (p == 0) s_pos[t] = at;
    s_angle[t * kMaxPairs + p] = angle(r, p, at);
  }
  __syncthreads();
  const int each = a.units + a.copies, items = heads * each;
  typedef typename T::store Store;
  for (int i = threadIdx.x; i < n * items; i += kRotateThreads) {
    const int t = i / items, j = i - t * items;
    const int h = j / each, u = j - h * each;
    if (s_pos[t] < 0) continue;
    const Store* x = static_cast<const Store*>(a.x) + static_cast<int64_t>(t0 + t) * a.x_token +
                     static_cast<int64_t>(h0 + h) * a.x_head;
    Store* out = static_cast<Store*>(a.out) + static_cast<int64_t>(t0 + t) * a.out_token +
                 static_cast<int64_t>(h0 + h) * a.out_head;
    if (u < a.units) {
      int first, second;
      unit_channels(r.layout, pairs, u, &first, &second);
      float v[2][8];
      get8<T, ALIGNED>(x + a.start + first, v[0]);
      get8<T, ALIGNED>(x + a.start + second, v[1]);
      const CosSin* of = s_angle + t * kMaxPairs + 8 * u;
      turn_unit(r.layout, v, [&](int e) { return of[e]; });
      put8<T, ALIGNED>(out + a.start + first, v[0]);
      put8<T, ALIGNED>(out + a.start + second, v[1]);
    } else {
      int d = 8 * (u - a.units);
      if (d >= a.start) d += r.dim;
      float v[8];
      get8<T, ALIGNED>(x + d, v);
      put8<T, ALIGNED>(out + d, v);
    }
  }
}

// Heads that are no whole units: a pair to a thread, then what is copied.
template <class T>
__global__ __launch_bounds__(kRotateThreads) void rotate_any_kernel(RotateArgs a, Rotary r) {
  typedef typename T::store Store;
  const int pairs = r.dim / 2, each = pairs + a.copies;
  const uint64_t t = blockIdx.x;
  const int at = a.positions[t];
  if (at < 0) return;
  for (int i = threadIdx.x; i < a.heads * each; i += kRotateThreads) {
    const int h = i / each, u = i - h * each;
    const Store* x = static_cast<const Store*>(a.x) + static_cast<int64_t>(t) * a.x_token + h * a.x_head;
    Store* out = static_cast<Store*>(a.out) + static_cast<int64_t>(t) * a.out_token + h * a.out_head;
    if (u < pairs) {
      const int d = a.start + (r.layout == kHalf ? u : 2 * u);
      const int e = r.layout == kHalf ? d + pairs : d + 1;
      float p = T::get(x[d]), q = T::get(x[e]);
      turn(angle(r, u, at), p, q);
      out[d] = T::put(p);
      out[e] = T::put(q);
    } else {
      int d = u - pairs;
      if (d >= a.start) d += r.dim;
      out[d] = x[d];
    }
  }
}

// As many tokens as a grid has room for.
template <class T>
static void launch_rotate(RotateArgs a, const Rotary& r, bool in_place, hipStream_t stream) {
  const int rest = in_place ? 0 : a.head_dim - r.dim;
  const bool whole = whole_units(r) && a.start % 8 == 0 && a.head_dim % 8 == 0;
  if (!whole) {
    a.copies = rest;
    rotate_any_kernel<T><<<static_cast<unsigned>(a.tokens), kRotateThreads, 0, stream>>>(a, r);
    return;
  }
  a.units = r.dim / 16;
  a.copies = rest / 8;
  // About two items to a thread; few tokens go to more blocks.
  const int each = a.units + a.copies;
  a.heads_each = std::max(1, std::min(a.heads, 2 * kRotateThreads / each));
  a.tokens_each = std::max(1, std::min(kRotateTokens, 2 * kRotateThreads / (a.heads_each * each)));
  while (a.tokens_each > 1 && a.tokens / a.tokens_each < 1024) a.tokens_each /= 2;
  const int64_t unit = sizeof(typename T::store) == 4 ? 4 : 8;
  const bool aligned = aligned16(a.x) && aligned16(a.out) &&
                       (a.x_token | a.x_head | a.out_token | a.out_head) % unit == 0;
  const dim3 grid(static_cast<unsigned>((a.tokens + a.tokens_each - 1) / a.tokens_each),
                  static_cast<unsigned>((a.heads + a.heads_each - 1) / a.heads_each));
  if (aligned) rotate_kernel<T, true><<<grid, kRotateThreads, 0, stream>>>(a, r);
  else rotate_kernel<T, false><<<grid, kRotateThreads, 0, stream>>>(a, r);
}

}  // namespace kv
}  // namespace grm

using namespace grm::kv;

extern "C" int grm_hip_rotate(const grm_rotary_desc* rotary, const void* x, int dtype,
                              int64_t x_token_stride, int64_t x_head_stride, void* out,
                              int64_t out_token_stride, int64_t out_head_stride,
                              const int32_t* positions, uint64_t tokens, int heads, int head_dim,
                              int start, void* stream) {
  if (dtype != grm::kF32 && dtype != grm::kBF16 && dtype != grm::kF16) {
    return grm::fail(-1, "values are F32, BF16 or F16");
  }
  if (heads <= 0 || heads > 65535 || head_dim <= 0 || head_dim > 65536 || start < 0 ||
      start > head_dim) {
    return grm::fail(-1, "bad heads, head_dim or start");
  }
  if (static_cast<int64_t>(heads) * head_dim > 0x7fffffff) return grm::fail(-1, "a row is too long");
  if (tokens > static_cast<uint64_t>(kMaxLen)) return grm::fail(-1, "too many tokens");
  Rotary r;
  GRM_CHECK_RC(rotary_of(rotary, head_dim - start, &r));
  if (tokens == 0) {
    grm::clear_error();
    return 0;
  }
  if (!x || !out || !positions) return grm::fail(-1, "null array");
  if ((out_token_stride == 0 && tokens > 1) || (out_head_stride == 0 && heads > 1)) {
    return grm::fail(-1, "rows or heads of the output are one another's memory");
  }
  RotateArgs a{};
  a.x_token = x_token_stride;
  a.x_head = x_head_stride;
  a.out_token = out_token_stride;
  a.out_head = out_head_stride;
  a.heads = heads;
  a.head_dim = head_dim;
  a.start = start;
  const bool in_place = x == out;
  if (in_place && (x_token_stride != out_token_stride || x_head_stride != out_head_stride)) {
    return grm::fail(-1, "in place, but with other strides");
  }
  const auto s = static_cast<hipStream_t>(stream);
  const int64_t size = dtype == grm::kF32 ? 4 : 2;
  for (uint64_t from = 0; from < tokens; from += kMaxBlocks) {
    const auto row = static_cast<int64_t>(from);
    a.x = static_cast<const char*>(x) + row * x_token_stride * size;
    a.out = static_cast<char*>(out) + row * out_token_stride * size;
    a.positions = positions + row;
    a.tokens = std::min(tokens - from, kMaxBlocks);
    if (dtype == grm::kF32) launch_rotate<F32>(a, r, in_place, s);
    else if (dtype == grm::kBF16) launch_rotate<BF16>(a, r, in_place, s);
    else launch_rotate<F16>(a, r, in_place, s);
  }
  GRM_HIP_CHECK(hipGetLastError());
  grm::clear_error();
  return 0;
}
