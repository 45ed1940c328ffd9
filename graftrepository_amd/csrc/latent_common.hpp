// latent_common.hpp -- what the latent cache's entry points share: the checked
// descriptor and where a request's rows are.
#pragma once

#include "rotary.hpp"

namespace grm {
namespace kv {

int check_latent(const grm_latent_desc* c);
int check_latent_pair(const grm_latent_desc* c, const grm_kv_batch_desc* b, bool with_arrays);

inline int block_log2(int tokens) { return tokens == 16 ? 4 : tokens == 32 ? 5 : tokens == 64 ? 6 : 7; }

// Rows of a request's positions, as a read and an expansion name them.
struct RowRanges {
  const int32_t* table;
  const int32_t* starts;
  const int32_t* cu;
  int32_t width, requests, block_log2;
  uint64_t rows, blocks;
};

int check_ranges(const int32_t* block_table, int table_width, int requests, const int32_t* starts,
                 const int32_t* cu_rows, uint64_t rows);

// Largest i in [0, n) with pre[i] <= x (pre ascending, pre[0] <= x).
__device__ inline int last_not_past(const int32_t* pre, int n, int x) {
  int lo = 0, len = n;
  while (len > 1) {
    const int half = len >> 1;
    if (pre[lo + half] <= x) lo += half;
    len -= half;
  }
  return lo;
}

// The cache's row (block * block_tokens + place) that output row `row` is, -1
// where there is none.
__device__ inline int64_t cache_row(const RowRanges& a, int row) {
  if (static_cast<uint64_t>(static_cast<int64_t>(row)) >= a.rows) return -1;
  const int r = last_not_past(a.cu, a.requests, row);
  if (row < a.cu[r] || row >= a.cu[r + 1]) return -1;
  const int64_t pos = static_cast<int64_t>(a.starts[r]) + row - a.cu[r];
  const int64_t j = pos >> a.block_log2;
  if (pos < 0 || j >= a.width) return -1;
  const int block = a.table[static_cast<size_t>(r) * a.width + j];
  if (static_cast<uint64_t>(static_cast<int64_t>(block)) >= a.blocks) return -1;
  return (static_cast<int64_t>(block) << a.block_log2) + (pos & ((1 << a.block_log2) - 1));
}

}  // namespace kv
}  // namespace grm
