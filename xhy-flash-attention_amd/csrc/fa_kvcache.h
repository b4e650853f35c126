// Addressing of the key/value cache (KvCache, fa_params.h) and of the tree mask, shared by the attention, eviction
// and commit kernels.
#pragma once

#include "fa_common.h"
#include "fa_params.h"

namespace fa {

// whether a sequence's length is one, with room for sq more keys behind it
__host__ __device__ inline bool seq_ok(const KvCache& c, int len, int sq) { return len >= 0 && len <= c.slots - sq; }

// Element offset of key j's row of a sequence (without the head); bad: its page is outside the cache
__host__ __device__ inline int64_t slot_offset(const KvCache& c, int bidb, int j, bool& bad) {
  if (c.table == nullptr) return (int64_t)bidb * c.batch + (int64_t)j * c.row;
  const int blk = j / c.page;
  const int pg = c.table[(int64_t)bidb * c.table_row + blk];
  const bool in = pg >= 0 && pg < c.num_pages;
  if (!in) bad = true;
  return (int64_t)(in ? pg : 0) * c.batch + (int64_t)(j - blk * c.page) * c.row;
}

// The tree mask of a sequence is sq rows of sq bytes, mask_row apart: its bytes, and the byte that says whether
// token t sees key j (outside the mask for a key that is no drafted one: cached, or behind the last)
__host__ __device__ inline int mask_bytes(int sq, int mask_row) { return (sq - 1) * mask_row + sq; }
__host__ __device__ inline int mask_offset(int t, int j, int len, int total, int mask_row, int outside) {
  return j >= len && j < total ? t * mask_row + j - len : outside;
}

}  // namespace fa
