// Addressing of the key/value cache (KvCache, fa_params.h), shared by the attention, eviction and commit
// kernels.
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

}  // namespace fa
