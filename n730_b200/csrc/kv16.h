// Paged key/value cache in 16 bits behind a prefix that the batch shares: shared definitions of its kernels.
//
// Pools lie as [pages][n_kv][page_size][head_dim] of fp16 or bf16.  The prefix's position p lies in page
// prefix_table[p / page_size], position p of sequence b's own part in page block_table[b * max_pages +
// p / page_size]; an id outside [0, n_pages) is no page.
#pragma once
#include "kv8.h"

namespace n730 {

// What every call refuses of a cache.
int kv16_check(const N730KV16Cache* c, int batch, const char* what);

// positions of the prefix, within its table's capacity
__device__ __forceinline__ int kv16_prefix(const N730KV16Cache& c) {
  return c.prefix_pages ? min(max(*c.prefix_len, 0), c.prefix_pages * c.page_size) : 0;
}

}  // namespace n730
