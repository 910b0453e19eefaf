// Paged key/value cache in 16 bits behind a prefix that the batch shares: shared definitions of its kernels.
//
// Pools lie as [pages][n_kv][page_size][head_dim] of fp16 or bf16.  The prefix's position p lies in page
// prefix_table[p / page_size], position p of sequence b's own part in page block_table[b * max_pages +
// p / page_size]; an id outside [0, n_pages) is no page.
#pragma once
#include "kv8.h"

namespace n730 {

// n / d for n < 2^31 by a product: integer divisions by what a launch gives took a third of the rotary kernel's time
struct FastDiv {
  uint32_t d, m, s;
  FastDiv() = default;
  explicit FastDiv(uint32_t x) : d(x), s(0) {
    while ((1ull << s) < x) ++s;
    m = (uint32_t)((((1ull << s) - x) << 32) / x + 1);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, m) + n) >> s; }
};

// What every call refuses of a cache.
int kv16_check(const N730KV16Cache* c, int batch, const char* what);

// positions of the prefix, within its table's capacity
__device__ __forceinline__ int kv16_prefix(const N730KV16Cache& c) {
  return c.prefix_pages ? min(max(*c.prefix_len, 0), c.prefix_pages * c.page_size) : 0;
}

}  // namespace n730
