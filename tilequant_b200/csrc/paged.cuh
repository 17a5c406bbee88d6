// Shared by the paged-cache kernels: how attention's work over a request's keys is cut.
#pragma once

#include <stdint.h>

namespace tq {
// floor(i * total / parts) for i <= parts < 2^12, total < 2^31: the product is exact in f64, and so is a
// whole quotient, while any other is at least 2^-12 from a whole number (the 64-bit integer division
// takes several times as long).
__device__ __forceinline__ int64_t share(int64_t i, int64_t total, int64_t parts) {
  return (int64_t)((double)(i * total) / (double)parts);
}
}  // namespace tq

// Keys of one attention chunk: 32 for each of a block's four warps (see paged_attn.cu).
#define TQ_ATTN_CHUNK 128

// What starting and ending a (request, KV head, row tile) costs a block, in chunks: the plan
// counts so many empty chunks before a group's first, so that blocks with many short groups get
// fewer keys.  (1, 2, 3, 4: 36.1, 33.5, 33.2, 33.3 us for 64 decoding requests of 61 to 4096 keys,
// 46.9, 44.8, 42.5, 42.9 us for 16 requests with up to four new tokens.)
#define TQ_ATTN_LEAD 3
