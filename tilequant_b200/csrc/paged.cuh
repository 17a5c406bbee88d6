// Shared by the paged-cache kernels: how attention's work over a request's keys is cut.
#pragma once

// Keys of one attention chunk: 32 for each of a block's four warps (see paged_attn.cu).
#define TQ_ATTN_CHUNK 128

// What starting and ending a (request, KV head, row tile) costs a block, in chunks: the plan
// counts so many empty chunks before a group's first, so that blocks with many short groups get
// fewer keys.  (1, 2, 3, 4: 36.1, 33.5, 33.2, 33.3 us for 64 decoding requests of 61 to 4096 keys,
// 46.9, 44.8, 42.5, 42.9 us for 16 requests with up to four new tokens.)
#define TQ_ATTN_LEAD 3
