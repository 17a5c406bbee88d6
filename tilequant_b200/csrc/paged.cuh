// Shared by the paged-cache kernels: how attention's work over a request's keys is cut.
#pragma once

// Keys of one attention chunk: 32 for each of a block's four warps (see paged_attn.cu).
#define TQ_ATTN_CHUNK 128

// What starting and ending a (request, KV head, row tile) costs a block, in chunks: the plan
// counts so many empty chunks before a group's first, so that blocks with many short groups get
// fewer keys.
#define TQ_ATTN_LEAD 2
