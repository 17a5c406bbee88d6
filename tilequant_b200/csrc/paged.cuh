// Shared by the paged-cache kernels: how attention's work over a request's keys is cut.
#pragma once

// Keys of one attention chunk: 32 for each of a block's four warps (see paged_attn.cu).
#define TQ_ATTN_CHUNK 128
