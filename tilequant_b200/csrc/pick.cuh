// The bookkeeping pass shared by the greedy and the sampled pick of a decode step.
#pragma once

#include "common.cuh"

// Decode keys[b] (low word: ~id) into next, token and generated, clear the keys, advance the
// position (see tq_greedy_pick).
int tq_launch_pick_finish(unsigned long long* keys, int n_rows, int64_t* next, int64_t* token, int64_t* generated,
                          int64_t gen_ld, int64_t gen_cols, int64_t* position, int64_t prompt_tokens, cudaStream_t st);
