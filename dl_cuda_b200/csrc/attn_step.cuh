// A few bf16 queries against a cache (attn_step.cu).
#pragma once

#include "attn_common.cuh"

namespace dlb {

// Shares the keys are split into for `rows` = q_len * group rows per key/value head.
int attn_step_splits(int batch, int kv_heads, int rows, int kv_len, int dim);
int attn_step(const AttnArgs &a, cudaStream_t st);

}  // namespace dlb
