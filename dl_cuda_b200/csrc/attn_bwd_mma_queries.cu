// Gradients of the queries and of the bias table on the tensor cores (attn_bwd_mma.cuh).
#include "attn_bwd_mma.cuh"

namespace dlb {
bool attn_bwd_mma_room(const AttnArgs &a) { return !(a.table && a.dtable) || bwd_table_shape(a).parts > 0; }

int attn_bwd_mma_queries(const AttnArgs &a, cudaStream_t st) { return bwd_mma_launch<false>(a, st); }
}  // namespace dlb
