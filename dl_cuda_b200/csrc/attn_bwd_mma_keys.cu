// Gradients of the keys, the values and the bias table on the tensor cores (attn_bwd_mma.cuh).
#include "attn_bwd_mma.cuh"

namespace dlb {
int attn_bwd_mma_keys(const AttnArgs &a, const BwdMaps &maps, cudaStream_t st) { return bwd_mma_launch<true>(a, maps, st); }
}  // namespace dlb
