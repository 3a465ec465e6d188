// Gradients of the queries and of the bias table on the tensor cores (attn_bwd_mma.cuh).
#include "attn_bwd_mma.cuh"

namespace dlb {
namespace {
constexpr size_t kMaxSmem = 227 * 1024;
}

bool attn_bwd_mma_room(const AttnArgs &a) {
  const int ring = a.dim <= kBlockCols                ? BwdShape<1, 4>::kRest
                   : a.table && a.dtable != nullptr ? BwdShape<2, 2>::kRest
                                                    : BwdShape<2, 4>::kRest;
  const size_t keys = 1024 + (a.dim <= kBlockCols ? BwdShape<1, 4>::kRest : BwdShape<2, 4>::kRest) + bwd_rest(a, true).total;
  // about 1 KB of static shared memory beside the dynamic
  return std::max(keys, static_cast<size_t>(1024 + ring + bwd_rest(a, false).total)) + 1024 <= kMaxSmem;
}

int attn_bwd_mma_queries(const AttnArgs &a, cudaStream_t st) { return bwd_mma_launch<false>(a, st); }
}  // namespace dlb
