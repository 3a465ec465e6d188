// Gradients of the queries on the tensor cores (attn_bwd_mma.cuh).
#include "attn_bwd_mma.cuh"

namespace dlb {
int attn_bwd_mma_queries(const AttnArgs &a, const BwdMaps &maps, cudaStream_t st) {
  return bwd_mma_launch<false>(a, maps, st);
}

int make_bwd_maps(const AttnArgs &a, BwdMaps *maps) {
  auto make = [&](CUtensorMap *m, const Heads &h, int tokens, int heads) {
    return make_heads_map(m, h.ptr, a.dim, tokens, heads, a.batch, h.token, h.head, h.batch, kTileRows);
  };
  int rc = make(&maps->q, a.q, a.q_len, a.heads);
  if (!rc) rc = make(&maps->dout, a.dout, a.q_len, a.heads);
  if (!rc) rc = make(&maps->k, a.k, a.kv_len, a.kv_heads);
  if (!rc) rc = make(&maps->v, a.v, a.kv_len, a.kv_heads);
  DLB_REQUIRE(rc == 0, DLB_ERR_CUDA, "attn_bwd: tensor map refused (%d)", rc);
  return DLB_OK;
}
}  // namespace dlb
