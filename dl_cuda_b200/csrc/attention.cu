// Entry points of the attention operators: argument checks, the choice between the kernels, and the
// workspace layout.  The kernels: attn_generic.cuh (fp32 arithmetic, any layout),
// attn_fwd_mma.cu and attn_bwd_mma.cuh (bf16, whole sequences), attn_step.cu (bf16, few queries).
#include <algorithm>
#include <type_traits>

#include "attn_generic.cuh"
#include "attn_mma.cuh"
#include "attn_step.cuh"

namespace dlb {
namespace {

int check_heads(const char *call, const char *name, const dlb_heads &h, long long elements, int dtype) {
  DLB_REQUIRE(h.ptr != nullptr || elements == 0, DLB_ERR_INVALID_ARG, "%s: null pointer %s", call, name);
  DLB_REQUIRE(on_elements(h.ptr, dtype == DLB_F32 ? 4 : 2), DLB_ERR_INVALID_ARG, "%s: address of %s is not on an element", call, name);
  DLB_REQUIRE(h.batch_stride >= 0 && h.token_stride >= 0 && h.head_stride >= 0, DLB_ERR_INVALID_ARG,
              "%s: negative stride of %s", call, name);
  return DLB_OK;
}

// An output whose elements coincide would be written by several threads at once.
int check_output(const char *call, const char *name, const dlb_heads &h, int batch, int tokens, int heads) {
  DLB_REQUIRE((batch <= 1 || h.batch_stride > 0) && (tokens <= 1 || h.token_stride > 0) && (heads <= 1 || h.head_stride > 0),
              DLB_ERR_INVALID_ARG, "%s: output %s has a stride of 0", call, name);
  return DLB_OK;
}

int check(const char *call, const dlb_attn *a) {
  DLB_REQUIRE(a != nullptr, DLB_ERR_INVALID_ARG, "%s: null argument block", call);
  DLB_REQUIRE(a->batch >= 0 && a->q_len >= 0 && a->kv_len >= 0 && a->heads > 0 && a->kv_heads > 0 && a->head_dim > 0,
              DLB_ERR_INVALID_ARG, "%s: batch=%d heads=%d kv_heads=%d q_len=%d kv_len=%d head_dim=%d", call, a->batch,
              a->heads, a->kv_heads, a->q_len, a->kv_len, a->head_dim);
  DLB_REQUIRE(a->heads % a->kv_heads == 0, DLB_ERR_INVALID_ARG, "%s: heads=%d is no multiple of kv_heads=%d", call,
              a->heads, a->kv_heads);
  DLB_REQUIRE(a->dtype == DLB_F32 || a->dtype == DLB_BF16, DLB_ERR_INVALID_ARG, "%s: dtype=%d", call, a->dtype);
  DLB_REQUIRE(a->causal == 0 || a->causal == 1, DLB_ERR_INVALID_ARG, "%s: causal=%d", call, a->causal);
  DLB_REQUIRE(std::isfinite(a->scale), DLB_ERR_INVALID_ARG, "%s: scale=%g", call, a->scale);
  DLB_REQUIRE(std::isfinite(a->cap) && a->cap >= 0.f, DLB_ERR_INVALID_ARG, "%s: cap=%g", call, a->cap);
  // (an array without elements may have any address, NULL too: that of an empty tensor is)
  DLB_REQUIRE(a->batch == 0 || a->q_len == 0 || a->kv_len == 0 || (a->q_docs == nullptr) == (a->kv_docs == nullptr),
              DLB_ERR_INVALID_ARG, "%s: document numbers are needed for queries and keys, or for neither", call);
  if (a->table) {
    DLB_REQUIRE(a->bucket_of != nullptr, DLB_ERR_INVALID_ARG, "%s: table without bucket_of", call);
    DLB_REQUIRE(a->buckets > 0 && a->max_distance >= 0, DLB_ERR_INVALID_ARG, "%s: buckets=%d max_distance=%d", call,
                a->buckets, a->max_distance);
    DLB_REQUIRE(a->buckets <= DLB_ATTN_MAX_BUCKETS && a->max_distance <= DLB_ATTN_MAX_DISTANCE, DLB_ERR_UNSUPPORTED,
                "%s: buckets=%d (at most %d), max_distance=%d (at most %d)", call, a->buckets, DLB_ATTN_MAX_BUCKETS,
                a->max_distance, DLB_ATTN_MAX_DISTANCE);
  }
  DLB_REQUIRE(a->head_dim <= DLB_ATTN_MAX_HEAD_DIM, DLB_ERR_UNSUPPORTED, "%s: head_dim=%d (at most %d)", call,
              a->head_dim, DLB_ATTN_MAX_HEAD_DIM);
  constexpr int kMaxLen = 1 << 29;
  DLB_REQUIRE(a->q_len <= kMaxLen && a->kv_len <= kMaxLen, DLB_ERR_UNSUPPORTED, "%s: q_len=%d kv_len=%d", call,
              a->q_len, a->kv_len);
  // rows and tiles of rows are counted by 32-bit grids
  const long long tiles = static_cast<long long>(a->batch) * a->heads * (ceil_div(std::max(a->q_len, a->kv_len), 64) + 1);
  const long long rows = static_cast<long long>(a->batch) * a->heads * std::max(a->q_len, 1);
  DLB_REQUIRE(tiles < (1ll << 31) && rows < (1ll << 31), DLB_ERR_UNSUPPORTED,
              "%s: batch=%d heads=%d lengths %d, %d make too many rows", call, a->batch, a->heads, a->q_len, a->kv_len);
  for (const void *p : {static_cast<const void *>(a->kv_lens), static_cast<const void *>(a->q_start), static_cast<const void *>(a->prefix),
                        static_cast<const void *>(a->q_docs), static_cast<const void *>(a->kv_docs), static_cast<const void *>(a->slopes),
                        static_cast<const void *>(a->table), static_cast<const void *>(a->bucket_of), static_cast<const void *>(a->lse)})
    DLB_REQUIRE(on_elements(p, 4), DLB_ERR_INVALID_ARG, "%s: address %p is not a multiple of 4", call, p);
  const long long nq = static_cast<long long>(a->batch) * a->q_len, nk = static_cast<long long>(a->batch) * a->kv_len;
  if (int st = check_heads(call, "q", a->q, nq, a->dtype)) return st;
  if (int st = check_heads(call, "k", a->k, nk, a->dtype)) return st;
  if (int st = check_heads(call, "v", a->v, nk, a->dtype)) return st;
  return check_heads(call, "o", a->o, nq, a->dtype);
}

Heads heads_of(const dlb_heads &h) { return {h.ptr, h.batch_stride, h.token_stride, h.head_stride}; }

AttnArgs args_of(const dlb_attn *a) {
  AttnArgs p = {};
  p.batch = a->batch;
  p.heads = a->heads;
  p.kv_heads = a->kv_heads;
  p.group = a->heads / a->kv_heads;
  p.q_len = a->q_len;
  p.kv_len = a->kv_len;
  p.dim = a->head_dim;
  p.causal = a->causal;
  p.scale = a->scale;
  p.cap = a->cap;
  p.kv_lens = a->kv_lens;
  p.q_start = a->q_start;
  p.prefix = a->prefix;
  const bool docs = a->q_docs && a->kv_docs;  // one alone: the other side is empty, and no pair is left to hide
  p.q_docs = docs ? a->q_docs : nullptr;
  p.kv_docs = docs ? a->kv_docs : nullptr;
  p.slopes = a->slopes;
  p.table = a->table;
  p.buckets = a->table ? a->buckets : 0;
  p.reach = a->table ? a->max_distance : 0;
  p.bucket_of = a->table ? a->bucket_of : nullptr;
  p.q = heads_of(a->q);
  p.k = heads_of(a->k);
  p.v = heads_of(a->v);
  p.o = heads_of(a->o);
  p.lse = a->lse;
  p.splits = 1;
  return p;
}

// Can rows be read 16 bytes at a time?
bool vector_rows(const Heads &h, int dim, int esize) {
  const int v = 16 / esize;
  return aligned16(h.ptr) && dim % v == 0 && h.batch % v == 0 && h.token % v == 0 && h.head % v == 0;
}

// Head width, in the blocks of 32 columns that the fp32-arithmetic kernels are built for.
template <typename F>
auto by_width(int dim, F &&f) {
  if (dim <= 32) return f(std::integral_constant<int, 32>());
  if (dim <= 64) return f(std::integral_constant<int, 64>());
  if (dim <= 96) return f(std::integral_constant<int, 96>());
  return f(std::integral_constant<int, 128>());
}
// Groups of 16 rows per CTA.
template <typename F>
auto by_row_groups(int groups, F &&f) {
  if (groups == 1) return f(std::integral_constant<int, 1>());
  if (groups == 2) return f(std::integral_constant<int, 2>());
  return f(std::integral_constant<int, 4>());
}

// From this many queries on, bf16 goes to the 128-row tiles of the tensor cores; below, the cache is what
// takes time, and the 16 rows of the few-queries kernel are enough.  Measured for 8 sequences, 8192 keys,
// 32 query heads on 8 key heads of 128 (this kernel / the 128-row tiles): 1 query 59 / 225 us, 8 queries
// 111 / 225, 16 queries 196 / 226, 32 queries 360 / 227; one sequence of 32768 keys: 38 / 120, 53 / 118,
// 108 / 119, 195 / 119.
constexpr int kMmaQueries = 17;

enum FwdKind { kGeneric, kMma, kStep };

struct FwdPlan {
  FwdKind kind;
  int pack, splits, row_groups;
  size_t bytes;
};

FwdPlan plan_fwd(const dlb_attn *a, const AttnArgs &args) {
  FwdPlan p = {kGeneric, 1, 1, 4, 0};
  const int group = a->heads / a->kv_heads;
  if (a->dtype == DLB_BF16 && attn_mma_fits(args, false)) p.kind = a->q_len >= kMmaQueries ? kMma : kStep;
  if (p.kind == kMma) {
    p.splits = attn_fwd_mma_splits(args);
  } else if (p.kind == kStep) {
    p.splits = attn_step_splits(a->batch, a->kv_heads, a->q_len * group, a->kv_len, a->head_dim);
  } else {
    // Few queries: the heads that share a key/value head go into one tile, and the keys are split until
    // the grid fills the GPU twice (a share keeps at least two tiles).
    if (static_cast<long long>(a->q_len) * group <= 64) p.pack = group;
    const long long rows = static_cast<long long>(a->q_len) * p.pack, units = static_cast<long long>(a->batch) * (a->heads / p.pack);
    p.row_groups = rows <= 16 ? 1 : rows <= 32 || units * ceil_div(rows, 64ll) < 4 * sm_count() ? 2 : 4;
    const long long ctas = units * ceil_div(rows, 16ll * p.row_groups);
    const int key_tiles = ceil_div(a->kv_len, kGenCols);
    if (ctas > 0 && ctas < sm_count())
      p.splits = static_cast<int>(std::max(1ll, std::min({2ll * sm_count() / ctas, key_tiles / 2ll,
                                                          static_cast<long long>(kMaxSplits)})));
  }
  if (p.splits > 1) {
    const size_t rows = static_cast<size_t>(a->batch) * a->heads * a->q_len * p.splits;
    p.bytes = (rows * sizeof(float2) + 15) / 16 * 16 + rows * sizeof(float) * a->head_dim;
  }
  return p;
}

template <typename T>
int launch_join(const AttnArgs &p, cudaStream_t st) {
  const size_t rows = static_cast<size_t>(p.batch) * p.heads * p.q_len;
  launch_pdl(attn_join_kernel<T>, dim3(static_cast<unsigned>(rows)), dim3(kJoinThreads), 0, st, p);
  DLB_LAUNCH_CHECK("attn_join");
  return DLB_OK;
}

template <typename T>
int launch_fwd(AttnArgs p, const FwdPlan &plan, cudaStream_t st) {
  const bool vec = vector_rows(p.q, p.dim, sizeof(T)) && vector_rows(p.k, p.dim, sizeof(T)) && vector_rows(p.v, p.dim, sizeof(T));
  const int rc = by_width(p.dim, [&](auto width) -> int {
    return by_row_groups(plan.row_groups, [&](auto groups) -> int {
      constexpr int DP = decltype(width)::value, RG = decltype(groups)::value;
      const size_t smem = gen_fwd_smem<DP, RG>();
      auto kern = attn_fwd_generic_kernel<T, DP, RG>;
      if (int s = allow_smem(kern, smem, "attn_fwd")) return s;
      const int tiles = ceil_div(p.q_len * plan.pack, 16 * RG);
      launch_pdl(kern, dim3(tiles * (p.heads / plan.pack) * p.batch, plan.splits), dim3(kGenThreads), smem, st, p, plan.pack, vec);
      DLB_LAUNCH_CHECK("attn_fwd_generic");
      return DLB_OK;
    });
  });
  return rc != DLB_OK || plan.splits == 1 ? rc : launch_join<T>(p, st);
}

struct BwdPlan {
  int parts;  // partial tables per head
  size_t stats_bytes, bytes;
};

BwdPlan plan_bwd(const dlb_attn *a, const dlb_attn_grad *g) {
  BwdPlan p;
  p.stats_bytes = static_cast<size_t>(a->batch) * a->heads * stat_tiles(a->q_len) * 2 * kStatRows * sizeof(float);
  // of the smallest tiles that any kernel uses: 32 queries, or 128 keys
  p.parts = a->batch * std::max(ceil_div(a->q_len, 32), ceil_div(a->kv_len, kTileRows));
  p.bytes = p.stats_bytes;
  if (g->dtable && a->table) p.bytes += sizeof(float) * static_cast<size_t>(a->heads) * p.parts * a->buckets;
  return p;
}

int launch_table_sum(const AttnArgs &p, cudaStream_t st) {
  if (!p.dtable) return DLB_OK;
  launch_pdl(attn_table_sum_kernel, dim3(p.heads * p.buckets), dim3(128), 0, st, p);
  DLB_LAUNCH_CHECK("attn_table_sum");
  return DLB_OK;
}

int launch_bwd_mma(const AttnArgs &p, cudaStream_t st) {
  BwdMaps maps;
  if (int s = make_bwd_maps(p, &maps)) return s;
  if (int s = attn_bwd_mma_queries(p, maps, st)) return s;  // also fills the row statistics for the keys
  if (int s = attn_bwd_mma_keys(p, maps, st)) return s;
  return launch_table_sum(p, st);
}

template <typename T>
int launch_bwd(const AttnArgs &p, cudaStream_t st) {
  const bool vec = vector_rows(p.q, p.dim, sizeof(T)) && vector_rows(p.k, p.dim, sizeof(T)) &&
                   vector_rows(p.v, p.dim, sizeof(T)) && vector_rows(p.dout, p.dim, sizeof(T));
  const size_t rows = static_cast<size_t>(p.batch) * p.heads * stat_tiles(p.q_len) * kStatRows;
  if (rows > 0) {
    const bool pairs = vector_rows(p.o, p.dim, sizeof(T)) && vector_rows(p.dout, p.dim, sizeof(T));
    auto kern = pairs ? attn_row_stats_kernel<T, 8, true> : attn_row_stats_kernel<T, 32, false>;
    launch_pdl(kern, dim3(static_cast<unsigned>(ceil_div(rows, size_t{pairs ? 32u : 8u}))), dim3(256), 0, st, p);
    DLB_LAUNCH_CHECK("attn_row_stats");
  }
  return by_width(p.dim, [&](auto width) -> int {
    // 64-row tiles where they fill the GPU twice, else 32-row ones
    auto blocks = [&](int rows, bool keys) {
      return (keys ? ceil_div(p.kv_len, rows) * p.kv_heads : ceil_div(p.q_len, rows) * p.heads) * p.batch;
    };
    const bool fill = blocks(64, true) + blocks(64, false) >= 2 * sm_count() && blocks(64, true) >= sm_count();
    // (the sums of more than 32 buckets do not fit beside the widest 64-row tiles)
    // one 64-row tile may be the whole sequence: smaller ones would only load the other side twice
    const bool short_rows = p.q_len <= 64 && p.kv_len <= 64;
    const int groups = (fill || short_rows) && !(p.dtable && p.buckets > 32 && p.dim > 64) ? 4 : 2;
    auto launch = [&](auto row_groups) -> int {
      constexpr int DP = decltype(width)::value, RG = decltype(row_groups)::value;
      AttnArgs args = p;
      args.table_parts = p.batch * ceil_div(p.q_len, 16 * RG);
      const size_t smem = gen_bwd_smem<DP, RG>() + gen_table_bytes<RG>(p);
      auto kern = attn_bwd_generic_kernel<T, DP, RG>;
      if (int s = allow_smem(kern, smem, "attn_bwd")) return s;
      const int key_blocks = blocks(16 * RG, true), query_blocks = blocks(16 * RG, false);
      auto pass = [&](int all, int of_keys) -> int {
        if (all == 0) return DLB_OK;
        launch_pdl(kern, dim3(all), dim3(kGenThreads), smem, st, args, vec, of_keys);
        DLB_LAUNCH_CHECK("attn_bwd_generic");
        return DLB_OK;
      };
      if (sizeof(T) == 2) {  // the query pass mends delta for the key pass
        if (int s = pass(query_blocks, 0)) return s;
        if (int s = pass(key_blocks, key_blocks)) return s;
      } else {
        if (int s = pass(key_blocks + query_blocks, key_blocks)) return s;
      }
      return launch_table_sum(args, st);
    };
    return groups == 4 ? launch(std::integral_constant<int, 4>()) : launch(std::integral_constant<int, 2>());
  });
}

int check_workspace(const char *call, const void *workspace, size_t have, size_t need) {
  DLB_REQUIRE(need == 0 || (workspace != nullptr && have >= need && aligned16(workspace)), DLB_ERR_WORKSPACE,
              "%s: workspace of %zu bytes (16-byte aligned) needed, %zu given", call, need, have);
  return DLB_OK;
}

}  // namespace
}  // namespace dlb

using namespace dlb;

extern "C" size_t dlb_attn_fwd_workspace_bytes(const dlb_attn *a) {
  if (check("attn_fwd", a) != DLB_OK || a->batch == 0 || a->q_len == 0) return 0;
  return plan_fwd(a, args_of(a)).bytes;
}

extern "C" int dlb_attn_fwd(const dlb_attn *a, void *workspace, size_t workspace_bytes, void *stream) {
  if (int st = check("attn_fwd", a)) return st;
  if (int st = check_output("attn_fwd", "o", a->o, a->batch, a->q_len, a->heads)) return st;
  if (a->batch == 0 || a->q_len == 0) return DLB_OK;
  AttnArgs p = args_of(a);
  const FwdPlan plan = plan_fwd(a, p);
  if (int rc = check_workspace("attn_fwd", workspace, workspace_bytes, plan.bytes)) return rc;
  cudaStream_t st = as_stream(stream);
  p.splits = plan.splits;
  if (plan.splits > 1) {
    const size_t rows = static_cast<size_t>(a->batch) * a->heads * a->q_len * plan.splits;
    p.part_ml = static_cast<float2 *>(workspace);
    p.part_o = reinterpret_cast<float *>(static_cast<char *>(workspace) + (rows * sizeof(float2) + 15) / 16 * 16);
  }
  if (plan.kind != kGeneric) {
    const int rc = plan.kind == kMma ? attn_fwd_mma(p, st) : attn_step(p, st);
    return rc != DLB_OK || plan.splits == 1 ? rc : launch_join<__nv_bfloat16>(p, st);
  }
  return a->dtype == DLB_F32 ? launch_fwd<float>(p, plan, st) : launch_fwd<__nv_bfloat16>(p, plan, st);
}

extern "C" size_t dlb_attn_bwd_workspace_bytes(const dlb_attn *a, const dlb_attn_grad *g) {
  if (check("attn_bwd", a) != DLB_OK || g == nullptr) return 0;
  return plan_bwd(a, g).bytes;
}

extern "C" int dlb_attn_bwd(const dlb_attn *a, const dlb_attn_grad *g, void *workspace, size_t workspace_bytes,
                            void *stream) {
  if (int st = check("attn_bwd", a)) return st;
  DLB_REQUIRE(g != nullptr, DLB_ERR_INVALID_ARG, "attn_bwd: null gradient block");
  const long long nq = static_cast<long long>(a->batch) * a->q_len, nk = static_cast<long long>(a->batch) * a->kv_len;
  if (int st = check_heads("attn_bwd", "dout", g->dout, nq, a->dtype)) return st;
  if (int st = check_heads("attn_bwd", "dq", g->dq, nq, a->dtype)) return st;
  if (int st = check_heads("attn_bwd", "dk", g->dk, nk, a->dtype)) return st;
  if (int st = check_heads("attn_bwd", "dv", g->dv, nk, a->dtype)) return st;
  if (int st = check_output("attn_bwd", "dq", g->dq, a->batch, a->q_len, a->heads)) return st;
  if (int st = check_output("attn_bwd", "dk", g->dk, a->batch, a->kv_len, a->kv_heads)) return st;
  if (int st = check_output("attn_bwd", "dv", g->dv, a->batch, a->kv_len, a->kv_heads)) return st;
  DLB_REQUIRE(a->lse != nullptr || nq == 0, DLB_ERR_INVALID_ARG, "attn_bwd: lse is needed");
  DLB_REQUIRE(g->dtable == nullptr || a->table != nullptr, DLB_ERR_INVALID_ARG, "attn_bwd: dtable without table");
  DLB_REQUIRE(on_elements(g->dtable, 4), DLB_ERR_INVALID_ARG, "attn_bwd: address of dtable is not a multiple of 4");
  const BwdPlan plan = plan_bwd(a, g);
  if (int st = check_workspace("attn_bwd", workspace, workspace_bytes, plan.bytes)) return st;
  AttnArgs p = args_of(a);
  p.dout = heads_of(g->dout);
  p.dq = heads_of(g->dq);
  p.dk = heads_of(g->dk);
  p.dv = heads_of(g->dv);
  p.dtable = g->dtable;
  p.row_stats = static_cast<float *>(workspace);
  p.table_part = reinterpret_cast<float *>(static_cast<char *>(workspace) + plan.stats_bytes);
  p.table_parts = plan.parts;
  cudaStream_t st = as_stream(stream);
  const bool mma = a->dtype == DLB_BF16 && a->batch > 0 && attn_mma_fits(p, true);
  if (mma) {
    p.table_parts = a->batch * ceil_div(a->kv_len, kTileRows);
    return launch_bwd_mma(p, st);
  }
  return a->dtype == DLB_F32 ? launch_bwd<float>(p, st) : launch_bwd<__nv_bfloat16>(p, st);
}

